"""Rows that a decoder drops again (drafted tokens that were not kept) leave nothing behind."""
import pytest
import torch

from test_speculative_gpu import _policy, _prompt

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _decoders(kind, d=64, seed=0, block=32):
    """Two decoders of one policy whose keys and values are many times larger for rows with a large first channel."""
    from neko_amd import engine
    m = _policy(seed=seed, d=d, heads=max(2, d // 128), ctx=192)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "c_attn.weight" in n:
                p[0] *= 40.0
    m._flat.ensure_shadow()
    sp = m.transformer._stack_params()
    dt = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}[kind]
    return [engine.KV8Decoder(sp, 192, torch.device(DEV), dtype=dt, block=block) for _ in range(2)]


def _rows(n, d, large, seed):
    x = torch.randn(n, d, generator=torch.Generator().manual_seed(seed))
    x[:, 0] = large
    return x.to(DEV)


def _held(dec):
    from neko_amd import ops
    k, v = ops.kv8_read(dec.cache, torch.full((len(dec.P.layers),), dec.n, dtype=torch.int32, device=DEV), dec.n)
    return torch.stack([k, v])


# positions inside a block, at its border and just before it; with one row for the stack's products and with more than the row kernels take
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("d,block", [(64, 32), (128, 16), (1024, 64)])
@pytest.mark.parametrize("n0,drafted,kept", [(10, 4, 0), (10, 5, 2), (30, 6, 0), (30, 6, 1), (30, 7, 4), (32, 4, 0), (32, 4, 2), (47, 7, 1), (62, 7, 0), (61, 7, 5), (0, 3, 1)])
def test_dropped_rows_leave_nothing(kind, d, block, n0, drafted, kept):
    a, b = _decoders(kind, d, block=block)
    history = _rows(n0, d, 0.0, 1)
    judged, drafts, later = _rows(1, d, 0.0, 2), _rows(drafted, d, 0.0, 3), _rows(3, d, 0.5, 4)
    drafts[kept:, 0] = 60.0                       # what is dropped has far larger keys and values than what stays
    for dec in (a, b):
        dec.extend(history) if n0 else None
    a.mark()
    ha = a.extend(torch.cat([judged, drafts]))
    before = a.n
    a.truncate(n0 + 1 + kept)
    assert before == n0 + 1 + drafted and a.n == int(a.pos) == n0 + 1 + kept
    hb = torch.cat([b.extend(r[None]) for r in torch.cat([judged, drafts[:kept]])])
    assert torch.equal(_held(a), _held(b))
    if d <= 768:                                  # (wider stacks take other products for one row than for several: equal but for rounding)
        assert torch.equal(ha[:kept + 1], hb)
    a.mark()
    for r in later:
        assert torch.equal(a.extend(r[None]), b.extend(r[None]))
    assert torch.equal(_held(a), _held(b))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_single_rows_behind_a_mark(kind):
    """A drafting policy's way: rows one by one behind the mark, dropped in part, twice behind one mark, then in whole."""
    a, b = _decoders(kind)
    for dec in (a, b):
        dec.extend(_rows(20, 64, 0.0, 1))
    a.mark()
    x = _rows(6, 64, 0.0, 2)
    x[2:, 0] = 60.0
    for r in x:
        a.extend(r[None])
    a.truncate(24)
    a.truncate(22)
    for r in x[:2]:
        b.extend(r[None])
    assert torch.equal(_held(a), _held(b))
    assert torch.equal(a.extend(x[2:3]), b.extend(x[2:3]))
    a.truncate(20)
    fresh = _decoders(kind)[0]
    fresh.extend(_rows(20, 64, 0.0, 1))
    assert torch.equal(_held(a), _held(fresh))


def test_truncate_refuses_what_it_cannot_undo():
    a, _ = _decoders("int8")
    a.extend(_rows(40, 64, 0.0, 1))
    with pytest.raises(ValueError, match="mark"):
        a.truncate(37)
    a.mark()
    a.extend(_rows(5, 64, 0.0, 2))
    a.extend(_rows(5, 64, 0.0, 3))                # more rows than a mark covers
    with pytest.raises(ValueError, match="mark"):
        a.truncate(42)
    a.truncate(50)
    a.truncate(32)                                # whole blocks
    a.mark()
    a.extend(_rows(3, 64, 0.0, 2))
    with pytest.raises(ValueError, match="mark"):
        a.truncate(31)
    a.truncate(32)
    a.extend(_rows(3, 64, 0.0, 2))
    a.reset()
    a.extend(_rows(10, 64, 0.0, 2))
    with pytest.raises(ValueError, match="mark"):
        a.truncate(9)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_drafted_decoding_does_not_depend_on_the_draft(kind):
    """From an 8-bit cache, tokens and logits of greedy drafted decoding are those of plain decoding to the bit, whoever drafts and however many."""
    m = _policy(seed=0)
    m.kv_cache = kind
    want, tokens = m.predict_text(_prompt(25), max_length=30)
    for draft, n_draft in ((m, 4), (_policy(seed=3, layers=1), 1), (_policy(seed=3, layers=1), 7), (_policy(seed=5), 3)):
        draft.kv_cache = kind
        got, t = m.predict_text_speculative(_prompt(25), draft, max_length=30, n_draft=n_draft)
        assert [int(x) for x in t] == [int(x) for x in tokens]
        assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_a_mark_ends_where_rows_before_it_go(kind):
    """Whole blocks dropped from before a mark take the mark with them: rows that follow are ordinary ones."""
    a, b = _decoders(kind)
    for dec in (a, b):
        dec.extend(_rows(40, 64, 0.0, 1))
    a.mark()
    a.extend(_rows(3, 64, 60.0, 2))
    for dec in (a, b):
        dec.truncate(32)
        for n, seed in ((1, 3), (4, 4), (5, 5), (2, 6)):              # past the position that the mark stood at
            h = dec.extend(_rows(n, 64, 0.5, seed))
            assert bool(torch.isfinite(h.float()).all())
    assert a.n == b.n == 44 and torch.equal(_held(a), _held(b))
    with pytest.raises(ValueError, match="mark"):
        a.truncate(41)


def test_replayed_steps_end_a_mark():
    """A captured step keeps no rows: what it appended cannot be dropped in part, and is what it would be without a mark."""
    m = _policy(ctx=96)
    m.kv_cache = "int8"
    table, hp = m._flat.view("embed_token.weight"), m._head_params()
    got = []
    for marked in (False, True):
        dec = m._new_decoder(96, torch.device(DEV))
        dec.capture_greedy_step(hp, table, 0, 127)
        dec.extend(m.tokenize_input_dicts([_prompt(20)])[0][0].float())
        if marked:
            dec.mark()
        dec.g_x.copy_(table[5].reshape(1, -1))
        out = [dec.replay_greedy_step() for _ in range(6)]
        got.append((torch.stack([l for l, _ in out]), [int(t) for _, t in out], _held(dec)))
        with pytest.raises(ValueError, match="mark"):
            dec.truncate(22)
    assert torch.equal(got[0][0], got[1][0]) and got[0][1] == got[1][1] and torch.equal(got[0][2], got[1][2])


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(16, 4), (9, 0)])
def test_drafted_decoding_under_a_window(kind, window, sinks):
    """The same with a sliding window that leaves most of the sequence behind."""
    m, draft = _policy(seed=0), _policy(seed=3, layers=1)
    for p in (m, draft):
        p.kv_cache, p.decode_window, p.decode_sinks = kind, window, sinks
    want, tokens = m.predict_text(_prompt(35), max_length=30)
    got, t = m.predict_text_speculative(_prompt(35), draft, max_length=30, n_draft=5)
    assert [int(x) for x in t] == [int(x) for x in tokens] and torch.equal(got, want)
