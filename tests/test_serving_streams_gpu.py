"""Calls in flight on two streams at once, each with a workspace of its own."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _both(run):
    """run(i), a generator of launches, for i = 0, 1: one after the other, then interleaved on two streams without a wait in between."""
    want = [[x.clone() for x in run(i)] for i in (0, 1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    its = [run(0), run(1)]
    for _ in want[0]:
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(next(its[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert len(got[i]) == len(want[i]) and all(torch.equal(a, b) for a, b in zip(got[i], want[i]))


@pytest.mark.parametrize("T,H", [(1, 2), (6, 2), (100, 1)])
def test_attention_with_split_keys(T, H):
    from neko_amd import _lib, ops
    S, hd, cap = 1, 64, 8192
    assert _lib.load().neko_attn_kv8_ws_floats(S, H, 1, cap, hd, T, 0, 0, 0) > 0
    caches, qs = [], []
    for i in (0, 1):
        g = torch.Generator(device="cuda").manual_seed(i)
        c = ops.KV8Cache(S, H, cap, hd, dtype=torch.int8 if i else torch.float8_e4m3fn)
        x = torch.randn(S, cap, 2, H, hd, device="cuda", generator=g).to(BF16)
        ops.kv8_append(c, x[:, :, 0], x[:, :, 1], torch.zeros(S, dtype=torch.int32, device="cuda"))
        caches.append(c)
        qs.append([torch.randn(S, T, H, hd, device="cuda", generator=g).to(BF16) for _ in range(40)])
    pos = torch.full((S,), cap - T, dtype=torch.int32, device="cuda")

    def run(i):
        for q in qs[i]:
            yield ops.attn_kv8(caches[i], q, pos)
    torch.cuda.synchronize()
    _both(run)


def test_appends_and_attention():
    """Whole decode steps: every stream writes its own cache and reads it back."""
    from neko_amd import ops
    S, H, hd, cap, N = 2, 4, 64, 4096, 40
    rows = [torch.randn(S, N, 3, H, hd, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).to(BF16) for i in (0, 1)]
    at = [torch.full((S,), 3000 + t, dtype=torch.int32, device="cuda") for t in range(N)]
    fill = torch.randn(S, 3000, 2, H, hd, device="cuda").to(BF16)
    zero = torch.zeros(S, dtype=torch.int32, device="cuda")

    def run(i):
        c = ops.KV8Cache(S, H, cap, hd, dtype=torch.int8)
        ops.kv8_append(c, fill[:, :, 0], fill[:, :, 1], zero)
        for t in range(N):
            ops.kv8_append(c, rows[i][:, t:t + 1, 1], rows[i][:, t:t + 1, 2], at[t])
            yield ops.attn_kv8(c, rows[i][:, t:t + 1, 0], at[t])
    torch.cuda.synchronize()
    _both(run)


@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_verification(temperature):
    from neko_amd import ops
    B, K, V = 4, 5, 30000
    cases = []
    for i in (0, 1):
        g = torch.Generator(device="cuda").manual_seed(i)
        one = []
        for _ in range(20):
            t = 2 * torch.randn(B, K + 1, V, device="cuda", generator=g)
            d = t[:, :K] + 0.5 * torch.randn(B, K, V, device="cuda", generator=g)
            one.append((t, d, d.argmax(-1), torch.rand(B, K, device="cuda", generator=g), torch.rand(B, device="cuda", generator=g)))
        cases.append(one)

    def run(i):
        for t, d, x, u, r in cases[i]:
            kw = dict(draft_logits=d, u=u, r=r) if temperature else {}
            acc, out = ops.verify_draft(t, x, temperature=temperature, **kw)
            yield torch.cat([acc.long()[:, None], out], 1)
    torch.cuda.synchronize()
    _both(run)
