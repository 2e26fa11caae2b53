"""The 8-bit key / value cache and the attention over it, through the tensor-level entry points, against 64-bit restatements."""
import pytest
import torch

from serving_ref import RefCache, attention

pytestmark = pytest.mark.gpu
E4, I8 = torch.float8_e4m3fn, torch.int8
BF16 = torch.bfloat16


def _rows(S, T, H, hd, g, spread=1.0):
    """K and V as views of one fused [S, T, 3, H, hd] projection."""
    x = torch.randn(S, T, 3, H, hd, generator=g) * torch.exp(spread * torch.randn(S, T, 3, H, 1, generator=g))
    return x.to(BF16)


def _dev_i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _check_cache(cache, ref, length):
    from neko_amd import ops
    k, v = ops.kv8_read(cache, _dev_i(length), cache.cap)
    rk, rv = ref.read(length, cache.cap)
    assert torch.equal(k.cpu().double(), rk) and torch.equal(v.cpu().double(), rv)
    for got, want, n in ((cache.k_scale, ref.scale[0], length), (cache.v_scale, ref.scale[1], length)):
        for s in range(cache.nseq):
            nb = (n[s] + cache.block - 1) // cache.block
            assert torch.equal(got[s, :, :nb].cpu().double(), want[s, :, :nb])


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("dtype", [E4, I8], ids=["e4m3", "int8"])
def test_append_read_bitexact(hd, block, dtype):
    """Several appends of different lengths, at positions inside a block, with growing magnitudes (older codes are rounded again)."""
    from neko_amd import ops
    S, H, cap = 3, 5, 192
    g = torch.Generator().manual_seed(hd + block)
    cache = ops.KV8Cache(S, H, cap, hd, dtype=dtype, block=block)
    ref = RefCache(S, H, cap, hd, dtype, block)
    pos = [0, 7, 100]
    ref_pos0 = list(pos)
    # positions below the first append were written earlier
    x = _rows(S, 100, H, hd, g)
    ops.kv8_append(cache, x.cuda()[:, :, 1], x.cuda()[:, :, 2], _dev_i([0, 0, 0]), n_new=_dev_i(ref_pos0))
    ref.append(x[:, :, 1], x[:, :, 2], [0, 0, 0], ref_pos0)
    for T, n in ((1, [1, 1, 1]), (5, [5, 0, 3]), (40, [40, 33, 17]), (1, [1, 1, 1]), (64, [64, 64, 64])):
        x = _rows(S, T, H, hd, g) * (1.0 + T)
        xd = x.cuda()
        ops.kv8_append(cache, xd[:, :, 1], xd[:, :, 2], _dev_i(pos), n_new=_dev_i(n))
        ref.append(x[:, :, 1], x[:, :, 2], pos, n)
        pos = [min(cap, p + m) for p, m in zip(pos, n)]
        _check_cache(cache, ref, pos)


@pytest.mark.parametrize("dtype", [E4, I8], ids=["e4m3", "int8"])
def test_append_edges(dtype):
    """Past the end, outside, zero rows, NaN and infinities, a block that starts afresh, bytes behind the new rows untouched."""
    from neko_amd import ops
    S, H, cap, hd, block = 6, 2, 64, 32, 32
    g = torch.Generator().manual_seed(1)
    cache = ops.KV8Cache(S, H, cap, hd, dtype=dtype, block=block)
    cache.k.view(torch.uint8).fill_(0x35)
    cache.v.view(torch.uint8).fill_(0x35)
    before_k, before_v = cache.k.view(torch.uint8).clone(), cache.v.view(torch.uint8).clone()
    x = _rows(S, 9, H, hd, g)
    x[0, 0, 1:, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0])
    x[1] = 0
    pos, n = [0, 0, 60, 64, -3, 5], [9, 9, 9, 9, 9, 0]
    xd = x.cuda()
    ops.kv8_append(cache, xd[:, :, 1], xd[:, :, 2], _dev_i(pos), n_new=_dev_i(n))
    ref = RefCache(S, H, cap, hd, dtype, block)
    ref.codes = [torch.full_like(c, 0) for c in ref.codes]
    ref.append(x[:, :, 1], x[:, :, 2], pos, n)
    k, v = ops.kv8_read(cache, _dev_i([9, 9, 64, 0, 0, 0]), cap)
    rk, rv = ref.read([9, 9, 64, 0, 0, 0], cap)
    assert torch.equal(k[0].cpu().double(), rk[0]) and torch.equal(v[0].cpu().double(), rv[0])
    assert torch.equal(k[1].cpu().double(), rk[1]) and torch.equal(v[1].cpu().double(), rv[1])
    assert torch.equal(k[2, 60:].cpu().double(), rk[2, 60:]) and torch.equal(v[2, 60:].cpu().double(), rv[2, 60:])
    assert int(k[3:].count_nonzero()) == 0
    ku, vu = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    assert torch.equal(ku[:, :, 9:60], before_k[:, :, 9:60]) and torch.equal(ku[3:], before_k[3:])
    rows = vu.transpose(3, 4).reshape(S, H, cap, hd)
    rows0 = before_v.transpose(3, 4).reshape(S, H, cap, hd)
    assert torch.equal(rows[:2, :, 9:], rows0[:2, :, 9:]) and torch.equal(rows[3:], rows0[3:])
    # set back to 0 and written again: the block forgets its scale
    y = torch.full((S, 1, 3, H, hd), 2.0 ** -20, dtype=BF16)
    yd = y.cuda()
    ops.kv8_append(cache, yd[:, :, 1], yd[:, :, 2], _dev_i([0] * S))
    assert float(cache.k_scale[0, 0, 0]) < 2.0 ** -20
    k, _ = ops.kv8_read(cache, _dev_i([1] * S), 1)
    assert torch.equal(k, yd[:, :, 1])


def _attn_case(S, H, G, hd, cap, T, pos, n, start, window, sinks, dtype, block, seed=0, poison=True):
    from neko_amd import ops
    g = torch.Generator().manual_seed(seed)
    ref = RefCache(S, H, cap, hd, dtype, block)
    end = [max(0, min(cap, p + min(m, T))) if 0 <= p < cap else 0 for p, m in zip(pos, n)]
    x = _rows(S, cap, H, hd, g, spread=0.4)
    ref.append(x[:, :, 1], x[:, :, 2], [0] * S, end)
    cache = ops.KV8Cache(S, H, cap, hd, dtype=dtype, block=block)
    if poison:      # whatever lies outside [start, last row] must not matter: NaN codes (e4m3) or large ones, wild scales
        cache.k.view(torch.uint8).fill_(0x7f)
        cache.v.view(torch.uint8).fill_(0x7f)
        cache.k_scale.fill_(float("inf"))
        cache.v_scale.fill_(float("nan"))
    xd = x.cuda()
    ops.kv8_append(cache, xd[:, :, 1], xd[:, :, 2], _dev_i([0] * S), n_new=_dev_i(end))
    if poison:      # positions before start: NaN values under a finite scale
        ku, vu = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
        for s in range(S):
            if start[s] > 0:
                ku[s, :, :start[s]] = 0x7f
                full = start[s] // 16
                vu[s, :, :full] = 0x7f
                if start[s] % 16:
                    vu[s, :, full, :, :start[s] % 16] = 0x7f
    q = torch.randn(S, T, H * G, hd, generator=g).to(BF16)
    out0 = torch.full((S, T, H * G, hd), 7.0, dtype=BF16)
    out = out0.cuda()
    ops.attn_kv8(cache, q.cuda(), _dev_i(pos), n_new=_dev_i(n), start=_dev_i(start), window=window, sinks=sinks, out=out)
    want, absv, big = attention(q, ref.values(0), ref.values(1), pos, n, start, window, sinks, hd ** -0.5, out0)
    # output rounding 2^-8 |o|; probabilities: rounded to bf16 (2^-8, more than 64 rows a key head) or kept to 16 bits (2^-16); a score's
    # fp32 sum of hd products of magnitude `big` in any order, in numerator and normaliser; sums of up to cap terms; exponential 2^-21
    p_round = 2.0 ** -8 if T * G > 64 else 2.0 ** -16
    tol = 2.0 ** -8 * want.abs() + (p_round + 2 * hd * 2.0 ** -23 * big + cap * 2.0 ** -23 + 2.0 ** -21) * absv
    err = (out.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    for s in range(S):      # rows behind a sequence's last
        last = min(n[s], T, cap - pos[s]) if 0 <= pos[s] < cap else 0
        assert torch.equal(out[s, max(0, last):].cpu(), out0[s, max(0, last):])


@pytest.mark.parametrize("dtype", [E4, I8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("T,G", [(1, 1), (1, 4), (6, 3), (7, 8), (70, 1), (40, 3), (150, 2), (300, 1)])
def test_attn_rows(T, G, hd, dtype):
    """One row, a few, more than one row tile; grouped heads; lengths of one position, of tile borders, at the end of the cache."""
    cap = 320
    pos = [0, 63 - min(T, 63), 64, 129, cap - T, 200]             # (long calls run past the end: the rows behind it stay)
    n = [T] * 5 + [max(1, T // 2)]
    _attn_case(6, 2, G, hd, cap, T, pos, n, [0] * 6, 0, 0, dtype, {32: 16, 64: 32, 128: 64}[hd], seed=T + hd)


@pytest.mark.parametrize("window,sinks", [(1, 0), (17, 0), (64, 4), (100, 70), (500, 3)])
@pytest.mark.parametrize("T", [1, 5, 80])
def test_attn_window_start_empty(T, window, sinks):
    """Windows and sinks around tile borders, left padding, rows that see nothing, sequences without rows."""
    cap = 256
    pos = [0, 100, cap - T, 30, 50, -1, cap, 150]
    n = [T, T, T, T, 0, T, T, 1]
    start = [0, 37, 64, 33 + T // 2, 0, 0, 0, 149]
    _attn_case(8, 2, 2, 64, cap, T, pos, n, start, window, sinks, E4, 16, seed=window)


def test_attn_all_before_start():
    _attn_case(2, 1, 1, 32, 64, 3, [0, 10], [3, 3], [40, 5], 0, 0, I8, 32)


def test_attn_strides_and_heads():
    """q inside a fused projection, out inside a wider buffer; default output and counts."""
    from neko_amd import ops
    S, H, hd, T, cap = 2, 3, 64, 4, 128
    g = torch.Generator().manual_seed(5)
    x = _rows(S, T, H, hd, g)
    xd = x.cuda()
    cache = ops.KV8Cache(S, H, cap, hd, dtype=I8, block=64)
    pos = _dev_i([0, 0])
    ops.kv8_append(cache, xd[:, :, 1], xd[:, :, 2], pos)
    a = ops.attn_kv8(cache, xd[:, :, 0], pos)
    wide = torch.zeros(S, T, 2, H, hd, dtype=BF16, device="cuda")
    b = ops.attn_kv8(cache, xd[:, :, 0].contiguous(), pos, out=wide[:, :, 1], max_len=T)
    assert torch.equal(a, b) and torch.equal(wide[:, :, 1], a) and int(wide[:, :, 0].count_nonzero()) == 0
    assert torch.equal(a[:, 0], ops.kv8_read(cache, _dev_i([1, 1]), 1)[1][:, 0])       # the first row sees itself only


@pytest.mark.parametrize("max_len", [0, 64, 2048])
def test_attn_splits_agree(max_len):
    """The split of the key axis (sized by max_len) changes nothing but roundings; two calls of one split are bit-equal."""
    from neko_amd import ops
    S, H, hd, cap = 1, 2, 64, 2048
    g = torch.Generator().manual_seed(9)
    x = _rows(S, cap, H, hd, g, spread=0.3)
    xd = x.cuda()
    cache = ops.KV8Cache(S, H, cap, hd, block=32)
    ops.kv8_append(cache, xd[:, :, 1], xd[:, :, 2], _dev_i([0]))
    q = torch.randn(S, 1, H, hd, generator=g).to(BF16).cuda()
    a = ops.attn_kv8(cache, q, _dev_i([cap - 1]), max_len=max_len)
    assert torch.equal(a, ops.attn_kv8(cache, q, _dev_i([cap - 1]), max_len=max_len))
    k, v = (t.cpu().double().transpose(1, 2) for t in ops.kv8_read(cache, _dev_i([cap]), cap))
    want, absv, big = attention(q.cpu(), k, v, [cap - 1], [1], [0], 0, 0, hd ** -0.5, torch.zeros(S, 1, H, hd))
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -16 + 2 * hd * 2.0 ** -23 * big + cap * 2.0 ** -23 + 2.0 ** -21) * absv
    assert bool(((a.cpu().double() - want).abs() <= tol).all())


def test_large_offsets():
    """A cache whose bytes pass 2^32: the last sequence's rows land where they belong, the first one's stay."""
    from neko_amd import ops
    S, H, hd, cap = 5, 16, 128, 1 << 19
    k = torch.zeros(S, H, cap, hd, dtype=torch.uint8, device="cuda").view(I8)
    v = torch.zeros(S, H, cap // 16, hd, 16, dtype=torch.uint8, device="cuda").view(I8)
    ks = torch.ones(S, H, cap // 64, device="cuda")
    vs = torch.ones_like(ks)
    cache = ops.KV8Cache.from_tensors(k, v, ks, vs)
    x = torch.randn(S, 2, 3, H, hd, device="cuda").to(BF16)
    pos = _dev_i([0, 1, 2, 3, cap - 2])
    ops.kv8_append(cache, x[:, :, 1], x[:, :, 2], pos)
    start = pos.clone()
    o = ops.attn_kv8(cache, x[:, :, 0], pos, start=start)
    small = ops.KV8Cache(S, H, 64, hd, dtype=I8, block=64)
    there = _dev_i([0, 1, 2, 3, 62])                             # the same places inside a block, older rows of zeros under a scale of 1
    ops.kv8_append(small, x[:, :, 1], x[:, :, 2], there)
    want = ops.attn_kv8(small, x[:, :, 0], there, start=there)
    assert torch.equal(o[:, 0], want[:, 0])                      # one visible key: its value
    assert float((o.float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())


def test_two_streams_and_capture():
    """Append and attention captured into a graph that advances the positions; two graphs and eager calls in between."""
    from neko_amd import ops
    S, H, hd, cap, N = 2, 2, 32, 128, 12
    g = torch.Generator().manual_seed(3)
    x = _rows(S, N, H, hd, g).cuda()

    def eager(dtype):
        cache = ops.KV8Cache(S, H, cap, hd, dtype=dtype)
        pos = _dev_i([0, 3])
        outs = []
        for i in range(N):
            ops.kv8_append(cache, x[:, i:i + 1, 1], x[:, i:i + 1, 2], pos)
            outs.append(ops.attn_kv8(cache, x[:, i:i + 1, 0], pos, start=_dev_i([0, 3])))
            pos += 1
        return torch.cat(outs, 1)

    class Graph:
        def __init__(self, dtype):
            self.cache = ops.KV8Cache(S, H, cap, hd, dtype=dtype)
            self.pos, self.start = _dev_i([0, 3]), _dev_i([0, 3])
            self.row = torch.zeros(S, 1, 3, H, hd, dtype=BF16, device="cuda")
            self.out = torch.zeros(S, 1, H, hd, dtype=BF16, device="cuda")
            self.graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(self.graph):
                ops.kv8_append(self.cache, self.row[:, :, 1], self.row[:, :, 2], self.pos)
                ops.attn_kv8(self.cache, self.row[:, :, 0], self.pos, start=self.start, out=self.out)
                self.pos.add_(1)

        def step(self, r):
            self.row.copy_(r)
            self.graph.replay()
            return self.out.clone()

    want = {d: eager(d) for d in (E4, I8)}
    graphs = {d: Graph(d) for d in (E4, I8)}
    got = {E4: [], I8: []}
    for i in range(N):
        for d in (E4, I8):
            got[d].append(graphs[d].step(x[:, i:i + 1]))
        if i % 3 == 0:
            assert torch.equal(eager(E4)[:, :i + 1], want[E4][:, :i + 1])
            torch.cuda.synchronize()
    for d in (E4, I8):
        assert torch.equal(torch.cat(got[d], 1), want[d])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = eager(I8)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want[I8])


@pytest.mark.parametrize("hd", [32, 128])
@pytest.mark.parametrize("T", [1, 20, 150])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attn_rising_and_falling_scores(hd, T, sign):
    """Scores that climb (or fall) by some hundreds along the keys: the running reference moves many times, or never after the first keys."""
    from neko_amd import ops
    S, H, cap = 1, 2, 512
    g = torch.Generator().manual_seed(T + hd)
    u = torch.randn(1, 1, H, hd, generator=g)
    ramp = sign * torch.linspace(-60.0, 60.0, cap).view(1, cap, 1, 1)
    k = (ramp * u / hd ** 0.5 + 0.1 * torch.randn(S, cap, H, hd, generator=g)).to(BF16)
    v = torch.randn(S, cap, H, hd, generator=g).to(BF16)
    q = (8.0 * u + 0.1 * torch.randn(S, T, H, hd, generator=g)).to(BF16)
    cache = ops.KV8Cache(S, H, cap, hd, dtype=E4, block=16)
    ops.kv8_append(cache, k.cuda(), v.cuda(), _dev_i([0]))
    pos = [cap - T]
    got = ops.attn_kv8(cache, q.cuda(), _dev_i(pos))
    kk, vv = (t.cpu().double().transpose(1, 2) for t in ops.kv8_read(cache, _dev_i([cap]), cap))
    want, absv, big = attention(q, kk, vv, pos, [T], [0], 0, 0, hd ** -0.5, torch.zeros(S, T, H, hd))
    # as in _attn_case, and the exponent (score and reference up to `big` in size): its fp32 roundings, four of big 2^-23 at most
    p_round = 2.0 ** -8 if T > 64 else 2.0 ** -16
    tol = 2.0 ** -8 * want.abs() + (p_round + (2 * hd + 8) * 2.0 ** -23 * big + cap * 2.0 ** -23 + 2.0 ** -21) * absv
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("window,sinks", [(90, 0), (200, 70), (1000, 3)])
def test_attn_window_over_row_tiles(window, sinks):
    """More rows than one row tile takes, with a window and sinks: tiles of keys that some of the rows see, in ragged sequences."""
    _attn_case(3, 1, 2, 64, 1024, 300, [0, 500, 900], [300, 211, 300], [0, 130, 450], window, sinks, E4, 32, seed=window)


@pytest.mark.parametrize("T", [1, 9, 150])
def test_attn_in_place_and_beside(T):
    """`out` may be q itself, or the rows beside q's in one buffer (query rows interleaved over sequences among them)."""
    from neko_amd import ops
    S, H, hd, cap = 3, 2, 64, 256
    g = torch.Generator().manual_seed(T)
    x = _rows(S, T, H, hd, g).cuda()
    cache = ops.KV8Cache(S, H, cap, hd, dtype=I8, block=64)
    pos = _dev_i([0, 40, 100])
    ops.kv8_append(cache, x[:, :, 1], x[:, :, 2], pos)
    want = ops.attn_kv8(cache, x[:, :, 0], pos)
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)              # rows of a position side by side
    assert torch.equal(ops.attn_kv8(cache, turned[:, :, 0], pos, out=turned[:, :, 2]), want)
    assert torch.equal(ops.attn_kv8(cache, x[:, :, 0], pos, out=x[:, :, 0]), want)
    flat = want.clone()
    with pytest.raises(RuntimeError):                                    # one output row for all sequences
        ops.attn_kv8(cache, x[:, :, 1], pos, out=flat[:1].expand(S, T, H, hd))


def test_attn_fresh_output_is_defined():
    """Rows at positions outside the cache are no rows of the call: zeros in a fresh output, without any count given."""
    from neko_amd import ops
    S, H, hd, T, cap = 3, 2, 64, 3, 64
    x = _rows(S, T, H, hd, torch.Generator().manual_seed(1)).cuda()
    cache = ops.KV8Cache(S, H, cap, hd)
    pos = _dev_i([-1, cap, cap - 1])
    ops.kv8_append(cache, x[:, :, 1], x[:, :, 2], pos)
    torch.full((S, T, H, hd), 7.0, dtype=BF16, device="cuda")          # (memory that a fresh output may come from)
    out = ops.attn_kv8(cache, x[:, :, 0], pos)
    assert int(out[:2].count_nonzero()) == 0 and int(out[2, 1:].count_nonzero()) == 0 and bool(torch.isfinite(out).all())
    assert int(out[2, 0].count_nonzero()) > 0


def _attention_by_heads(q, k, v, pos, n, start, window, sinks, scale, out):
    """serving_ref.attention, all rows of a head at once: q [S, T, Hq, hd], k / v fp64 [S, H, cap, hd]."""
    S, T, HQ, hd = q.shape
    H, cap = k.shape[1], k.shape[2]
    G = HQ // H
    want, absv, big = out.double().clone(), torch.zeros(out.shape, dtype=torch.float64), torch.zeros(S, T, HQ, 1, dtype=torch.float64)
    t = torch.arange(cap)
    for s in range(S):
        m = min(n[s], T, cap - pos[s]) if 0 <= pos[s] < cap else 0
        if m <= 0:
            continue
        p = pos[s] + torch.arange(m)[:, None]
        seen = (t <= p) & (t >= start[s])
        if window:
            seen &= (t > p - window) | (t < start[s] + sinks)
        seen = seen[None, None]                                              # [1, 1, m, cap]
        qq = q[s, :m].double().view(m, H, G, hd).permute(1, 2, 0, 3)           # [H, G, m, hd]
        sc = (qq @ k[s].transpose(1, 2)[:, None]) * scale
        sc = sc.masked_fill(~seen, -float("inf"))
        w = torch.nan_to_num(torch.softmax(sc, -1), nan=0.0)
        put = lambda x: x.permute(2, 0, 1, 3).reshape(m, HQ, -1)
        want[s, :m] = put(w @ v[s][:, None])
        absv[s, :m] = put(w @ v[s].abs()[:, None])
        big[s, :m] = put(((qq.abs() @ k[s].abs().transpose(1, 2)[:, None]) * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True))
    return want, absv, big


# heads and rows that take each of the kernels: 16 and 32 rows a wave, 128 and 256 rows through LDS, with one split of the keys and several
@pytest.mark.parametrize("hd,S,H,G,T,cap", [(32, 16, 16, 1, 100, 320), (32, 16, 16, 1, 130, 320), (32, 8, 8, 3, 100, 320), (32, 8, 8, 1, 520, 1024), (64, 16, 16, 1, 20, 320),
                                            (64, 8, 8, 1, 100, 320), (64, 8, 8, 1, 130, 320), (64, 8, 8, 1, 130, 1024), (64, 8, 8, 2, 150, 1024), (64, 16, 16, 1, 100, 320),
                                            (128, 8, 8, 1, 20, 1024), (128, 8, 8, 1, 100, 1024), (128, 8, 8, 1, 130, 1024), (128, 8, 8, 4, 130, 1024), (128, 2, 4, 1, 520, 1024)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 70)])
def test_attn_many_heads(hd, S, H, G, T, cap, window, sinks):
    from neko_amd import ops
    g = torch.Generator().manual_seed(hd + T + window)
    dtype, block = (E4, 16) if (T + window) % 4 else (I8, 64)
    pos = [int(x) for x in torch.randint(0, cap - T // 2, (S,), generator=g)]
    n = [int(x) for x in torch.randint(0, T + 1, (S,), generator=g)]
    n[0], pos[0], n[1], pos[1] = T, cap - T, T, 0
    end = [min(cap, p + m) if m else 0 for p, m in zip(pos, n)]
    start = [int(x) for x in (torch.rand(S, generator=g) * 0.7 * torch.tensor(end))]
    start[0] = 0
    start[1] = min(T // 3, cap - 1)                                            # its first rows see nothing
    cache = ops.KV8Cache(S, H, cap, hd, dtype=dtype, block=block)
    cache.k.view(torch.uint8).fill_(0x7f)                                      # outside the rows: NaN or large codes under wild scales
    cache.v.view(torch.uint8).fill_(0x7f)
    cache.k_scale.fill_(float("inf"))
    cache.v_scale.fill_(float("nan"))
    x = _rows(S, cap, H, hd, g, spread=0.4).cuda()
    ops.kv8_append(cache, x[:, :, 1], x[:, :, 2], _dev_i([0] * S), n_new=_dev_i(end))
    k, v = (a.cpu().double().transpose(1, 2) for a in ops.kv8_read(cache, _dev_i(end), cap))
    q = torch.randn(S, T, H * G, hd, generator=g).to(BF16)
    out0 = torch.full((S, T, H * G, hd), 7.0, dtype=BF16)
    out = out0.cuda()
    ops.attn_kv8(cache, q.cuda(), _dev_i(pos), n_new=_dev_i(n), start=_dev_i(start), window=window, sinks=sinks, out=out)
    want, absv, big = _attention_by_heads(q, k, v, pos, n, start, window, sinks, hd ** -0.5, out0)
    p_round = 2.0 ** -8 if T * G > 64 else 2.0 ** -16                          # tolerances as in _attn_case
    tol = 2.0 ** -8 * want.abs() + (p_round + 2 * hd * 2.0 ** -23 * big + cap * 2.0 ** -23 + 2.0 ** -21) * absv
    err = (out.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    for s in range(S):
        assert torch.equal(out[s, n[s]:].cpu(), out0[s, n[s]:])


@pytest.mark.parametrize("hd,S,H,T,cap", [(32, 16, 16, 100, 320), (32, 16, 16, 130, 320), (128, 8, 8, 130, 1024)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attn_rising_scores_many_heads(hd, S, H, T, cap, sign):
    """test_attn_rising_and_falling_scores through LDS tiles, where the running reference moves only when probabilities outgrow 2^40."""
    from neko_amd import ops
    g = torch.Generator().manual_seed(T + hd)
    u = torch.randn(S, 1, H, hd, generator=g)
    ramp = sign * torch.linspace(-60.0, 60.0, cap).view(1, cap, 1, 1)
    k = (ramp * u / hd ** 0.5 + 0.1 * torch.randn(S, cap, H, hd, generator=g)).to(BF16)
    v = torch.randn(S, cap, H, hd, generator=g).to(BF16)
    q = (8.0 * u + 0.1 * torch.randn(S, T, H, hd, generator=g)).to(BF16)
    cache = ops.KV8Cache(S, H, cap, hd, dtype=E4, block=16)
    ops.kv8_append(cache, k.cuda(), v.cuda(), _dev_i([0] * S))
    pos = [cap - T] * S
    got = ops.attn_kv8(cache, q.cuda(), _dev_i(pos))
    kk, vv = (t.cpu().double().transpose(1, 2) for t in ops.kv8_read(cache, _dev_i([cap] * S), cap))
    want, absv, big = _attention_by_heads(q, kk, vv, pos, [T] * S, [0] * S, 0, 0, hd ** -0.5, torch.zeros(S, T, H, hd))
    # as in test_attn_rising_and_falling_scores
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + (2 * hd + 8) * 2.0 ** -23 * big + cap * 2.0 ** -23 + 2.0 ** -21) * absv
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
