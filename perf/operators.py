"""Measured cases of the serving and distillation operators: the 8-bit key / value cache (written, read back and attended to), the
verification of drafted tokens and the distillation from a teacher's top logits.

``run`` computes a case either in plain torch (``own`` false) or through the framework's own entry points (``own`` true).
"""
import math

import torch

own = False

F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}
VOCAB = 52305            # text + continuous + discrete tokens of the default policy

# ------------------------------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # one decode step of the default 768-wide policy: the newest row of every head goes into the cache
        dict(name="cache_step", op="cache", S=1, H=24, hd=32, cap=1024, T=1, top=701, ragged=False, dtype="e4m3", block=32),
        # a few drafted rows for eight sequences that stand at different places inside a block of tokens
        dict(name="cache_chunk_odd", op="cache", S=8, H=16, hd=128, cap=1024, T=37, top=1003, ragged=True, dtype="int8", block=64),
        # the prompts of 64 sequences are written at once
        dict(name="cache_prefill", op="cache", S=64, H=24, hd=32, cap=1024, T=1024, top=1024, ragged=True, dtype="e4m3", block=16),
        # one token for one sequence: latency
        dict(name="attn_one_token", op="attn", S=1, H=24, G=1, hd=32, top=1000, T=1, ragged=False, dtype="e4m3", block=32, window=0, sinks=0),
        # one token for each of 32 long sequences of different lengths: the cache's bytes
        dict(name="attn_batch_long", op="attn", S=32, H=16, G=1, hd=128, top=8192, T=1, ragged=True, dtype="int8", block=64, window=0, sinks=0),
        # drafted rows to be checked, shared key heads, a sliding window and four first tokens that stay visible
        dict(name="attn_draft_window", op="attn", S=8, H=8, G=4, hd=64, top=5000, T=6, ragged=True, dtype="e4m3", block=16, window=2048, sinks=4),
        # a prompt's second chunk over what the cache holds: matrix products
        dict(name="attn_chunk", op="attn", S=4, H=16, G=1, hd=128, top=4000, T=1024, ragged=False, dtype="e4m3", block=64, window=0, sinks=0),
        # one sequence, four drafted tokens, sampling
        dict(name="verify_one", op="verify", B=1, K=4, V=VOCAB, T=0.8, draft=True, dtype="f32"),
        # a batch of sequences, seven drafted tokens each
        dict(name="verify_batch", op="verify", B=64, K=7, V=VOCAB, T=1.0, draft=True, dtype="f32"),
        # greedy decoding: the draft has to match the target's best token
        dict(name="verify_greedy", op="verify", B=16, K=5, V=VOCAB, T=0.0, draft=False, dtype="bf16"),
        # the loss rows of a small control batch
        dict(name="distill_small", op="distill", R=77, V=VOCAB, k=16, tau=2.0, hard=0.0, dtype="f32"),
        # the loss rows of a text batch, mixed with the labels' cross-entropy
        dict(name="distill_batch", op="distill", R=8192, V=VOCAB, k=64, tau=1.5, hard=0.25, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)))))))


def draw(rng):
    op = rng.choice(["cache", "attn", "attn", "verify", "distill"])
    if op == "cache":
        hd, H = rng.choice([32, 64, 128]), rng.randint(1, 32)
        cap = 64 * rng.randint(1, 32)
        S = _log(rng, 1, max(1, min(64, 34_000_000 // (H * cap * hd))))
        top = rng.randint(1, cap)
        return dict(op=op, S=S, H=H, hd=hd, cap=cap, T=_log(rng, 1, top), top=top, ragged=rng.random() < 0.6, dtype=rng.choice(["e4m3", "int8"]),
                    block=rng.choice([16, 32, 64]))
    if op == "attn":
        hd, H, G = rng.choice([32, 64, 128]), rng.randint(1, 16), rng.choice([1, 1, 2, 3, 4, 8])
        top = _log(rng, 1, 8192)
        S = _log(rng, 1, max(1, min(32, 700_000_000 // (2 * H * top * hd))))
        T = _log(rng, 1, max(1, min(1024, top, 240_000_000 // (S * H * G * top))))
        window = rng.choice([0, 0, _log(rng, 1, top)])
        return dict(op=op, S=S, H=H, G=G, hd=hd, top=top, T=T, ragged=rng.random() < 0.6, dtype=rng.choice(["e4m3", "int8"]), block=rng.choice([16, 32, 64]),
                    window=window, sinks=rng.choice([0, 1, 4, 21]) if window else 0)
    if op == "verify":
        K, V = rng.randint(1, 8), _log(rng, 500, VOCAB)
        return dict(op=op, B=_log(rng, 1, 56), K=K, V=V, T=rng.choice([0.0, 0.6, 1.0, 1.3]), draft=rng.random() < 0.7, dtype=rng.choice(["f32", "bf16"]))
    return dict(op=op, R=_log(rng, 1, 4096), V=_log(rng, 500, VOCAB), k=_log(rng, 1, 128), tau=rng.choice([1.0, 1.5, 2.0, 4.0]),
                hard=rng.choice([0.0, 0.3, 1.0]), dtype=rng.choice(["f32", "bf16"]))


# ----------------------------------------------------------------------------------------------------------------- inputs


def _scale_of(amax, dtype):
    """Smallest power of two s with amax <= qmax * s (amax > 0; 2^-100 at least)."""
    f, x = torch.frexp(amax)
    top, bits = (0.875, 9) if dtype == "e4m3" else (127.0 / 128.0, 7)
    e = torch.where(amax > 0, x - bits + (f > top).to(x.dtype), torch.full_like(x, -100)).clamp(min=-100)
    return torch.ldexp(torch.ones_like(amax), e)


def _round_codes(x, dtype):
    return x.to(CODES["e4m3"]) if dtype == "e4m3" else torch.round(x).to(torch.int8)


def _rows_to_v(x):
    """[S, H, cap, hd] -> the cache's layout of values [S, H, cap / 16, hd, 16]."""
    S, H, cap, hd = x.shape
    return x.view(S, H, cap // 16, 16, hd).transpose(3, 4).contiguous()


def _v_to_rows(x):
    S, H, n, hd, _ = x.shape
    return x.transpose(3, 4).reshape(S, H, n * 16, hd)


def _heldout_cache(S, H, cap, hd, block, dtype, g, dev):
    """A cache as an earlier part of the sequence left it: channels of different size, a few large tokens."""
    def one(grow):
        x = torch.randn(S, H, cap, hd, generator=g, device=dev)
        x *= torch.exp(0.5 * torch.randn(1, H, 1, hd, generator=g, device=dev))
        x *= 1.0 + grow * (torch.rand(S, 1, cap, 1, generator=g, device=dev) < 0.02)
        s = _scale_of(x.view(S, H, cap // block, block * hd).abs().amax(-1), dtype)
        x /= s.repeat_interleave(block, 2).unsqueeze(-1)
        return _round_codes(x, dtype), s
    k, ks = one(3.0)
    v, vs = one(1.0)
    v8 = _rows_to_v(v.view(torch.uint8)).view(CODES[dtype])
    return k, v8, ks, vs


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    c = dict(case)
    st = {"case": c}
    if c["op"] in ("cache", "attn"):
        S, H, hd, T = c["S"], c["H"], c["hd"], c["T"]
        cap = c["cap"] if c["op"] == "cache" else (c["top"] + 63) // 64 * 64
        st["k8"], st["v8"], st["ks"], st["vs"] = _heldout_cache(S, H, cap, hd, c["block"], c["dtype"], g, dev)
        if c["ragged"]:      # the first sequence is the longest; the others stand elsewhere, and bring fewer rows
            n = torch.randint(1, T + 1, (S,), generator=g, device=dev)
            pos = (torch.rand(S, generator=g, device=dev) ** 0.5 * (c["top"] - n + 1)).long()
            n[0], pos[0] = T, c["top"] - T
        else:
            n = torch.full((S,), T, device=dev)
            pos = torch.full((S,), c["top"] - T, device=dev)
        st["pos"], st["n"] = pos.to(torch.int32), n.to(torch.int32)
        if c["op"] == "cache":
            # the fused projection's output: rows of [q | k | v]
            st["qkv"] = torch.randn(S, T, 3, H, hd, generator=g, device=dev).mul_(1.5).to(BF16)
            st["end"] = st["pos"] + st["n"]
        else:
            st["q"] = torch.randn(S, T, H * c["G"], hd, generator=g, device=dev).to(BF16)
            # left-padded prompts where lengths differ
            st["start"] = (st["pos"] // 16 if c["ragged"] else torch.zeros_like(st["pos"])).to(torch.int32)
            st["out"] = torch.zeros(S, T, H * c["G"], hd, dtype=BF16, device=dev)
    elif c["op"] == "verify":
        B, K, V = c["B"], c["K"], c["V"]
        dt = F32 if c["dtype"] == "f32" else BF16
        ld = (V + 63) // 64 * 64                         # rows of the vocabulary head are padded
        base = torch.randn(B, K + 1, V, generator=g, device=dev) * 2.5
        st["target"] = torch.zeros(B, K + 1, ld, dtype=dt, device=dev)[:, :, :V].copy_(base)
        tau = c["T"] if c["T"] > 0 else 1.0
        d = base[:, :K] + 0.7 * torch.randn(B, K, V, generator=g, device=dev)
        st["draft"] = torch.zeros(B, K, ld, dtype=dt, device=dev)[:, :, :V].copy_(d) if c["draft"] else None
        gumbel = -torch.log(-torch.log(torch.rand(B, K, V, generator=g, device=dev).clamp(1e-9, 1 - 1e-7)))
        st["tokens"] = (d / tau + (gumbel if c["draft"] else 0.0)).argmax(-1)
        st["u"] = torch.rand(B, K, generator=g, device=dev)
        st["r"] = torch.rand(B, generator=g, device=dev)
        st["n"] = torch.randint(max(1, K // 2), K + 1, (B,), generator=g, device=dev).to(torch.int32)
    else:
        R, V, k = c["R"], c["V"], min(c["k"], c["V"])
        dt = F32 if c["dtype"] == "f32" else BF16
        ld = (V + 255) // 256 * 256
        st["z"] = torch.zeros(R, ld, dtype=dt, device=dev)
        st["z"][:, :V] = torch.randn(R, V, generator=g, device=dev).mul_(1.5)
        st["tv"] = torch.sort(torch.randn(R, k, generator=g, device=dev) * 2.0 + 6.0, dim=1, descending=True)[0].contiguous()
        st["ti"] = ((torch.randint(0, V, (R, 1), generator=g, device=dev) + torch.arange(k, device=dev) * (V // k)) % V).to(torch.int32)
        st["w"] = (torch.rand(R, generator=g, device=dev) < 0.9).to(F32) / R
        st["y"] = torch.randint(0, V, (R,), generator=g, device=dev)
    return st


# --------------------------------------------------------------------------------------------------------------- one pass


def run(st):
    c = st["case"]
    return {"cache": _cache, "attn": _attn, "verify": _verify, "distill": _distill}[c["op"]](st, c)


def _cache(st, c):
    k, v = st["qkv"][:, :, 1], st["qkv"][:, :, 2]
    if own:
        from neko_amd import ops
        cache = ops.KV8Cache.from_tensors(st["k8"], st["v8"], st["ks"], st["vs"])
        ops.kv8_append(cache, k, v, st["pos"], n_new=st["n"])
        kr, vr = ops.kv8_read(cache, st["end"], c["top"])
        return {"k": kr, "v": vr, "k_scale": cache.k_scale, "v_scale": cache.v_scale}
    kr, ks = _append_plain(st, c, k, st["k8"], st["ks"])
    vr, vs = _append_plain(st, c, v, _v_to_rows(st["v8"].view(torch.uint8)).view(CODES[c["dtype"]]), st["vs"])
    return {"k": kr, "v": vr, "k_scale": ks, "v_scale": vs}


def _append_plain(st, c, rows, codes, scale):
    """Rows [S, T, H, hd] into codes [S, H, cap, hd]: what the cache then holds below `top`, and its scales."""
    S, T, H, hd = rows.shape
    cap, block, dt = codes.shape[2], c["block"], c["dtype"]
    t = torch.arange(cap, device=rows.device)
    pos, end = st["pos"].long()[:, None], st["end"].long()[:, None]
    new, old = (t >= pos) & (t < end), t < pos                                            # [S, cap]
    at = (t - pos).clamp(0, T - 1)
    x = torch.gather(rows.float(), 1, at[:, :, None, None].expand(S, cap, H, hd)).transpose(1, 2)
    x = torch.where(new[:, None, :, None], x, 0.0)
    amax = x.reshape(S, H, cap // block, block * hd).abs().amax(-1)
    kept = old[:, ::block][:, None, :]                                                    # the block holds older rows
    touched = new.view(S, cap // block, block).any(-1)[:, None, :]
    s1 = _scale_of(amax, dt)
    s1 = torch.where(kept, torch.maximum(scale, s1), s1)
    s1 = torch.where(touched, s1, scale)
    per_row = s1.repeat_interleave(block, 2).unsqueeze(-1)
    was = scale.repeat_interleave(block, 2).unsqueeze(-1)
    val = torch.where(new[:, None, :, None], x / per_row, codes.float() * (was / per_row))
    out = _round_codes(torch.where((new | old)[:, None, :, None], val, 0.0), dt).float() * per_row
    return out.transpose(1, 2)[:, :c["top"]].to(BF16).contiguous(), s1


def _attn(st, c):
    if own:
        from neko_amd import ops
        cache = ops.KV8Cache.from_tensors(st["k8"], st["v8"], st["ks"], st["vs"])
        return ops.attn_kv8(cache, st["q"], st["pos"], n_new=st["n"], start=st["start"], window=c["window"], sinks=c["sinks"], max_len=c["top"], out=st["out"])
    S, T, HG, hd = st["q"].shape
    H, G, L = c["H"], c["G"], c["top"]
    block = c["block"]
    k = (st["k8"].float() * st["ks"].repeat_interleave(block, 2).unsqueeze(-1))[:, :, :L]
    v = (_v_to_rows(st["v8"].view(torch.uint8)).view(CODES[c["dtype"]]).float() * st["vs"].repeat_interleave(block, 2).unsqueeze(-1))[:, :, :L]
    q = st["q"].float().view(S, T, H, G, hd).permute(0, 2, 3, 1, 4).reshape(S, H, G * T, hd)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(hd)).view(S, H, G, T, L)
    t = torch.arange(L, device=q.device)
    p = st["pos"].long()[:, None] + torch.arange(T, device=q.device)                      # [S, T]
    first = st["start"].long()[:, None, None]
    seen = (t <= p[:, :, None]) & (t >= first)
    if c["window"]:
        seen &= (t > p[:, :, None] - c["window"]) | (t < first + c["sinks"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    e = s.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    z = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(S, H, G * T, L), v).view(S, H, G, T, hd) / torch.where(z > 0, z, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(S, T, HG, hd).to(BF16)
    mine = torch.arange(T, device=q.device) < st["n"][:, None]                            # rows behind a sequence's last stay as they are
    return torch.where(mine[:, :, None, None], o, st["out"])


def _verify(st, c):
    if own:
        from neko_amd import ops
        n, tok = ops.verify_draft(st["target"], st["tokens"], draft_logits=st["draft"], u=st["u"], r=st["r"], n_draft=st["n"], temperature=c["T"])
        return {"accepted": n, "tokens": tok}
    B, K, V = c["B"], c["K"], c["V"]
    x = st["tokens"]
    i = torch.arange(K + 1, device=x.device)
    have = i[:K] < st["n"][:, None]
    if c["T"] == 0.0:
        best = st["target"].float().argmax(-1)                                            # [B, K + 1]
        ok = (best[:, :K] == x) & have
        n = ok.long().cumprod(1).sum(1)
        nxt = torch.gather(best, 1, n[:, None])[:, 0]
    else:
        # the CDF of 50 thousand tokens and its border in 64 bits
        p = torch.softmax(st["target"].double() / c["T"], -1)
        px = torch.gather(p[:, :K], 2, x[:, :, None])[:, :, 0]
        if st["draft"] is not None:
            q = torch.softmax(st["draft"].double() / c["T"], -1)
        else:
            q = torch.zeros(B, K, V, dtype=F64, device=x.device).scatter_(2, x[:, :, None], 1.0)
        qx = torch.gather(q, 2, x[:, :, None])[:, :, 0]
        ok = (st["u"].double() * qx < px) & have
        n = ok.long().cumprod(1).sum(1)
        row = n[:, None, None].expand(B, 1, V)
        pn = torch.gather(p, 1, row)[:, 0]
        qn = torch.gather(torch.cat([q, torch.zeros(B, 1, V, dtype=F64, device=x.device)], 1), 1, row)[:, 0]
        qn = torch.where((n < st["n"])[:, None], qn, 0.0)                                 # all accepted: the target's own row
        w = (pn - qn).clamp(min=0.0)
        w = torch.where(w.sum(-1, keepdim=True) > 0, w, pn)
        cum = w.cumsum(-1)
        nxt = (cum <= st["r"].double()[:, None] * cum[:, -1:]).sum(-1).clamp(max=V - 1)
    drafted = torch.cat([x, x[:, :1]], 1)
    tok = torch.where(i < n[:, None], drafted, torch.where(i == n[:, None], nxt[:, None], -1))
    return {"accepted": n.to(torch.int32), "tokens": tok}


def _distill(st, c):
    V, tau, a = c["V"], c["tau"], c["hard"]
    if own:
        from neko_amd import ops
        loss = torch.empty(st["z"].shape[0], dtype=F32, device=st["z"].device)
        dz = torch.empty_like(st["z"])
        ops.distill_topk(st["z"], V, st["z"].shape[1], st["tv"], st["ti"], st["w"], tau=tau, target=st["y"], hard=a, loss_row=loss, dlogits=dz)
        return {"loss": loss, "dz": dz}
    z, w = st["z"][:, :V].float(), st["w"]
    R = z.shape[0]
    ti = st["ti"].long()
    t = torch.softmax(st["tv"] / tau, -1)
    logs = torch.log_softmax(z / tau, -1)
    soft = (t * (torch.log(t) - torch.gather(logs, 1, ti))).sum(-1) * (tau * tau)
    d = torch.exp(logs).scatter_add_(1, ti, -t).mul_((1.0 - a) * tau)
    loss = (1.0 - a) * soft
    if a > 0.0:
        logp = torch.log_softmax(z, -1)
        loss = loss + a * -torch.gather(logp, 1, st["y"][:, None])[:, 0]
        d += a * torch.exp(logp).scatter_add_(1, st["y"][:, None], torch.full((R, 1), -1.0, device=z.device))
    dz = torch.zeros(R, st["z"].shape[1], dtype=st["z"].dtype, device=z.device)
    dz[:, :V] = d.mul_(w[:, None])
    return {"loss": torch.where(w > 0, loss, 0.0), "dz": dz}


# ------------------------------------------------------------------------------------------------------------------- work


def work(case):
    c = case
    if c["op"] == "cache":
        # rows are read in bf16 and written in 8 bits; the sequences are then read in 8 bits and written in bf16 (the longest for all of them:
        # the rows behind a shorter one's end are written as zeros); a scale per block
        rows = c["S"] * c["T"] * (0.5 if c["ragged"] and c["S"] > 1 else 1.0)
        back = c["S"] * c["top"]
        return {"bytes": 2 * c["H"] * c["hd"] * (rows * 3 + back * (1.0 * (0.7 if c["ragged"] and c["S"] > 1 else 1.0) + 2)), "flops": 0}
    if c["op"] == "attn":
        mean = 0.66 if c["ragged"] and c["S"] > 1 else 1.0
        rows = c["T"] * (0.5 if c["ragged"] and c["S"] > 1 and c["T"] > 1 else 1.0)
        keys = mean * c["top"] - 0.5 * rows
        if c["window"]:
            keys = min(keys, c["window"] + c["sinks"])
        held = min(mean * c["top"], keys + rows)
        Hq = c["H"] * c["G"]
        return {"bytes": 2 * c["S"] * c["H"] * held * c["hd"] + 4 * c["S"] * rows * Hq * c["hd"], "flops": 4 * c["S"] * Hq * rows * keys * c["hd"]}
    if c["op"] == "verify":
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["B"] * c["V"] * size * (c["K"] + 1 + (c["K"] if c["draft"] and c["T"] > 0 else 0)), "flops": 0}
    size = 4 if c["dtype"] == "f32" else 2
    return {"bytes": 2 * size * c["R"] * c["V"] + 8 * c["R"] * c["k"], "flops": 0}


# ------------------------------------------------------------------------------------------------------- the definition, 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    return {"cache": _cache_exact, "attn": _attn_exact, "verify": _verify_exact, "distill": _distill_exact}[case["op"]](st, case)


def _cache_exact(st, c):
    dt, block, top = c["dtype"], c["block"], c["top"]
    S, H, hd, cap = c["S"], c["H"], c["hd"], c["cap"]
    t = torch.arange(cap, device=st["pos"].device)
    out = {}
    for name, j, codes, scale in (("k", 1, st["k8"].double(), st["ks"]), ("v", 2, st["v8"].double().transpose(3, 4).reshape(S, H, cap, hd), st["vs"])):
        val = torch.zeros(S, H, cap, hd, dtype=F64, device=t.device)
        sc = scale.double().clone()
        for s in range(S):
            pos, n = int(st["pos"][s]), int(st["n"][s])
            b0, b1 = pos // block, (pos + n - 1) // block + 1
            lo, hi = b0 * block, b1 * block
            x = torch.zeros(H, hi - lo, hd, dtype=F64, device=t.device)
            x[:, pos - lo:pos - lo + n] = st["qkv"][s, :n, j].double().transpose(0, 1)
            e = torch.ceil(torch.log2(x.reshape(H, b1 - b0, -1).abs().amax(-1).clamp(min=2.0 ** -110) / QMAX[dt])).clamp(min=-100)
            if pos > lo:
                e[:, 0] = torch.maximum(e[:, 0], torch.log2(sc[s, :, b0]))
                x[:, :pos - lo] = codes[s, :, lo:pos] * sc[s, :, b0, None, None]
            val[s, :, :lo] = codes[s, :, :lo] * sc[s].repeat_interleave(block, 1)[:, :lo, None]
            sc[s, :, b0:b1] = torch.exp2(e)
            x /= sc[s, :, b0:b1].repeat_interleave(block, 1).unsqueeze(-1)
            grid = torch.ones_like(x) if dt == "int8" else torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0) - 3.0)
            x = torch.round(x / grid) * grid * sc[s, :, b0:b1].repeat_interleave(block, 1).unsqueeze(-1)
            val[s, :, lo:pos + n] = x[:, :pos + n - lo]
        out[name], out[name + "_scale"] = val.transpose(1, 2)[:, :top], sc
    return {k: out[k] for k in ("k", "v", "k_scale", "v_scale")}


def _attn_exact(st, c):
    S, T, HG, hd = st["q"].shape
    G = c["G"]
    out = st["out"].double()
    for s in range(S):
        n, pos, first = int(st["n"][s]), int(st["pos"][s]), int(st["start"][s])
        t = torch.arange(pos + n, device=out.device)
        p = pos + torch.arange(n, device=out.device)[:, None]
        hide = (t > p) | (t < first)
        if c["window"]:
            hide |= (t <= p - c["window"]) & (t >= first + c["sinks"])
        for h in range(c["H"]):
            per = torch.arange(pos + n, device=out.device) // c["block"]
            k = st["k8"][s, h, :pos + n].double() * st["ks"][s, h].double()[per][:, None]
            v = st["v8"][s, h].double().transpose(1, 2).reshape(-1, hd)[:pos + n] * st["vs"][s, h].double()[per][:, None]
            x = torch.einsum("tgd,ld->gtl", st["q"][s, :n, h * G:(h + 1) * G].double(), k) / hd ** 0.5
            w = torch.softmax(x.masked_fill(hide, -math.inf), -1)
            out[s, :n, h * G:(h + 1) * G] = torch.einsum("gtl,ld->tgd", torch.nan_to_num(w, nan=0.0), v)
    return out


def _verify_exact(st, c):
    B, K, V = c["B"], c["K"], c["V"]
    acc = torch.zeros(B, dtype=torch.int32, device=st["u"].device)
    tok = torch.full((B, K + 1), -1, dtype=torch.int64, device=st["u"].device)
    for b in range(B):
        n, nd = 0, int(st["n"][b])
        x = [int(v) for v in st["tokens"][b]]
        tok[b, :nd] = st["tokens"][b, :nd]
        residual = None
        while True:
            l = st["target"][b, n].double()
            if c["T"] == 0.0:
                p = l
                if n == nd or int(torch.argmax(l)) != x[n]:
                    break
            else:
                p = torch.exp((l - l.max()) / c["T"])
                p = p / p.sum()
                if n == nd:
                    break
                q = torch.zeros_like(p)
                if st["draft"] is None:
                    q[x[n]] = 1.0
                else:
                    d = st["draft"][b, n].double()
                    q = torch.exp((d - d.max()) / c["T"])
                    q = q / q.sum()
                if not float(st["u"][b, n]) * float(q[x[n]]) < float(p[x[n]]):
                    residual = torch.clamp(p - q, min=0.0)
                    break
            n += 1
        if c["T"] == 0.0:
            nxt = int(torch.argmax(p))
        else:
            w = p if residual is None or float(residual.sum()) <= 0 else residual
            cum = torch.cumsum(w, 0)
            nxt = min(V - 1, int((cum <= float(st["r"][b]) * cum[-1]).sum()))
        acc[b] = n
        tok[b, n] = nxt
        tok[b, n + 1:] = -1
    return {"accepted": acc, "tokens": tok}


def _distill_exact(st, c):
    V, tau, a = c["V"], c["tau"], c["hard"]
    R = c["R"]
    loss = torch.zeros(R, dtype=F64, device=st["z"].device)
    dz = torch.zeros(R, st["z"].shape[1], dtype=F64, device=st["z"].device)
    for r0 in range(0, R, 512):
        r = slice(r0, min(R, r0 + 512))
        z, w = st["z"][r, :V].double(), st["w"][r].double()
        tl = st["tv"][r].double() / tau
        t = torch.exp(tl - torch.logsumexp(tl, 1, keepdim=True))
        teacher = torch.zeros_like(z).scatter_add_(1, st["ti"][r].long(), t)
        lse_t, lse = torch.logsumexp(z / tau, 1, keepdim=True), torch.logsumexp(z, 1, keepdim=True)
        entropy = (t * (tl - torch.logsumexp(tl, 1, keepdim=True))).sum(1)
        soft = entropy - (teacher * (z / tau - lse_t)).sum(1)
        label = torch.zeros_like(z).scatter_(1, st["y"][r, None], 1.0)
        hard = lse[:, 0] - (z * label).sum(1)
        loss[r] = ((1.0 - a) * tau * tau * soft + a * hard) * (w > 0)
        dz[r, :V] = w[:, None] * ((1.0 - a) * tau * (torch.exp(z / tau - lse_t) - teacher) + a * (torch.exp(z - lse) - label))
    return {"loss": loss, "dz": dz}
