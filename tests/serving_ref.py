"""Plain 64-bit restatements of the serving and distillation operators (tests only)."""
import math

import torch

F64 = torch.float64
QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def pow2_scale(amax, dtype):
    """Smallest power of two s with amax <= qmax s, at least 2^-100."""
    if amax == 0:
        return 2.0 ** -100
    e = math.ceil(math.log2(amax / QMAX[dtype]) - 1e-12)
    while amax > QMAX[dtype] * 2.0 ** e:
        e += 1
    while e > -100 and amax <= QMAX[dtype] * 2.0 ** (e - 1):
        e -= 1
    return 2.0 ** max(e, -100)


def round_codes(x, dtype):
    """Nearest-even rounding to the 8-bit grid, as fp64 code values."""
    if dtype == torch.int8:
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0) - 3.0)
    return torch.round(x / step) * step


class RefCache:
    """values: fp64 codes k, v [S, H, cap, hd] and scales [S, H, cap / block] (row layout for both)."""

    def __init__(self, S, H, cap, hd, dtype, block):
        self.S, self.H, self.cap, self.hd, self.dtype, self.block = S, H, cap, hd, dtype, block
        self.codes = [torch.zeros(S, H, cap, hd, dtype=F64) for _ in range(2)]
        self.scale = [torch.ones(S, H, cap // block, dtype=F64) for _ in range(2)]

    def append(self, k, v, pos, n_new):
        """k, v [S, T, H, hd] cpu tensors; pos, n_new lists."""
        for j, x in enumerate((k, v)):
            x = x.to(F64)
            x = torch.nan_to_num(x, nan=0.0, posinf=1e300, neginf=-1e300).clamp(-1.75 * 2.0 ** 127, 1.75 * 2.0 ** 127)
            for s in range(self.S):
                p, n = pos[s], min(n_new[s], x.shape[1])
                if p < 0 or p >= self.cap or n <= 0:
                    continue
                n = min(n, self.cap - p)
                for h in range(self.H):
                    for b in range(p // self.block, (p + n - 1) // self.block + 1):
                        lo, hi = max(p, b * self.block), min(p + n, (b + 1) * self.block)
                        rows = x[s, lo - p:hi - p, h]
                        sc = pow2_scale(float(rows.abs().max()), self.dtype)
                        if b * self.block < p:
                            old = float(self.scale[j][s, h, b])
                            if sc > old:
                                o = self.codes[j][s, h, b * self.block:p]
                                o.copy_(round_codes(o * (old / sc), self.dtype))
                            sc = max(sc, old)
                        self.scale[j][s, h, b] = sc
                        self.codes[j][s, h, lo:hi] = round_codes(rows / sc, self.dtype)

    def values(self, j):
        return self.codes[j] * self.scale[j].repeat_interleave(self.block, 2).unsqueeze(-1)

    def read(self, length, L):
        out = []
        for j in range(2):
            x = self.values(j)[:, :, :L].transpose(1, 2).clone()
            for s in range(self.S):
                x[s, max(0, length[s]):] = 0
            out.append(x)
        return out


def attention(q, k, v, pos, n_new, start, window, sinks, scale, out):
    """q [S, T, Hq, hd], k / v fp64 [S, H, cap, hd] -> (out with the rows of the call replaced, bound-weights): the second value is
    sum_t p_t |v_t| per output element and the third max_t sum_c |q_c k_tc| scale per row, for tolerances."""
    S, T, HQ, hd = q.shape
    H, cap = k.shape[1], k.shape[2]
    G = HQ // H
    out = out.to(F64).clone()
    absv = torch.zeros_like(out)
    big = torch.zeros(S, T, HQ, 1, dtype=F64)
    for s in range(S):
        if pos[s] < 0 or pos[s] >= cap:
            continue
        for i in range(min(n_new[s], T, cap - pos[s])):
            p = pos[s] + i
            t = torch.arange(cap)
            seen = (t <= p) & (t >= start[s])
            if window:
                seen &= (t > p - window) | (t < start[s] + sinks)
            t = t[seen]
            for hq in range(HQ):
                if len(t) == 0:
                    out[s, i, hq] = 0
                    continue
                kk, vv = k[s, hq // G, t], v[s, hq // G, t]
                qq = q[s, i, hq].to(F64)
                w = torch.softmax(kk @ qq * scale, 0)
                out[s, i, hq] = w @ vv
                absv[s, i, hq] = w @ vv.abs()
                big[s, i, hq] = (kk.abs() @ qq.abs()).max() * scale
    return out, absv, big


def verify(target, tokens, draft, u, r, n_draft, temperature):
    """Lists / cpu tensors in, (accepted list, tokens [B][K+1])."""
    B, K = tokens.shape
    acc, out = [], []
    for b in range(B):
        n = min(max(int(n_draft[b]), 0), K)
        x = [int(t) for t in tokens[b]]

        def dist(l):
            l = torch.where(l.isnan(), torch.full_like(l, -math.inf), l).to(F64)
            m = l.max()
            if m == -math.inf:
                return None
            e = torch.where(l == m, torch.ones_like(l), torch.exp((l - m) / temperature))
            return e / e.sum()
        kept, nxt = 0, None
        V = target.shape[-1]
        while True:
            l = target[b, kept]
            if temperature == 0:
                l = torch.where(l.isnan(), torch.full_like(l, -math.inf), l)
                best = int((l == l.max()).nonzero()[0]) if l.max() > -math.inf else -1
                if kept < n and best >= 0 and best == x[kept]:
                    kept += 1
                    continue
                nxt = best
                break
            p = dist(l)
            if kept == n:
                w = p
                break
            q = None
            if draft is not None:
                q = dist(draft[b, kept])
            else:
                q = torch.zeros(V, dtype=F64)
                if 0 <= x[kept] < V:
                    q[x[kept]] = 1
            inside = 0 <= x[kept] < V
            if p is not None and inside and q is not None and float(u[b, kept]) * float(q[x[kept]]) < float(p[x[kept]]):
                kept += 1
                continue
            w = p if p is None else (p if q is None else (p - q).clamp(min=0))
            if w is not None and float(w.sum()) <= 0:
                w = p
            break
        if temperature != 0:
            if w is None:
                nxt = -1
            else:
                c = w.cumsum(0)
                hit = (c > float(r[b]) * float(c[-1])).nonzero()
                nxt = int(hit[0]) if len(hit) else int((w > 0).nonzero()[-1])
        acc.append(kept)
        out.append(x[:kept] + [nxt] + [-1] * (K - kept))
    return acc, out


def distill(z, V, t_val, t_idx, weight, tau, target, hard):
    """fp64 -> (loss_row, gradient [R, V], scale of the gradient's terms [R, V])."""
    z = z[:, :V].to(F64)
    R = z.shape[0]
    loss, g, mag = torch.zeros(R, dtype=F64), torch.zeros(R, V, dtype=F64), torch.zeros(R, V, dtype=F64)
    for r in range(R):
        w = float(weight[r])
        if w == 0:
            continue
        if hard < 1:
            ok = [(int(i), float(t)) for i, t in zip(t_idx[r], t_val[r]) if 0 <= int(i) < V and float(t) > -math.inf]
            if ok:
                t = torch.softmax(torch.tensor([v for _, v in ok], dtype=F64) / tau, 0)
                ls = torch.log_softmax(z[r] / tau, 0)
                ids = torch.tensor([i for i, _ in ok])
                loss[r] += (1 - hard) * tau * tau * float((t * (torch.log(t) - ls[ids])).sum())
                dense = torch.zeros(V, dtype=F64).index_add_(0, ids, t)
                g[r] += w * (1 - hard) * tau * (ls.exp() - dense)
                mag[r] += abs(w) * (1 - hard) * tau * (ls.exp() + dense)
        if hard > 0 and target is not None and 0 <= int(target[r]) < V:
            lp = torch.log_softmax(z[r], 0)
            y = int(target[r])
            loss[r] += -hard * float(lp[y])
            one = torch.zeros(V, dtype=F64)
            one[y] = 1
            g[r] += w * hard * (lp.exp() - one)
            mag[r] += abs(w) * hard * (lp.exp() + one)
    return loss, g, mag
