"""Tensor-level wrappers over the C ABI (one Python function per entry point of include/neko_hip.h).

PyTorch is only plumbing here: it owns device memory and the stream; every computation is a
libneko_hip.so kernel.  All functions enqueue on ``torch.cuda.current_stream()`` and return
immediately.  Shape/dtype preconditions are asserted before the call.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
from typing import Optional

import torch

from . import _lib

BF16 = torch.bfloat16
SAFE_TRANSPOSE = int(os.environ.get("NEKO_GEMM_SAFE_T", "0"))


def _p(t: Optional[torch.Tensor]):
    return None if t is None else C.c_void_p(t.data_ptr())


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    """hipStream_t of torch's current stream on the current device.  torch.cuda.current_stream() builds a Python
    Stream object through four layers of device-index helpers (~9 us, ~400 calls per step); the raw getter is one
    C call."""
    if _raw_stream is not None:
        return C.c_void_p(_raw_stream(torch._C._cuda_getDevice()))
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _chk(t: torch.Tensor, dtype, name: str):
    assert t.is_cuda, f"{name} must be a device tensor"
    assert t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}"


class Drop:
    """One dropout site: thr = round(p*256) (0 = off), key = 32-bit site key, scale = 256/(256-thr)."""
    __slots__ = ("thr", "key", "scale")

    def __init__(self, p: float, key: int):
        self.thr = max(0, min(255, int(round(p * 256))))
        self.key = key & 0xFFFFFFFF
        self.scale = 256.0 / (256 - self.thr)


def _drop(d):
    return (0, 0, 1.0) if (d is None or d.thr == 0) else (d.thr, d.key, d.scale)


def mix32(x: int) -> int:
    """Host-side 32-bit mixer (lowbias32) used to derive per-site dropout keys from (seed, step, site)."""
    x &= 0xFFFFFFFF
    x ^= x >> 16; x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x ^= x >> 15; x = (x * 0x846CA68B) & 0xFFFFFFFF
    x ^= x >> 16
    return x


def dropout_f32(x, drop, out=None):
    _chk(x, torch.float32, "x")
    x = x.contiguous()
    y = torch.empty_like(x) if out is None else out
    _lib.call("neko_dropout_f32", _p(x), _p(y), x.numel(), *_drop(drop), _stream())
    return y


def pick_splitk(M: int, N: int, K: int, target_blocks: int = 256) -> tuple:
    """Split-K factor for skinny-output / long-K GEMMs (weight gradients, LM-head dH).  Split-K launches run the
    256x256 tile, one block per CU (gemm_glds.hip: launch()), so the model is: rounds of `target_blocks` tiles,
    each k-step of 32 costing ~1.05 us per round, plus the fixed-order workspace reduce (write + read at ~4 TB/s).
    Returns (splitk, k_per_split) with k_per_split a multiple of 64 (of 128 when K is: every slice is then a whole number of
    trips of the long-contraction loop, gemm_a16.hip), or (1, 0)."""
    if K < 4096:
        return 1, 0
    tiles = ((M + 255) // 256) * ((N + 255) // 256)
    if tiles >= 4 * target_blocks:            # >= 4 rounds: the partial last round costs less than the reduce pass
        return 1, 0
    best_t, best = None, (1, 0)
    for sk in range(1, 33):
        q = 128 if K % 128 == 0 else 64
        kps = ((K + sk - 1) // sk + q - 1) // q * q
        if (K + kps - 1) // kps != sk:
            continue
        if sk > 1 and kps < 1024:
            break
        rounds = (tiles * sk + target_blocks - 1) // target_blocks
        t = rounds * kps * (1.05e-6 / 32)
        if sk > 1:
            t += 2.0 * sk * M * N * 4 / 4e12 + 4e-6
        if best_t is None or t < best_t * 0.97:          # prefer the smaller split on near-ties
            best_t, best = t, ((sk, kps) if sk > 1 else (1, 0))
    return best


def gemm(A: torch.Tensor, B: torch.Tensor, M: int, N: int, K: int, *, a_kstrided=False, b_kstrided=False,
         lda: Optional[int] = None, ldb: Optional[int] = None, alpha: float = 1.0,
         alpha_dev: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
         resid: Optional[torch.Tensor] = None, act: int = 0, act_in: Optional[torch.Tensor] = None,
         pre_out: Optional[torch.Tensor] = None, out_f32: Optional[torch.Tensor] = None, ldcf: Optional[int] = None,
         accumulate: bool = False, out_bf16: Optional[torch.Tensor] = None, ldcb: Optional[int] = None,
         splitk: int = 1, k_per_split: int = 0, safe_transpose: Optional[int] = None,
         deterministic_splitk: bool = True, drop=None) -> None:
    """C[M,N] = alpha * opA(A) @ opB(B) (+bias)(act)(+resid)(+C).  See neko_gemm_bf16 in include/neko_hip.h."""
    _chk(A, BF16, "A"); _chk(B, BF16, "B")
    if lda is None:
        lda = A.stride(0) if A.dim() == 2 else (M if a_kstrided else K)
    if ldb is None:
        ldb = B.stride(0) if B.dim() == 2 else (N if b_kstrided else K)
    if bias is not None:
        _chk(bias, torch.float32, "bias"); assert bias.numel() >= N
    ldr = 0
    if resid is not None:
        _chk(resid, torch.float32, "resid"); ldr = resid.stride(0) if resid.dim() == 2 else N
    ldact = ldpre = 0
    if act_in is not None:
        _chk(act_in, BF16, "act_in"); ldact = act_in.stride(0) if act_in.dim() == 2 else N
    if pre_out is not None:
        _chk(pre_out, BF16, "pre_out"); ldpre = pre_out.stride(0) if pre_out.dim() == 2 else N
    if out_f32 is not None:
        _chk(out_f32, torch.float32, "out_f32")
        if ldcf is None:
            ldcf = out_f32.stride(0) if out_f32.dim() == 2 else N
    if out_bf16 is not None:
        _chk(out_bf16, BF16, "out_bf16")
        if ldcb is None:
            ldcb = out_bf16.stride(0) if out_bf16.dim() == 2 else N
    if alpha_dev is not None:
        _chk(alpha_dev, torch.float32, "alpha_dev")
    st = SAFE_TRANSPOSE if safe_transpose is None else safe_transpose
    ws = None
    if splitk > 1 and deterministic_splitk and N % 4 == 0:
        ws = torch.empty(splitk * M * N, dtype=torch.float32, device=A.device)
    _lib.call("neko_gemm_bf16", _p(A), lda, int(a_kstrided), _p(B), ldb, int(b_kstrided), M, N, K, float(alpha),
              _p(alpha_dev), _p(bias), _p(resid), ldr, act, _p(act_in), ldact, _p(pre_out), ldpre, _p(out_f32),
              ldcf or 0, int(accumulate), _p(out_bf16), ldcb or 0, splitk, k_per_split, _p(ws), *_drop(drop), st, _stream())


def gemm_dgrad_gelu_colsum(dY: torch.Tensor, W: torch.Tensor, M: int, N: int, K: int, act_in: torch.Tensor,
                           out_bf16: torch.Tensor, colsum_out: torch.Tensor, ldb: Optional[int] = None,
                           act_in_is_factor: bool = False) -> None:
    """out_bf16[M,N] = (dY[M,K] @ W[N,K]^T) * gelu'(act_in); colsum_out[N] += its column sums (the c_fc bias gradient),
    one launch (+ a 10 us band reduction).  act_in_is_factor: act_in already holds gelu'(pre) (forward ran with act=3).
    See neko_gemm_dgrad_gelu_colsum in include/neko_hip.h."""
    _chk(dY, BF16, "dY"); _chk(W, BF16, "W"); _chk(act_in, BF16, "act_in"); _chk(out_bf16, BF16, "out_bf16")
    _chk(colsum_out, torch.float32, "colsum_out"); assert colsum_out.numel() >= N
    ws = torch.empty(int(_lib.load().neko_gemm_colsum_ws_floats(M, N)), dtype=torch.float32, device=dY.device)
    _lib.call("neko_gemm_dgrad_gelu_colsum", _p(dY), dY.stride(0) if dY.dim() == 2 else K, _p(W),
              ldb if ldb is not None else (W.stride(0) if W.dim() == 2 else K), M, N, K, _p(act_in),
              act_in.stride(0) if act_in.dim() == 2 else N, int(bool(act_in_is_factor)), _p(out_bf16),
              out_bf16.stride(0) if out_bf16.dim() == 2 else N, _p(ws), _p(colsum_out), _stream())


def layernorm_fwd(x, gamma, beta, y16=None, y32=None, mean=None, rstd=None, eps: float = 1e-5):
    _chk(x, torch.float32, "x")
    M, d = x.shape[0], x.shape[1]
    assert x.is_contiguous()
    _lib.call("neko_layernorm_fwd", _p(x), _p(gamma), _p(beta), _p(y16), _p(y32), _p(mean), _p(rstd), M, d,
              float(eps), _stream())


def layernorm_bwd(dy, x, gamma, mean, rstd, dgamma, dbeta, g_in=None, dx=None, dx16=None, accumulate=True, drop=None,
                  colsum16=None, row_map=None):
    """dy fp32 or bf16 [M,d] (neko_layernorm_bwd / neko_layernorm_bwd_bf16dy).  colsum16: fp32 [d] that receives (+=) the
    column sums of dx16 -- the bias gradient of the Linear that consumes dx16.  row_map (int32 [M]): dy is fp32 [n, d] and holds the
    gradient of row r at dy[row_map[r]], zero where row_map[r] < 0 (neko_layernorm_bwd_rows)."""
    assert dy.is_cuda and dy.dtype in (torch.float32, BF16) and dy.is_contiguous(), "dy must be a contiguous f32 / bf16 device tensor"
    M, d = x.shape[0], x.shape[1]
    nblk = _lib.load().neko_layernorm_bwd_blocks(M)
    ws = torch.empty(nblk * 3 * d, dtype=torch.float32, device=x.device)
    if colsum16 is not None:
        _chk(colsum16, torch.float32, "colsum16"); assert dx16 is not None and colsum16.numel() >= d
    if row_map is not None:
        _chk(dy, torch.float32, "dy"); _chk(row_map, torch.int32, "row_map")
        assert row_map.numel() == M and row_map.is_contiguous() and dy.shape[1] == d
        _lib.call("neko_layernorm_bwd_rows", _p(dy), _p(row_map), _p(x), _p(gamma), _p(mean), _p(rstd), _p(g_in), _p(dx), _p(dx16),
                  _p(dgamma), _p(dbeta), int(accumulate), _p(ws), M, d, *_drop(drop), _p(colsum16), _stream())
        return
    _lib.call("neko_layernorm_bwd_bf16dy" if dy.dtype == BF16 else "neko_layernorm_bwd", _p(dy), _p(x), _p(gamma), _p(mean), _p(rstd), _p(g_in), _p(dx), _p(dx16),
              _p(dgamma), _p(dbeta), int(accumulate), _p(ws), M, d, *_drop(drop), _p(colsum16), _stream())


def mask_bias(mask: torch.Tensor):
    """(B,T) 0/1 float mask -> additive key bias (B,T) f32 and first-real-key index (B,) int32."""
    _chk(mask, torch.float32, "mask")
    B, T = mask.shape
    mask = mask.contiguous()
    kb = torch.empty(B, T, dtype=torch.float32, device=mask.device)
    ks = torch.empty(B, dtype=torch.int32, device=mask.device)
    _lib.call("neko_mask_bias", _p(mask), _p(kb), _p(ks), B, T, _stream())
    return kb, ks


def gemm_set_mainloop(mode: int) -> int:
    """1 / 0: send every launch the hand-placed long-contraction main loop (gemm_a16.hip) can serve to it / none, -1: the
    built-in per-shape choice; returns the previous mode (neko_gemm_set_mainloop)."""
    return int(_lib.load().neko_gemm_set_mainloop(int(mode)))


MAINLOOP_NAMES = {0: "glds", 1: "a16", 2: "b16", 3: "glds64", 4: "bf16", 5: "p16", -1: "none"}


def gemm_last_mainloop() -> int:
    """Which main loop served this thread's last `gemm` launch (neko_gemm_last_mainloop; names: MAINLOOP_NAMES)."""
    return int(_lib.load().neko_gemm_last_mainloop())


def attn_set_path(mode: int) -> int:
    """0 = automatic (head-resident kernels when hd = 32 and T <= 1024; their backward in one pass for 256 < T <= 512, as two kernels
    otherwise), 1 = always the streaming kernels, 2 / 3 = head-resident with the two-kernel (bit-reproducible) / one-pass backward at
    every length; returns the previous mode (neko_attn_set_path)."""
    return int(_lib.load().neko_attn_set_path(int(mode)))


def attn_fwd(qkv, kbias, kstart, B, T, H, hd, drop=None, out=None, want_mask=False, mask_buf=None):
    """out (optional): a contiguous [B*T, H*hd] bf16 row range to write into (ragged groups share one buffer).
    want_mask: with dropout on, also return the keep-mask buffer the backward of this call can reuse (int32 tensor, or
    None when the schedule in use does not exchange masks): (out, lse, mask) instead of (out, lse).
    mask_buf (optional, tests): a caller-provided int32 buffer of neko_attn_mask_dwords elements to use as that mask buffer."""
    _chk(qkv, BF16, "qkv")
    assert qkv.is_contiguous() and qkv.shape[0] == B * T
    if out is None:
        out = torch.empty(B * T, H * hd, dtype=BF16, device=qkv.device)
    else:
        _chk(out, BF16, "out"); assert out.is_contiguous() and out.shape == (B * T, H * hd)
    lse = torch.empty(B, H, T, dtype=torch.float32, device=qkv.device)
    mask = None
    if want_mask and drop is not None and drop.thr > 0:
        n = int(_lib.load().neko_attn_mask_dwords(B, T, H, hd))
        if n > 0:
            if mask_buf is not None:
                _chk(mask_buf, torch.int32, "mask_buf"); assert mask_buf.numel() == n
            mask = mask_buf if mask_buf is not None else torch.empty(n, dtype=torch.int32, device=qkv.device)
    _lib.call("neko_attn_fwd", _p(qkv), _p(kbias), _p(kstart), _p(out), _p(lse), B, T, H, hd, *_drop(drop), _p(mask), _stream())
    return (out, lse, mask) if want_mask else (out, lse)


class VarlenGeom:
    """Packed sequences for the single-launch attention (neko_attn_*_varlen): lengths (host ints, in row order) -> row offsets,
    keep-mask offsets and sizes; the two offset arrays live on the device.

    Geometries are built once per (lengths, H, device) and kept (`VarlenGeom.get`): the two uploads go from PINNED host buffers
    that the object owns, so a training step that is being captured into a HIP graph either finds the device arrays ready or
    records copies whose source stays alive and constant for every replay -- never a copy from a temporary pageable tensor
    (that form stalls the host in eager mode and leaves a dangling host pointer in a captured graph)."""

    _cache: "dict" = {}
    _CACHE_MAX = 256          # unpinned entries
    _PINNED_WARN = 64         # warn once when captured steps hold this many
    _warned = False

    def __init__(self, lengths, H: int, device):
        self.lengths = [int(t) for t in lengths]
        self.nseq, self.Tmax, self.H = len(self.lengths), max(self.lengths), int(H)
        off, moff = [0], [0]
        for t in self.lengths:
            off.append(off[-1] + t)
            nb = (t + 31) // 32
            moff.append(moff[-1] + self.H * nb * nb * 32)
        self.rows, self.mask_dwords = off[-1], moff[-1]
        self.pinned_by_capture = False          # set on first use under stream capture; never cleared (the graph may be replayed any time)
        pin = torch.device(device).type == "cuda"
        self._host_off = torch.tensor(off, dtype=torch.int32)
        self._host_moff = torch.tensor(moff[:-1], dtype=torch.int64)
        if pin:
            self._host_off, self._host_moff = self._host_off.pin_memory(), self._host_moff.pin_memory()
        self.seq_off = self._host_off.to(device, non_blocking=True)
        self.mask_off = self._host_moff.to(device, non_blocking=True)

    @classmethod
    def get(cls, lengths, H: int, device) -> "VarlenGeom":
        key = (tuple(int(t) for t in lengths), int(H), str(device))
        g = cls._cache.get(key)
        if g is None:
            # only geometries that no captured graph points at count against the limit and are evicted (a HIP graph bakes
            # seq_off / mask_off and, when the geometry was built inside the capture, the pinned sources of their uploads into its nodes;
            # with every entry pinned nothing was evicted and the cache grew without a bound that anybody saw)
            free = [k for k, old in cls._cache.items() if not old.pinned_by_capture]
            if len(free) >= cls._CACHE_MAX:
                del cls._cache[free[0]]
            npinned = len(cls._cache) - len(free)
            if npinned >= cls._PINNED_WARN and not cls._warned:
                cls._warned = True
                import warnings
                warnings.warn(f"VarlenGeom: {npinned} packed-attention geometries are held by captured steps (each keeps pinned host "
                              "buffers and device tensors for the life of the process)")
            g = cls._cache[key] = cls(lengths, H, device)
        if not g.pinned_by_capture and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            g.pinned_by_capture = True           # used (or built) while a step is being captured: lives as long as the process
        return g


def attn_varlen_supported(Tmax: int, hd: int) -> bool:
    return bool(_lib.load().neko_attn_varlen_supported(int(Tmax), int(hd)))


def attn_fwd_varlen(qkv, kbias, kstart, geom: VarlenGeom, hd, drop=None, out=None, want_mask=False):
    """Packed counterpart of attn_fwd: qkv [rows, 3 H hd], kbias [rows], kstart [nseq] -> (out [rows, H hd], lse [rows * H]
    laid out [sequence][head][position], keep masks or None)."""
    _chk(qkv, BF16, "qkv")
    H = geom.H
    assert qkv.is_contiguous() and qkv.shape[0] >= geom.rows and kbias.numel() >= geom.rows
    if out is None:
        out = torch.empty(qkv.shape[0], H * hd, dtype=BF16, device=qkv.device)
    lse = torch.empty(geom.rows * H, dtype=torch.float32, device=qkv.device)
    mask = None
    if want_mask and drop is not None and drop.thr > 0 and hd == 32:      # only the head-resident kernels hand keep masks on
        mask = torch.empty(geom.mask_dwords, dtype=torch.int32, device=qkv.device)
    _lib.call("neko_attn_fwd_varlen", _p(qkv), _p(kbias), _p(kstart), _p(geom.seq_off), _p(geom.mask_off), _p(out), _p(lse),
              geom.nseq, geom.Tmax, H, hd, *_drop(drop), _p(mask), _stream())
    return out, lse, mask


class _DetAttnPath:
    """Under NEKO_DETERMINISTIC (SCATTER_DET) the head-resident attention backward of THIS thread runs as its two kernels at every length
    (neko_attn_bwd_reproducible, thread-local in the library: the process-wide schedule knob is not touched): the one-pass form adds dQ
    up block by block in arrival order, the two-kernel form is bit-reproducible."""

    def __enter__(self):
        self.prev = int(_lib.load().neko_attn_bwd_reproducible(1)) if SCATTER_DET else None
        return self

    def __exit__(self, *exc):
        if self.prev is not None:
            _lib.load().neko_attn_bwd_reproducible(self.prev)
        return False


def attn_bwd_varlen(qkv, out, dout, kbias, kstart, lse, geom: VarlenGeom, hd, drop=None, dqkv=None, mask=None):
    _chk(dout, BF16, "dout")
    H = geom.H
    D = torch.empty(geom.rows * H, dtype=torch.float32, device=qkv.device)
    if dqkv is None:
        dqkv = torch.empty_like(qkv)
    if mask is not None:
        _chk(mask, torch.int32, "mask"); assert mask.numel() == geom.mask_dwords
    with _DetAttnPath():
        _lib.call("neko_attn_bwd_varlen", _p(qkv), _p(out), _p(dout), _p(kbias), _p(kstart), _p(geom.seq_off), _p(geom.mask_off),
                  _p(lse), _p(D), _p(dqkv), geom.nseq, geom.rows, geom.Tmax, H, hd, *_drop(drop), _p(mask), _stream())
    return dqkv


def attn_bwd(qkv, out, dout, kbias, kstart, lse, B, T, H, hd, drop=None, dqkv=None, mask=None):
    """dqkv (optional): a contiguous [B*T, 3*H*hd] bf16 row range to write into.
    mask: the keep-mask buffer attn_fwd(..., want_mask=True) returned for the SAME call (or None: decisions are re-hashed)."""
    _chk(dout, BF16, "dout")
    dev = qkv.device
    assert qkv.is_contiguous() and out.is_contiguous() and dout.is_contiguous() and qkv.shape[0] == B * T
    D = torch.empty(B * H * T, dtype=torch.float32, device=dev)
    qflags = torch.empty(B * ((T + 63) // 64), dtype=torch.int32, device=dev)
    if dqkv is None:
        dqkv = torch.empty(B * T, 3 * H * hd, dtype=BF16, device=dev)
    else:
        _chk(dqkv, BF16, "dqkv"); assert dqkv.is_contiguous() and dqkv.shape == (B * T, 3 * H * hd)
    if mask is not None:
        _chk(mask, torch.int32, "mask")
        assert mask.numel() == int(_lib.load().neko_attn_mask_dwords(B, T, H, hd)), "mask buffer of another call / schedule"
    with _DetAttnPath():
        _lib.call("neko_attn_bwd", _p(qkv), _p(out), _p(dout), _p(kbias), _p(kstart), _p(lse), _p(D), _p(qflags),
                  _p(dqkv), B, T, H, hd, *_drop(drop), _p(mask), _stream())
    return dqkv


def gemv(x, W, M, N, K, *, b_kstrided, ldw=None, bias=None, resid=None, act=0, out_f32=None, out_bf16=None):
    """y[M<=8, N] = x[M,K] . W (+bias)(GELU)(+resid): weight-streaming product for the decode step (neko_gemv_bf16)."""
    _chk(x, BF16, "x"); _chk(W, BF16, "W")
    assert x.stride(-1) == 1 and (out_f32 is not None or out_bf16 is not None)
    _lib.call("neko_gemv_bf16", _p(x), x.stride(0) if x.dim() == 2 else K, _p(W), ldw if ldw is not None else W.stride(0),
              int(b_kstrided), M, N, K, _p(bias), _p(resid), resid.stride(0) if resid is not None else 0, int(act),
              _p(out_f32), out_f32.stride(0) if out_f32 is not None else 0,
              _p(out_bf16), out_bf16.stride(0) if out_bf16 is not None else 0, _stream())


def attn_decode(cache, row, pos, out, H, hd):
    """Newest row (index *pos, device int32) of one sequence against its [cap, 3d] q|k|v cache; see neko_attn_decode."""
    _chk(cache, BF16, "cache"); _chk(row, BF16, "row"); _chk(out, BF16, "out"); _chk(pos, torch.int32, "pos")
    assert cache.is_contiguous() and cache.shape[1] == 3 * H * hd and row.numel() == 3 * H * hd and out.numel() == H * hd
    _lib.call("neko_attn_decode", _p(cache), _p(row), _p(pos), _p(out), H, hd, cache.shape[0], _stream())


def ce_bf16_inplace(z, V, Vpad, target, weight, loss_row=None, want_grad=True):
    """z bf16 [R, >=Vpad]: logits in, weight * (softmax - onehot) out (in place); see neko_ce_bf16_inplace."""
    _chk(z, BF16, "z"); _chk(target, torch.int64, "target"); _chk(weight, torch.float32, "weight")
    assert z.stride(1) == 1
    _lib.call("neko_ce_bf16_inplace", _p(z), z.stride(0), V, Vpad, _p(target), _p(weight), _p(loss_row),
              int(bool(want_grad)), z.shape[0], _stream())


def ce_fwd_bwd(logits, V, Vpad, target, weight, loss_row=None, dlogits=None):
    _chk(logits, torch.float32, "logits"); _chk(target, torch.int64, "target"); _chk(weight, torch.float32, "weight")
    R = logits.shape[0]
    _lib.call("neko_ce_fwd_bwd", _p(logits), logits.stride(0), V, Vpad, _p(target), _p(weight), _p(loss_row),
              _p(dlogits), dlogits.stride(0) if dlogits is not None else 0, R, _stream())


def pack_embed_fwd(desc, cont_vals, disc_vals, img_emb, embed, pos_embed, sep, ntok, d, mu, M, n_bins, cont_start,
                   disc_start):
    _chk(desc, torch.int32, "desc")
    dev = embed.device
    x = torch.empty(ntok, d, dtype=torch.float32, device=dev)
    tokens = torch.empty(ntok, dtype=torch.int64, device=dev)
    tmask = torch.empty(ntok, dtype=torch.float32, device=dev)
    pmask = torch.empty(ntok, dtype=torch.float32, device=dev)
    _lib.call("neko_pack_embed_fwd", _p(desc), _p(cont_vals), _p(disc_vals), _p(img_emb), _p(embed), _p(pos_embed),
              _p(sep), _p(x), _p(tokens), _p(tmask), _p(pmask), ntok, d, float(mu), float(M), n_bins, cont_start,
              disc_start, _stream())
    return x, tokens, tmask, pmask


#: NEKO_DETERMINISTIC=1: the embedding-table gradients (token / position / separator embeddings, patch position tables) are summed in
#: sorted, fixed order (ABI v15, segsum.hip) instead of by fp32 atomics -- the only order-dependent sums of a step: with it a training run
#: is bit-reproducible (tools/trajectory_noise_probe.py: identical losses over repeated runs).  Costs 0.15 ms per m-mix step (two stable
#: sorts of 65536 keys + the ordered row sums, against 0.29 + 0.21 ms of contended atomics), hence off by default.
SCATTER_DET = os.environ.get("NEKO_DETERMINISTIC", "0") == "1"


#: The position-table / separator gradients of the packing backward and the patch-position table gradients as fixed-order segment sums
#: over HOST-sorted (key, row) pairs (neko_pack_embed_bwd_sorted / neko_patch_pos_add_bwd_sorted, ABI v17) instead of fp32 atomics on a
#: few dozen heavily contended rows; NEKO_SORTED_SCATTER=0 returns to the atomics.
SORTED_SCATTER = os.environ.get("NEKO_SORTED_SCATTER", "1") != "0"
SEGSUM_KEY_NONE = 0xFFFFF


def sorted_pairs(keys):
    """numpy int array of destination rows (negative: none) -> (keys_sorted, idx_sorted) int32, stable ascending, entries without a
    destination last with the key SEGSUM_KEY_NONE -- the input format of the *_sorted backward entry points."""
    import numpy as np
    k = np.where(keys < 0, SEGSUM_KEY_NONE, keys).astype(np.int32)
    order = np.argsort(k.astype(np.int16) if k.max(initial=0) < 32767 else k, kind="stable").astype(np.int32)
    return k[order], order


def pack_embed_bwd(desc, tokens, dx, d_embed, d_pos, d_sep, d_img, ntok, d, sorted_tail=False):
    """sorted_tail: `desc` holds, behind its ntok x 4 descriptors, ntok sorted keys and ntok row indices (sorted_pairs of the local
    position, or d_pos.shape[0] for a separator token): position / separator gradients then come from fixed-order segment sums."""
    _chk(dx, torch.float32, "dx")
    if sorted_tail and SORTED_SCATTER and not SCATTER_DET and d_pos.shape[0] < SEGSUM_KEY_NONE:
        assert desc.numel() >= 6 * ntok and desc.dtype == torch.int32 and desc.is_contiguous()
        n = int(_lib.load().neko_pack_embed_bwd_sorted_ws_bytes(ntok, d))
        ws = torch.empty(n, dtype=torch.uint8, device=dx.device)
        flat = desc.view(-1)
        _lib.call("neko_pack_embed_bwd_sorted", _p(desc), _p(tokens), _p(dx), _p(d_embed), _p(d_pos), _p(d_sep), _p(d_img), ntok, d,
                  int(d_pos.shape[0]), _p(flat[4 * ntok:]), _p(flat[5 * ntok:]), _p(ws), n, _stream())
        return
    if SCATTER_DET and d_embed.shape[0] < 0xFFFFF and d_pos.shape[0] < 0xFFFFF:
        n = int(_lib.load().neko_pack_embed_bwd_det_ws_bytes(ntok, d))
        ws = torch.empty(n, dtype=torch.uint8, device=dx.device)
        _lib.call("neko_pack_embed_bwd_det", _p(desc), _p(tokens), _p(dx), _p(d_embed), _p(d_pos), _p(d_sep), _p(d_img),
                  ntok, d, int(d_embed.shape[0]), int(d_pos.shape[0]), _p(ws), n, _stream())
        return
    _lib.call("neko_pack_embed_bwd", _p(desc), _p(tokens), _p(dx), _p(d_embed), _p(d_pos), _p(d_sep), _p(d_img),
              ntok, d, _stream())


def tokenize_continuous(x, use_mu_law, mu, M, n_bins, offset):
    _chk(x, torch.float32, "x")
    x = x.contiguous()
    ids = torch.empty(x.shape, dtype=torch.int32, device=x.device)
    _lib.call("neko_tokenize_continuous", _p(x), _p(ids), x.numel(), int(use_mu_law), float(mu), float(M), n_bins,
              offset if offset is not None else 0, _stream())
    return ids


def gather_rows_bf16(src, idx, n, npad):
    """dst[r] = src[idx[r]] for r < n, zero rows up to npad."""
    _chk(src, BF16, "src"); _chk(idx, torch.int32, "idx")
    d = src.shape[1]
    dst = torch.empty(npad, d, dtype=BF16, device=src.device)
    _lib.call("neko_gather_rows_bf16", _p(src), _p(idx), _p(dst), n, npad, d, _stream())
    return dst


def scatter_rows_f32(src, idx, n, dst):
    _chk(src, torch.float32, "src"); _chk(dst, torch.float32, "dst")
    _lib.call("neko_scatter_rows_f32", _p(src), _p(idx), _p(dst), n, src.shape[1], _stream())


def cast_f32_bf16(x, y):
    _chk(x, torch.float32, "x"); _chk(y, BF16, "y")
    _lib.call("neko_cast_f32_bf16", _p(x), _p(y), x.numel(), _stream())


def colsum_bf16(x, M, N, out, accumulate=True, ld=None):
    _chk(x, BF16, "x"); _chk(out, torch.float32, "out")
    _lib.call("neko_colsum_bf16", _p(x), ld if ld is not None else x.stride(0), M, N, _p(out), int(accumulate),
              _stream())


def geglu_fwd(h, gate):
    """h (= gelu(pre), bf16, contiguous) *= gate in place (neko_geglu_fwd; MLP.forward trajectory_gpt2.py:275-276)."""
    _chk(h, BF16, "h"); _chk(gate, BF16, "gate")
    assert h.is_contiguous() and gate.is_contiguous() and h.numel() == gate.numel()
    _lib.call("neko_geglu_fwd", _p(h), _p(gate), h.numel(), _stream())


def geglu_bwd(dh, pre, gate):
    """(d_pre, d_gate) = (dh * gate * gelu'(pre), dh * gelu(pre)), bf16 (neko_geglu_bwd)."""
    _chk(dh, BF16, "dh"); _chk(pre, BF16, "pre"); _chk(gate, BF16, "gate")
    assert dh.is_contiguous() and pre.is_contiguous() and gate.is_contiguous()
    d_pre, d_gate = torch.empty_like(dh), torch.empty_like(dh)
    _lib.call("neko_geglu_bwd", _p(dh), _p(pre), _p(gate), _p(d_pre), _p(d_gate), dh.numel(), _stream())
    return d_pre, d_gate


def sqnorm_f32(g, out_accum):
    _chk(g, torch.float32, "g"); _chk(out_accum, torch.float64, "out_accum")
    _lib.call("neko_sqnorm_f32", _p(g), g.numel(), _p(out_accum), _stream())


def adamw_step(p, g, m, v, p16, lr, beta1, beta2, eps, wd, gnorm_sq, max_norm, grad_scale, step, active, lr_dev=None):
    _lib.call("neko_adamw_step", _p(p), _p(g), _p(m), _p(v), _p(p16), p.numel(), float(lr), float(beta1),
              float(beta2), float(eps), float(wd), _p(gnorm_sq), float(max_norm), _p(grad_scale), _p(step),
              _p(active), _p(lr_dev), _stream())


_salt_holder = [None]


def set_drop_salt(salt: Optional[torch.Tensor]) -> None:
    """Register (or, with None, remove) the device uint32 every dropout site adds to its key (neko_set_drop_salt): the
    per-step variation of the masks inside a captured training step.  The tensor is kept alive here."""
    if salt is not None:
        assert salt.is_cuda and salt.dtype == torch.int32 and salt.numel() == 1
    _lib.call("neko_set_drop_salt", _p(salt))
    _salt_holder[0] = salt


#: the patch forward hands its GroupNorm statistics to the backward (neko_patch_resblock_fwd_stats / _bwd_stats, ABI v17) instead of
#: letting it recompute them; NEKO_PATCH_STATS=0 returns to the recomputing backward
PATCH_STATS = os.environ.get("NEKO_PATCH_STATS", "1") != "0"


def patch_resblock_fwd(images, w1, b1, gw, gb, w2, b2, mid, groups, want_x=True, want_padded=False, want_stats=False):
    """-> (y16 [P, 768] bf16, x_patches [P, 768] fp32 | None), plus with `want_padded` the zero-padded storage y16 is the row prefix of
    ([Ppad, 768], Ppad a multiple of 128): the weight gradient of the projection contracts over ITS rows; plus with `want_stats` the
    GroupNorm statistics [P, 64] fp32 (mean | rstd per group) for patch_resblock_bwd, or None when x_patches was not asked for."""
    assert images.is_cuda and images.dim() == 4 and images.shape[1] == 3
    assert images.dtype in (torch.float32, torch.uint8)
    images = images.contiguous()
    n, _, H, W = images.shape
    if H % 16 or W % 16:
        raise AssertionError("Image dimensions must be divisible by patch size")
    P = n * (H // 16) * (W // 16)
    # the patch rows are the CONTRACTION of the projection's weight gradient: storage padded with zero rows to a multiple of 128
    # keeps that product on the LDS-DMA GEMMs (a patch count such as 12289 sent it to the register-staged fallback: 237 us)
    Ppad = (P + 127) // 128 * 128
    y16_all = torch.empty(Ppad, 768, dtype=BF16, device=images.device)
    if Ppad > P:
        y16_all[P:].zero_()
    y16 = y16_all[:P]
    xp = torch.empty(P, 768, dtype=torch.float32, device=images.device) if want_x else None
    stats = torch.empty(P, 64, dtype=torch.float32, device=images.device) if (want_stats and want_x and PATCH_STATS) else None
    if stats is not None:
        _lib.call("neko_patch_resblock_fwd_stats", _p(images), int(images.dtype == torch.uint8), n, H, W, _p(w1), _p(b1),
                  _p(gw), _p(gb), _p(w2), _p(b2), mid, groups, _p(y16), _p(xp), _p(stats), _stream())
    else:
        _lib.call("neko_patch_resblock_fwd", _p(images), int(images.dtype == torch.uint8), n, H, W, _p(w1), _p(b1),
                  _p(gw), _p(gb), _p(w2), _p(b2), mid, groups, _p(y16), _p(xp), _stream())
    out = (y16, xp)
    if want_padded:
        out += (y16_all,)
    if want_stats:
        out += (stats,)
    return out


def patch_resblock_bwd(xp, dy, w1, b1, gw, gb, w2, b2, mid, groups, dw1, db1, dgw, dgb, dw2, db2, stats=None):
    _chk(dy, torch.float32, "dy")
    ws = torch.empty(_lib.load().neko_patch_resblock_bwd_ws_floats(xp.shape[0]), dtype=torch.float32, device=xp.device)
    if stats is not None:
        _chk(stats, torch.float32, "stats"); assert stats.shape == (xp.shape[0], 64) and stats.is_contiguous()
        _lib.call("neko_patch_resblock_bwd_stats", _p(xp), _p(stats), _p(dy), xp.shape[0], _p(w1), _p(b1), _p(gw), _p(gb), _p(w2), _p(b2),
                  mid, groups, _p(dw1), _p(db1), _p(dgw), _p(dgb), _p(dw2), _p(db2), _p(ws), _stream())
        return
    _lib.call("neko_patch_resblock_bwd", _p(xp), _p(dy), xp.shape[0], _p(w1), _p(b1), _p(gw), _p(gb), _p(w2), _p(b2),
              mid, groups, _p(dw1), _p(db1), _p(dgw), _p(dgb), _p(dw2), _p(db2), _p(ws), _stream())


def patch_pos_add(out, hpos, wpos, row_emb, col_emb):
    P, d = out.shape
    _lib.call("neko_patch_pos_add", _p(out), _p(hpos), _p(wpos), _p(row_emb), _p(col_emb), P, d, _stream())


def patch_pos_add_bwd(dout, hpos, wpos, d_row, d_col, sorted_rows=None):
    """sorted_rows: int32 [4, P] = (sorted hpos, their patch indices, sorted wpos, their patch indices) from sorted_pairs, or None"""
    P, d = dout.shape
    if sorted_rows is not None and SORTED_SCATTER and not SCATTER_DET and P > 0 and d_row.shape[0] < SEGSUM_KEY_NONE:
        assert sorted_rows.dtype == torch.int32 and sorted_rows.shape == (4, P) and sorted_rows.is_contiguous()
        n = int(_lib.load().neko_patch_pos_add_bwd_sorted_ws_bytes(P, d))
        ws = torch.empty(n, dtype=torch.uint8, device=dout.device)
        _lib.call("neko_patch_pos_add_bwd_sorted", _p(dout), _p(sorted_rows[0]), _p(sorted_rows[1]), _p(sorted_rows[2]), _p(sorted_rows[3]),
                  _p(d_row), _p(d_col), P, d, int(d_row.shape[0]), _p(ws), n, _stream())
        return
    if SCATTER_DET and P > 0:
        n = int(_lib.load().neko_patch_pos_add_bwd_det_ws_bytes(P, d))
        ws = torch.empty(n, dtype=torch.uint8, device=dout.device)
        _lib.call("neko_patch_pos_add_bwd_det", _p(dout), _p(hpos), _p(wpos), _p(d_row), _p(d_col), P, d, int(d_row.shape[0]),
                  _p(ws), n, _stream())
        return
    _lib.call("neko_patch_pos_add_bwd", _p(dout), _p(hpos), _p(wpos), _p(d_row), _p(d_col), P, d, _stream())


# ---- serving: 8-bit key / value cache, attention over it, verification of drafted tokens ---------------------------------------------
# A decode step is a few microseconds of kernel per call, so these wrappers keep their own cost down: one combined test per argument (the
# detailed message is worked out only when it fails), memoised workspace sizes (functions of the sizes alone), entry points bound once.
_KV8_DTYPES = {torch.float8_e4m3fn: 0, torch.int8: 1}
_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32
_MAX_COLS = 1 << 30                  # logits of a row (columns are 32-bit integers in the kernels, and sums of them with a workgroup's width)


def _here(t: torch.Tensor, name: str) -> int:
    """The launch goes to the current device's current stream: the tensor has to live there."""
    assert t.is_cuda, f"{name} must be a device tensor"
    dev = torch._C._cuda_getDevice()
    assert t.get_device() == dev, f"{name} is on {t.device}, the current device is cuda:{dev}"
    return dev


def _vec(t: Optional[torch.Tensor], n: int, name: str, dev: int, dtype=torch.int32):
    """Address of `n` contiguous values of `dtype` on device `dev` (None stays None)."""
    if t is None:
        return None
    if not (t.dtype is dtype and t.numel() == n and t.get_device() == dev and t.is_contiguous()):
        _here(t, name)
        assert t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}"
        raise AssertionError(f"{name} must hold {n} contiguous values, got {tuple(t.shape)}")
    return t.data_ptr()


def _raw(dev: int) -> int:
    return _raw_stream(dev) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    return getattr(_lib.load(), name)


@functools.lru_cache(maxsize=4096)
def _size(name: str, *sizes: int) -> int:
    return int(_entry(name)(*sizes))


class KV8Cache:
    """Keys and values of one layer in 8 bits: `nseq` sequences x `heads` key heads x `cap` positions (a multiple of 64) of `hd` channels.

    k [nseq, heads, cap, hd] and v [nseq, heads, cap / 16, hd, 16] (16 positions of one channel side by side) hold codes of `dtype`
    (torch.float8_e4m3fn or torch.int8), k_scale and v_scale [nseq, heads, cap / block] fp32 powers of two: value = code * scale, one scale
    per block of 16 / 32 / 64 positions and head.  The cache does not know how much of it is filled: positions are arguments of kv8_append,
    kv8_read and attn_kv8 (device tensors, so that a captured step can advance them)."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "nseq", "heads", "cap", "hd", "block", "dtype", "_args")

    def __init__(self, nseq: int, heads: int, cap: int, hd: int, dtype=torch.float8_e4m3fn, block: int = 32, device="cuda"):
        assert dtype in _KV8_DTYPES, f"cache dtype must be one of {list(_KV8_DTYPES)}, got {dtype}"
        assert nseq > 0 and heads > 0 and cap > 0 and cap % 64 == 0, "cap must be a positive multiple of 64"
        assert hd in (32, 64, 128) and block in (16, 32, 64), "hd must be 32 / 64 / 128, block 16 / 32 / 64"
        u8 = torch.zeros((2, nseq, heads, cap, hd), dtype=torch.uint8, device=device)
        sc = torch.ones((2, nseq, heads, cap // block), dtype=torch.float32, device=device)
        self._set(u8[0].view(dtype), u8[1].view(nseq, heads, cap // 16, hd, 16).view(dtype), sc[0], sc[1], nseq, heads, cap, hd, block)

    def _set(self, k, v, k_scale, v_scale, S, H, cap, hd, block):
        # the leading arguments of every entry point of the cache
        args = (k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), _KV8_DTYPES[k.dtype], S, H, cap, hd, block)
        for put, value in zip(_KV8_PUT, (k, v, k_scale, v_scale, S, H, cap, hd, block, k.dtype, args)):
            put(self, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"KV8Cache.{name} stays what it is (its address and sizes are checked once): copy into the tensor, or make another cache")

    def __reduce__(self):                 # copies and pickles: over their own tensors
        return KV8Cache.from_tensors, (self.k, self.v, self.k_scale, self.v_scale)

    @property
    def device(self) -> torch.device:
        return self.k.device

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale) -> "KV8Cache":
        """A cache over tensors that the caller holds (no copy): k, v, k_scale, v_scale as in the class description, contiguous."""
        dt, dev, sc = k.dtype, k.get_device(), k_scale.shape
        assert dt in _KV8_DTYPES and v.dtype is dt and k.dim() == 4 and len(sc) == 3, "k [nseq, heads, cap, hd] and v in e4m3 or int8"
        S, H, cap, hd = k.shape
        nb = sc[2]
        assert cap > 0 and cap % 64 == 0 and hd in (32, 64, 128), "cap must be a positive multiple of 64, hd 32 / 64 / 128"
        assert nb > 0 and cap % nb == 0 and cap // nb in (16, 32, 64), "one scale per 16 / 32 / 64 positions"
        assert v.shape == (S, H, cap // 16, hd, 16), f"v must be {(S, H, cap // 16, hd, 16)}, got {tuple(v.shape)}"
        assert sc == (S, H, nb) and v_scale.shape == sc, "scales must be [nseq, heads, cap / block]"
        assert k_scale.dtype is _F32 and v_scale.dtype is _F32, "scales must be float32"
        assert k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous(), "cache tensors must be contiguous"
        assert dev == v.get_device() == k_scale.get_device() == v_scale.get_device(), "cache tensors must be on one device"
        c = cls.__new__(cls)
        c._set(k, v, k_scale, v_scale, S, H, cap, hd, cap // nb)
        assert (c._args[0] | c._args[1]) % 16 == 0, "cache tensors must be 16-byte aligned"
        return c

    def row_strides(self, x: torch.Tensor, heads: int, name: str, dev: int):
        """(rows per sequence, sequence stride, row stride, address) of x [nseq, T, heads, hd] bf16 whose heads lie side by side (a view of a
        fused projection will do)."""
        if x.get_device() != dev or x.dtype is not BF16 or x.dim() != 4:
            _here(x, name)
            assert x.dtype == BF16, f"{name} must be {BF16}, got {x.dtype}"
        S, T, H, hd = x.shape if x.dim() == 4 else (-1, 0, 0, 0)
        assert S == self.nseq and H == heads and hd == self.hd and T > 0, f"{name} must be [{self.nseq}, T, {heads}, {self.hd}], got {tuple(x.shape)}"
        ss, st, sh, sc = x.stride()
        assert sc == 1 and (sh == hd or H == 1), f"{name}: the heads of a row must be contiguous"
        if T == 1:
            st = H * hd
        if S == 1:
            ss = T * st
        p = x.data_ptr()
        assert (st | ss) % 8 == 0 and p % 16 == 0, f"{name}: rows must be 16-byte aligned"
        return T, ss, st, p


_KV8_PUT = [getattr(KV8Cache, name).__set__ for name in KV8Cache.__slots__]       # (past __setattr__)


def kv8_append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, n_new: Optional[torch.Tensor] = None) -> None:
    """Quantise rows 0 .. n_new[s]-1 of k, v [nseq, T, heads, hd] (bf16) into positions pos[s] .. of every sequence; see neko_kv8_append."""
    dev = _here(cache.k, "cache")
    S = cache.nseq
    T, k_ss, k_st, kp = cache.row_strides(k, cache.heads, "k", dev)
    Tv, v_ss, v_st, vp = cache.row_strides(v, cache.heads, "v", dev)
    assert T == Tv, "k and v must have the same number of rows"
    rc = _entry("neko_kv8_append")(*cache._args, kp, k_ss, k_st, vp, v_ss, v_st, _vec(pos, S, "pos", dev), _vec(n_new, S, "n_new", dev), T, _raw(dev))
    if rc:
        _lib.check(rc, "neko_kv8_append")


def kv8_read(cache: KV8Cache, length: torch.Tensor, L: int):
    """Rows 0 .. L-1 of every sequence as bf16 -> (k, v) [nseq, L, heads, hd]; rows at and behind length[s] are 0; see neko_kv8_read."""
    assert 0 < L <= cache.cap, f"L must be in 1 .. {cache.cap}"
    dev = _here(cache.k, "cache")
    n = _vec(length, cache.nseq, "length", dev)
    k = torch.empty((cache.nseq, L, cache.heads, cache.hd), dtype=BF16, device=cache.device)
    v = torch.empty_like(k)
    rc = _entry("neko_kv8_read")(*cache._args, n, L, k.data_ptr(), v.data_ptr(), _raw(dev))
    if rc:
        _lib.check(rc, "neko_kv8_read")
    return k, v


def attn_kv8(cache: KV8Cache, q: torch.Tensor, pos: torch.Tensor, n_new: Optional[torch.Tensor] = None, start: Optional[torch.Tensor] = None,
             window: int = 0, sinks: int = 0, scale: Optional[float] = None, max_len: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of q [nseq, T, heads * G, hd] (bf16) at positions pos[s] + i over the cache (which holds those positions already: append
    first); causal, keys from start[s] on, optionally a sliding `window` with the first `sinks` keys kept visible.  Rows at and behind
    n_new[s] of `out` are left as they are (a fresh output holds zeros there).  max_len: host-known bound on pos + T, sizes the launch.  Up to
    64 rows a key head (T * G) the probabilities keep 16 bits, above 8.  See neko_attn_kv8."""
    dev = _here(cache.k, "cache")
    S, H, cap, hd = cache.nseq, cache.heads, cache.cap, cache.hd
    HG = q.shape[2] if q.dim() == 4 else 0
    assert HG > 0 and HG % H == 0, f"q must be [{S}, T, G * {H}, {hd}], got {tuple(q.shape)}"
    T, q_ss, q_st, qp = cache.row_strides(q, HG, "q", dev)
    assert T <= cap, "more rows than the cache has positions"
    assert window >= 0 and sinks >= 0 and (sinks == 0 or window > 0), "sinks need a window"
    assert scale is None or scale > 0.0, "scale must be positive"
    window, sinks, max_len = min(window, cap), min(sinks, cap), min(max_len, cap)       # no more than everything (and within 32 bits)
    if out is None:
        out = torch.zeros((S, T, HG, hd), dtype=BF16, device=cache.device)          # (positions outside the cache are no rows of the call either)
    To, o_ss, o_st, op = cache.row_strides(out, HG, "out", dev)
    assert To == T, "out must have q's rows"
    G = HG // H
    nws = _size("neko_attn_kv8_ws_floats", S, H, G, cap, hd, T, window, sinks, max_len)
    ws = torch.empty(nws, dtype=_F32, device=cache.device) if nws else None
    rc = _entry("neko_attn_kv8")(*cache._args, qp, q_ss, q_st, op, o_ss, o_st, G, T, _vec(pos, S, "pos", dev), _vec(n_new, S, "n_new", dev),
                                 _vec(start, S, "start", dev), window, sinks, scale if scale is not None else hd ** -0.5, max_len,
                                 ws.data_ptr() if nws else None, nws, _raw(dev))
    if rc:
        _lib.check(rc, "neko_attn_kv8")
    return out


def _logit_rows(x: torch.Tensor, shape, name: str, dev: int):
    if x.get_device() != dev or x.dim() != 3:
        _here(x, name)
    assert x.dtype is _F32 or x.dtype is BF16, f"{name} must be float32 or bfloat16, got {x.dtype}"
    assert x.shape == shape, f"{name} must be {list(shape)}, got {list(x.shape)}"
    sb, sr, sc = x.stride()
    assert sc == 1 or shape[2] == 1, f"{name}: a row's logits must be contiguous"
    return x.data_ptr(), sb, sr


def verify_draft(logits: torch.Tensor, tokens: torch.Tensor, draft_logits: Optional[torch.Tensor] = None, u: Optional[torch.Tensor] = None,
                 r: Optional[torch.Tensor] = None, n_draft: Optional[torch.Tensor] = None, temperature: float = 1.0):
    """Which drafted `tokens` [B, K] (int64) the target's `logits` [B, K + 1, V] keep, given uniform numbers u [B, K] and r [B], and the token
    behind them -> (accepted [B] int32, out_tokens [B, K + 1] int64, -1 behind the last).  draft_logits [B, K, V]: what the drafts were
    sampled from at the same temperature (None: the draft was certain of its tokens).  temperature 0: greedy, u and r unused.  See
    neko_verify_draft."""
    assert tokens.dim() == 2, "tokens must be [B, K]"
    B, K = tokens.shape
    assert B > 0 and 0 < K <= 62, "1 to 62 drafted tokens"
    V = logits.shape[-1]
    assert 0 < V <= _MAX_COLS, f"1 to {_MAX_COLS} logits a row"
    assert temperature >= 0.0, "temperature must not be negative"
    dev = _here(logits, "logits")
    tp, t_sb, t_sr = _logit_rows(logits, (B, K + 1, V), "logits", dev)
    dp, d_sb, d_sr = None, 0, 0
    if temperature > 0:
        assert u is not None and r is not None, "sampling needs u [B, K] and r [B]"
        if draft_logits is not None:
            dp, d_sb, d_sr = _logit_rows(draft_logits, (B, K, V), "draft_logits", dev)
            assert draft_logits.dtype is logits.dtype, "logits and draft_logits must have one type"
    else:
        u = r = None
    where = logits.device
    accepted = torch.empty(B, dtype=_I32, device=where)
    out = torch.empty((B, K + 1), dtype=_I64, device=where)
    nws = _size("neko_verify_draft_ws_bytes", B, K, V)
    ws = torch.empty(nws, dtype=torch.uint8, device=where)
    rc = _entry("neko_verify_draft")(tp, t_sb, t_sr, dp, d_sb, d_sr, logits.dtype is BF16, B, K, V, _vec(tokens, B * K, "tokens", dev, _I64),
                                     _vec(u, B * K, "u", dev, _F32), _vec(r, B, "r", dev, _F32), _vec(n_draft, B, "n_draft", dev), temperature,
                                     accepted.data_ptr(), out.data_ptr(), ws.data_ptr(), nws, _raw(dev))
    if rc:
        _lib.check(rc, "neko_verify_draft")
    return accepted, out


# ---- distillation ---------------------------------------------------------------------------------------------------------------------
def distill_topk(z: torch.Tensor, V: int, Vpad: int, t_val: Optional[torch.Tensor], t_idx: Optional[torch.Tensor], weight: torch.Tensor,
                 tau: float = 1.0, target: Optional[torch.Tensor] = None, hard: float = 0.0, loss_row: Optional[torch.Tensor] = None,
                 dlogits: Optional[torch.Tensor] = None) -> None:
    """Rows of student logits z [R, >= Vpad] (bf16 or fp32, columns < V valid) against a teacher's top logits t_val [R, k] fp32 at t_idx [R, k]
    int32: loss_row [R] fp32 = (1 - hard) tau^2 KL + hard CE(target), dlogits (z's type, may be z) = weight * gradient; see neko_distill_topk."""
    dev = _here(z, "z")
    assert z.dtype is _F32 or z.dtype is BF16, f"z must be float32 or bfloat16, got {z.dtype}"
    assert z.dim() == 2 and z.shape[1] >= Vpad >= V > 0 and z.stride(1) == 1, "z must be [R, >= Vpad] with contiguous rows"
    R = z.shape[0]
    assert Vpad <= _MAX_COLS and R < 2 ** 31, f"at most {_MAX_COLS} columns and 2^31 - 1 rows"
    assert R > 0 and tau > 0.0 and 0.0 <= hard <= 1.0, "tau must be positive, hard in [0, 1]"
    assert loss_row is not None or dlogits is not None, "nothing to compute"
    k, tv, ti = 0, None, None
    if hard < 1.0:
        assert t_val is not None and t_idx is not None and t_val.dim() == 2 and t_val.shape == t_idx.shape, "t_val and t_idx must be [R, k]"
        k = t_val.shape[1]
        assert 0 < k <= 1024, "1 to 1024 teacher entries"
        tv, ti = _vec(t_val, R * k, "t_val", dev, _F32), _vec(t_idx, R * k, "t_idx", dev)
    assert hard == 0.0 or target is not None, "hard > 0 needs target"
    ldz, ldd, dp = (z.stride(0) if R > 1 else Vpad), 0, None        # (a single row has no stride)
    if dlogits is not None:
        if dlogits.get_device() != dev or dlogits.dtype is not z.dtype:
            _here(dlogits, "dlogits")
        assert dlogits.dtype is z.dtype and dlogits.dim() == 2 and dlogits.shape[0] == R and dlogits.shape[1] >= Vpad and dlogits.stride(1) == 1, \
            "dlogits must be like z"
        ldd, dp = (dlogits.stride(0) if R > 1 else Vpad), dlogits.data_ptr()
    rc = _entry("neko_distill_topk")(z.data_ptr(), ldz, z.dtype is BF16, R, V, Vpad, tv, ti, k, _vec(weight, R, "weight", dev, _F32), tau,
                                     _vec(target, R, "target", dev, _I64), hard, _vec(loss_row, R, "loss_row", dev, _F32), dp, ldd, _raw(dev))
    if rc:
        _lib.check(rc, "neko_distill_topk")
