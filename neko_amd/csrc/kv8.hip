// The 8-bit key / value cache: rows are quantised as they are written, and read back as bf16 (layout: kv8.h).
//
// append: rows [S, T, H, hd] bf16 go to positions pos[s] .. pos[s] + n[s] - 1.  For every block of `block` positions the rows touch:
//     e     = smallest exponent with max |new row value| <= qmax 2^e  (at least -100)
//     scale = 2^e, or the block's present scale where that is larger and the block holds older rows (positions < pos[s])
//     code  = round-to-nearest-even(x / scale)
// and where a block's scale grows, its older codes are rounded again to the new grid (a power of two: exact for e4m3 except below its
// smallest normal; int8 loses one bit per doubling, at most one step of the final grid in sum).  NaN is stored as 0, and what is larger than
// 1.75 2^127 (infinities among it) as that, the largest value that both code types give back finite: a cache written here holds no code
// that could spread beyond its own position.
//
// Both kernels are bound by HBM: append reads 2 B and writes 1 B a value, the read back 1 B and 2 B.  A lane owns 16 positions x 8
// channels: 16 row loads of 16 B in flight before the first is looked at, and the block's maximum meets in registers (shuffles inside the
// wave).  Consecutive units of a wave are consecutive heads: their row pieces are adjacent in the bf16 rows.  On the 8-bit side a head's
// bytes are contiguous instead, so the codes change hands through LDS: written and read there in the lane's own order, moved to and from
// memory as consecutive 16-byte pieces (as 8-byte rows and 16-byte pieces 128 B apart they were 3 x the requests).  A piece belongs to
// one lane: a partly filled one is read, changed and written by its owner.
// 64 sequences of up to 1024 rows x 24 heads of 32, K and V: append 42-53 us (151 MB: 2.8-3.6 TB/s), read back 45 us (272 MB: 6.0 TB/s, codes partly
// out of the last-level cache; a copy reaches 5.2).  What keeps the append from the copy's rate are its registers: sixteen rows in flight and their
// codes take 154-156 (int8 141-142), three waves per SIMD, where the read back has 52-60.  (Units that begin or end inside a block, and are read,
// changed and written, are a few in a hundred there: two at most for a sequence and head.)
#include "kv8.h"

namespace {

struct AppendArgs {
  uint8_t *k8, *v8;
  float *ks, *vs;
  const bf16_t *k, *v;
  long k_ss, k_st, v_ss, v_st;      // element strides: sequence, row
  const int *pos, *n_new;
  int S, H, cap, T, bshift, nslots;
  long units;
};

constexpr uint32_t TOP = 0x7f60u;         // bf16 bits of 1.75 2^127

// NaN -> 0, magnitudes above TOP -> TOP (two bf16 in a dword)
__device__ __forceinline__ uint32_t tame2(uint32_t w) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t x = (w >> (16 * i)) & 0xffffu;
    const uint32_t a = x & 0x7fffu;
    if (a > 0x7f80u) x = 0;
    else if (a > TOP) x = (x & 0x8000u) | TOP;
    r |= x << (16 * i);
  }
  return r;
}
__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
__device__ __forceinline__ uint32_t pkmax_u16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// bf16 bits of the largest magnitude -> the scale: am = (1 + m / 128) 2^(x - 127); qmax = 1.75 * 2^8 | (1 + 126 / 128) * 2^6
template <int DT>
__device__ __forceinline__ float scale_of(uint32_t am) {
  const int x = (int)(am >> 7), m = (int)(am & 0x7f);
  int e = DT == 0 ? x - 127 - 8 + (m > 96) : x - 127 - 6 + (m > 126);
  if (x == 0 || e < -100) e = -100;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// a unit (one block of one head, K or V) on its way out: where it goes, its first position, the new positions [pc, end) (end < 0: nothing),
// and the factor of its older codes if their grid grew (negative: it did not; 0 is a factor, where the grids lie further apart than fp32 reaches)
struct UnitOut { long base; int b0, pc, end; float ratio; };

template <int HD, int BLOCK, int DT>
__global__ __launch_bounds__(256) void kv8_append_kernel(AppendArgs a) {
  constexpr int C = HD / 8, R = BLOCK / 16, U = 64 / (C * R);      // channel lanes, tile lanes, units per wave
  constexpr int UB = BLOCK * HD, US = UB + 32;                      // bytes of a unit, and its stride in the image (8 units: all banks)
  __shared__ __attribute__((aligned(16))) char img[4][U * US];
  __shared__ UnitOut outs[4][U];
  const bool is_v = blockIdx.y != 0;
  const int lane = threadIdx.x & 63;
  const int c = lane % C, ui = (lane / C) % U, r = lane / (C * U);
  const long wave = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const long u = wave * U + ui;
  bool act = u < a.units;
  const long uu = act ? u : 0;
  const int h = (int)(uu % a.H);
  const long sj = uu / a.H;
  const int s = (int)(sj / a.nslots), j = (int)(sj % a.nslots);
  const int p = a.pos[s];
  int n = a.n_new ? a.n_new[s] : a.T;
  n = min(n, a.T);
  if (p < 0 || p >= a.cap || n <= 0) { act = false; n = 1; }
  const int pc = min(max(p, 0), a.cap - 1);
  n = min(n, a.cap - pc);
  const int blk = (pc >> a.bshift) + j;
  const int end = pc + n;
  const int b0 = blk << a.bshift;
  act = act && b0 < end;
  const int t0 = b0 + r * 16;                                       // this lane's 16 positions
  const bool any_new = act && t0 < end && t0 + 16 > pc;

  const bf16_t* src = (is_v ? a.v : a.k) + (is_v ? a.v_ss : a.k_ss) * s + (long)h * HD + c * 8;
  const long st = is_v ? a.v_st : a.k_st;
  uint4 raw[16];
  uint32_t mx = 0;
  if (any_new) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {                                  // clamped, unconditional: all sixteen in flight
      const int row = min(max(t0 + i - pc, 0), n - 1);
      raw[i] = *reinterpret_cast<const uint4*>(src + row * st);
    }
    // a clamped row repeats a row of the same call, of this block (both ends of the tile's new range lie in it): its maximum counts anyway
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      mx = pkmax_u16(mx, pkmax_u16(pkmax_u16(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu), pkmax_u16(raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu)));
    }
    if ((mx & 0xffffu) > TOP || (mx >> 16) > TOP) {                 // rare: NaN or an infinity among them
      mx = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        raw[i].x = tame2(raw[i].x); raw[i].y = tame2(raw[i].y); raw[i].z = tame2(raw[i].z); raw[i].w = tame2(raw[i].w);
        mx = pkmax_u16(mx, pkmax_u16(pkmax_u16(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu), pkmax_u16(raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu)));
      }
    }
  }
  uint32_t am = max(mx & 0xffffu, mx >> 16);
#pragma unroll
  for (int o = 1; o < C; o <<= 1) am = max(am, (uint32_t)__shfl_xor((int)am, o, 64));
#pragma unroll
  for (int o = C * U; o < 64; o <<= 1) am = max(am, (uint32_t)__shfl_xor((int)am, o, 64));
  float scale = scale_of<DT>(am);
  const long head = (long)s * a.H + h;
  float* sp = (is_v ? a.vs : a.ks) + head * (a.cap >> a.bshift) + blk;
  const bool held = act && b0 < pc;                                 // the block holds older rows
  const float was = held ? *sp : scale;
  scale = fmaxf(scale, was);
  const bool grew = held && scale > was;
  const float inv = 1.0f / scale;
  if (c == 0 && r == 0) {                 // (every lane of the unit is in this wave and has read the old scale: the loads stand before the store)
    if (act) *sp = scale;
    UnitOut& o = outs[threadIdx.x >> 6][ui];
    o.base = (head * a.cap + b0) * HD;    // K and V alike: a block's bytes are contiguous in both layouts
    o.b0 = b0;
    o.pc = pc;
    o.end = act ? end : -1;
    o.ratio = grew ? was * inv : -1.f;
  }
  // codes -> the wave's image of its units, as they will lie in memory (bytes of positions that are not new: whatever they are, dropped below)
  char* mine = img[threadIdx.x >> 6];
  if (any_new) {
    char* at = mine + ui * US + r * (16 * HD);
    if (!is_v) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        uint2 w;
        w.x = kv8_pack4<DT>(lo_f(raw[i].x) * inv, hi_f(raw[i].x) * inv, lo_f(raw[i].y) * inv, hi_f(raw[i].y) * inv);
        w.y = kv8_pack4<DT>(lo_f(raw[i].z) * inv, hi_f(raw[i].z) * inv, lo_f(raw[i].w) * inv, hi_f(raw[i].w) * inv);
        *reinterpret_cast<uint2*>(at + i * HD + c * 8) = w;
      }
    } else {
#pragma unroll
      for (int ch = 0; ch < 8; ++ch) {
        uint32_t q[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          float f[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4& w4 = raw[d * 4 + i];
            const uint32_t w = ch < 2 ? w4.x : ch < 4 ? w4.y : ch < 6 ? w4.z : w4.w;
            f[i] = ((ch & 1) ? hi_f(w) : lo_f(w)) * inv;
          }
          q[d] = kv8_pack4<DT>(f[0], f[1], f[2], f[3]);
        }
        *reinterpret_cast<uint4*>(at + (c * 8 + ch) * 16) = make_uint4(q[0], q[1], q[2], q[3]);
      }
    }
  }
  __syncthreads();
  // the image leaves in whole 16-byte pieces, consecutive lanes consecutive pieces; K: a piece of one row, V: sixteen positions of one channel
  uint8_t* out = is_v ? a.v8 : a.k8;
#pragma unroll 2
  for (int it = 0; it < 8; ++it) {
    const int p16 = it * 64 + lane;
    const int u2 = p16 / (UB / 16), off = (p16 % (UB / 16)) * 16;
    const UnitOut o = outs[threadIdx.x >> 6][u2];
    // positions of the piece: [t, t + len); new ones among them: [i0, i1)
    const int t = o.b0 + (is_v ? off / (16 * HD) * 16 : off / HD), len = is_v ? 16 : 1;
    const int i0 = max(o.pc - t, 0), i1 = min(o.end - t, len);
    const bool old = o.ratio >= 0.f && t < o.pc;                    // older positions whose grid grew
    if (o.end < 0 || (i0 >= i1 && !old)) continue;
    const uint4 w = *reinterpret_cast<const uint4*>(mine + u2 * US + off);
    uint32_t q[4] = {w.x, w.y, w.z, w.w};
    uint4* dst = reinterpret_cast<uint4*>(out + o.base + off);
    if (i0 > 0 || i1 < len) {                                       // partly new: this lane owns the piece, so it may change it in place
      const uint4 g = *dst;
      uint32_t k[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        uint32_t keep = 0xffffffffu, was_old = 0xffffffffu;
        if (is_v) {
          keep = was_old = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (4 * d + i < i0 || 4 * d + i >= i1) keep |= 0xffu << (8 * i);
            if (t + 4 * d + i < o.pc) was_old |= 0xffu << (8 * i);
          }
        }
        if (old) {
          const uint32_t re = kv8_pack4<DT>(kv8_code<DT>(k[d] & 0xff) * o.ratio, kv8_code<DT>((k[d] >> 8) & 0xff) * o.ratio,
                                            kv8_code<DT>((k[d] >> 16) & 0xff) * o.ratio, kv8_code<DT>(k[d] >> 24) * o.ratio);
          k[d] = (re & was_old) | (k[d] & ~was_old);
        }
        q[d] = (k[d] & keep) | (q[d] & ~keep);
      }
    }
    *dst = make_uint4(q[0], q[1], q[2], q[3]);
  }
}

// One row a sequence (a decode step): latency is all there is, and the general kernel's image, exchange and read-change-write of a tile cost four
// round trips to memory where this one has two (positions; row and scale): 24 heads of 32, 2.9 us against 8.6.  A lane owns 8 channels of one head's key or value; V's bytes are
// stored one by one.
template <int HD, int DT>
__global__ __launch_bounds__(256) void kv8_append_row_kernel(AppendArgs a) {
  constexpr int C = HD / 8;
  const bool is_v = blockIdx.y != 0;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  const int c = (int)(id % C);
  const long u = id / C;
  const long uu = min(u, a.units - 1);
  const int h = (int)(uu % a.H), s = (int)(uu / a.H);
  const int p = a.pos[s];
  const bool act = u < a.units && p >= 0 && p < a.cap && (!a.n_new || a.n_new[s] > 0);
  const int pc = min(max(p, 0), a.cap - 1);
  uint4 raw = *reinterpret_cast<const uint4*>((is_v ? a.v : a.k) + (is_v ? a.v_ss : a.k_ss) * s + (long)h * HD + c * 8);
  const long head = (long)s * a.H + h;
  const int blk = pc >> a.bshift, b0 = blk << a.bshift;
  float* sp = (is_v ? a.vs : a.ks) + head * (a.cap >> a.bshift) + blk;
  const float there = *sp;
  raw.x = tame2(raw.x); raw.y = tame2(raw.y); raw.z = tame2(raw.z); raw.w = tame2(raw.w);
  const uint32_t mx = pkmax_u16(pkmax_u16(raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu), pkmax_u16(raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu));
  uint32_t am = max(mx & 0xffffu, mx >> 16);
#pragma unroll
  for (int o = 1; o < C; o <<= 1) am = max(am, (uint32_t)__shfl_xor((int)am, o, 64));
  if (!act) return;
  float scale = scale_of<DT>(am);
  const bool held = b0 < pc;
  if (held) scale = fmaxf(scale, there);
  const float inv = 1.0f / scale;
  if (c == 0) *sp = scale;                 // (the head's lanes are in one wave and have read it)
  uint8_t* kp = a.k8 + (head * a.cap) * HD + c * 8;
  uint8_t* vp = a.v8 + (head * a.cap) * HD + c * 128;
  if (held && scale > there) {             // the grid grew: the block's older codes once more
    const float ratio = there * inv;
    auto again = [&](uint32_t w) {
      return kv8_pack4<DT>(kv8_code<DT>(w & 0xff) * ratio, kv8_code<DT>((w >> 8) & 0xff) * ratio, kv8_code<DT>((w >> 16) & 0xff) * ratio,
                           kv8_code<DT>(w >> 24) * ratio);
    };
    if (!is_v) {
      for (int t = b0; t < pc; ++t) {
        uint2* q = reinterpret_cast<uint2*>(kp + (long)t * HD);
        *q = make_uint2(again(q->x), again(q->y));
      }
    } else {
      for (int t = b0; t < pc; t += 4)
        for (int ch = 0; ch < 8; ++ch) {
          uint32_t* q = reinterpret_cast<uint32_t*>(vp + (long)(t >> 4) * (HD * 16) + ch * 16 + (t & 15));
          const uint32_t old = pc - t >= 4 ? 0xffffffffu : (1u << (8 * (pc - t))) - 1u;
          *q = (again(*q) & old) | (*q & ~old);
        }
    }
  }
  const uint2 w = make_uint2(kv8_pack4<DT>(lo_f(raw.x) * inv, hi_f(raw.x) * inv, lo_f(raw.y) * inv, hi_f(raw.y) * inv),
                             kv8_pack4<DT>(lo_f(raw.z) * inv, hi_f(raw.z) * inv, lo_f(raw.w) * inv, hi_f(raw.w) * inv));
  if (!is_v) {
    *reinterpret_cast<uint2*>(kp + (long)pc * HD) = w;
  } else {
    uint8_t* q = vp + (long)(pc >> 4) * (HD * 16) + (pc & 15);
#pragma unroll
    for (int ch = 0; ch < 8; ++ch) q[ch * 16] = (uint8_t)((ch < 4 ? w.x : w.y) >> (8 * (ch & 3)));
  }
}

struct ReadArgs {
  const uint8_t *k8, *v8;
  const float *ks, *vs;
  bf16_t *k, *v;                    // [S, L, H, hd]
  const int* length;
  int S, H, cap, L, bshift, ntile;
  long units;
};

template <int HD, int DT>
__global__ __launch_bounds__(256) void kv8_read_kernel(ReadArgs a) {
  constexpr int C = HD / 8, U = 64 / C;                             // lanes and units (16 positions of a head) of a wave
  constexpr int UB = 16 * HD, US = UB + 32;
  __shared__ __attribute__((aligned(16))) char img[4][U * US];
  const bool is_v = blockIdx.y != 0;
  const int lane = threadIdx.x & 63;
  const int c = lane % C, ui = lane / C;
  const long u = ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * U + ui;
  const bool act = u < a.units;
  const long uu = act ? u : a.units - 1;
  const int h = (int)(uu % a.H);
  const long sj = uu / a.H;
  const int s = (int)(sj / a.ntile), tile = (int)(sj % a.ntile);
  const int t0 = tile * 16;
  const int rows = act ? min(a.L - t0, 16) : 0;
  const int len = min(max(a.length[s], 0), a.cap) - t0;             // held rows of this tile (may be <= 0)
  const long head = (long)s * a.H + h;
  const float scale = (is_v ? a.vs : a.ks)[head * (a.cap >> a.bshift) + (t0 >> a.bshift)];
  char* mine = img[threadIdx.x >> 6];
  const uint8_t* src = is_v ? a.v8 : a.k8;
  const long base = (head * a.cap + t0) * HD;                       // K and V alike
  uint4 w[8];
#pragma unroll
  for (int it = 0; it < 8; ++it) {                                  // consecutive lanes, consecutive pieces (a tile without rows: not looked at)
    const int p16 = it * 64 + lane, u2 = p16 / HD, off = (p16 % HD) * 16;
    const long b = __shfl(base, u2 * C, 64);
    const int n = __shfl(len, u2 * C, 64);
    if (n > 0) w[it] = *reinterpret_cast<const uint4*>(src + b + off);
  }
#pragma unroll
  for (int it = 0; it < 8; ++it) {
    const int p16 = it * 64 + lane;
    *reinterpret_cast<uint4*>(mine + (p16 / HD) * US + (p16 % HD) * 16) = w[it];
  }
  __syncthreads();
  const long row = (long)a.H * HD;
  bf16_t* dst = (is_v ? a.v : a.k) + ((long)s * a.L + t0) * row + (long)h * HD + c * 8;
  const char* at = mine + ui * US;
  if (!is_v) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint2 q = *reinterpret_cast<const uint2*>(at + i * HD + c * 8);
      uint4 o = make_uint4(kv8_unpack2<DT, false>(q.x, scale), kv8_unpack2<DT, true>(q.x, scale), kv8_unpack2<DT, false>(q.y, scale),
                           kv8_unpack2<DT, true>(q.y, scale));
      if (i >= len) o = make_uint4(0, 0, 0, 0);
      if (i < rows) *reinterpret_cast<uint4*>(dst + i * row) = o;
    }
    return;
  }
#pragma unroll
  for (int ch = 0; ch < 8; ++ch) w[ch] = *reinterpret_cast<const uint4*>(at + (c * 8 + ch) * 16);
#pragma unroll
  for (int d = 0; d < 8; ++d) {                                     // positions 2 d, 2 d + 1
    uint32_t p[8];                                                  // per channel: the two positions as bf16
#pragma unroll
    for (int ch = 0; ch < 8; ++ch) {
      const uint32_t x = d < 2 ? w[ch].x : d < 4 ? w[ch].y : d < 6 ? w[ch].z : w[ch].w;
      p[ch] = (d & 1) ? kv8_unpack2<DT, true>(x, scale) : kv8_unpack2<DT, false>(x, scale);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * d + e;
      const uint32_t sel = e ? 0x07060302u : 0x05040100u;
      uint4 o = make_uint4(__builtin_amdgcn_perm(p[1], p[0], sel), __builtin_amdgcn_perm(p[3], p[2], sel), __builtin_amdgcn_perm(p[5], p[4], sel),
                           __builtin_amdgcn_perm(p[7], p[6], sel));
      if (i >= len) o = make_uint4(0, 0, 0, 0);
      if (i < rows) *reinterpret_cast<uint4*>(dst + i * row) = o;
    }
  }
}

template <int HD, int DT>
int append_block(const AppendArgs& a, int block, dim3 grid, hipStream_t s) {
  switch (block) {
    case 16: hipLaunchKernelGGL((kv8_append_kernel<HD, 16, DT>), grid, dim3(256), 0, s, a); break;
    case 32: hipLaunchKernelGGL((kv8_append_kernel<HD, 32, DT>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((kv8_append_kernel<HD, 64, DT>), grid, dim3(256), 0, s, a); break;
  }
  NEKO_CHECK_LAUNCH();
  return NEKO_OK;
}

}  // namespace

// sizes every entry point of the cache accepts (the 32-bit index inside one head's bytes included)
int neko_kv8_geometry(int dtype, int S, int H, int cap, int hd, int block) {
  if (S <= 0 || H <= 0 || cap <= 0 || (dtype != 0 && dtype != 1)) return NEKO_ERR_ARG;
  if (hd != 32 && hd != 64 && hd != 128) return NEKO_ERR_UNSUPPORTED;
  if (block != 16 && block != 32 && block != 64) return NEKO_ERR_UNSUPPORTED;
  if (cap % 64 || cap > (1 << 24) || S > 65535 || H > 65535) return NEKO_ERR_UNSUPPORTED;
  return NEKO_OK;
}

int neko_kv8_append_impl(uint8_t* k8, uint8_t* v8, float* ks, float* vs, int dtype, int S, int H, int cap, int hd, int block, const bf16_t* k, long k_ss,
                         long k_st, const bf16_t* v, long v_ss, long v_st, const int* pos, const int* n_new, int T, hipStream_t s) {
  if (!k8 || !v8 || !ks || !vs || !k || !v || !pos || T <= 0) return NEKO_ERR_ARG;
  const int rc = neko_kv8_geometry(dtype, S, H, cap, hd, block);
  if (rc) return rc;
  if (((uintptr_t)k | (uintptr_t)v) & 15 || (k_ss | k_st | v_ss | v_st) & 7) return NEKO_ERR_ARG;     // 16-byte row pieces
  const int bshift = block == 16 ? 4 : block == 32 ? 5 : 6;
  T = min(T, cap);
  AppendArgs a{k8, v8, ks, vs, k, v, k_ss, k_st, v_ss, v_st, pos, n_new, S, H, cap, T, bshift, (T - 1 + block - 1) / block + 1, 0};
  a.units = (long)S * a.nslots * H;
  if (T == 1) {
    const dim3 grid((unsigned)((a.units * (hd / 8) + 255) / 256), 2);
#define NEKO_KV8_ROW(HD)                                                                                    \
  if (dtype == 0) hipLaunchKernelGGL((kv8_append_row_kernel<HD, 0>), grid, dim3(256), 0, s, a);             \
  else hipLaunchKernelGGL((kv8_append_row_kernel<HD, 1>), grid, dim3(256), 0, s, a)
    if (hd == 32) { NEKO_KV8_ROW(32); }
    else if (hd == 64) { NEKO_KV8_ROW(64); }
    else { NEKO_KV8_ROW(128); }
#undef NEKO_KV8_ROW
    NEKO_CHECK_LAUNCH();
    return NEKO_OK;
  }
  const int per_wave = 64 / ((hd / 8) * (block / 16));
  const long blocks = (a.units + 4 * per_wave - 1) / (4 * per_wave);
  if (blocks > 0x7fffffffL) return NEKO_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)blocks, 2);
#define NEKO_KV8_APPEND(HD) return dtype == 0 ? append_block<HD, 0>(a, block, grid, s) : append_block<HD, 1>(a, block, grid, s)
  if (hd == 32) NEKO_KV8_APPEND(32);
  if (hd == 64) NEKO_KV8_APPEND(64);
  NEKO_KV8_APPEND(128);
#undef NEKO_KV8_APPEND
}

int neko_kv8_read_impl(const uint8_t* k8, const uint8_t* v8, const float* ks, const float* vs, int dtype, int S, int H, int cap, int hd, int block,
                       const int* length, int L, bf16_t* k, bf16_t* v, hipStream_t s) {
  if (!k8 || !v8 || !ks || !vs || !k || !v || !length || L <= 0) return NEKO_ERR_ARG;
  const int rc = neko_kv8_geometry(dtype, S, H, cap, hd, block);
  if (rc) return rc;
  if (L > cap) return NEKO_ERR_ARG;
  const int bshift = block == 16 ? 4 : block == 32 ? 5 : 6;
  ReadArgs a{k8, v8, ks, vs, k, v, length, S, H, cap, L, bshift, (L + 15) / 16, 0};
  a.units = (long)S * a.ntile * H;
  const long per_block = 4 * (64 / (hd / 8));
  const long blocks = (a.units + per_block - 1) / per_block;
  if (blocks > 0x7fffffffL) return NEKO_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)blocks, 2);
#define NEKO_KV8_READ(HD)                                                                              \
  if (dtype == 0) hipLaunchKernelGGL((kv8_read_kernel<HD, 0>), grid, dim3(256), 0, s, a);              \
  else hipLaunchKernelGGL((kv8_read_kernel<HD, 1>), grid, dim3(256), 0, s, a)
  if (hd == 32) { NEKO_KV8_READ(32); }
  else if (hd == 64) { NEKO_KV8_READ(64); }
  else { NEKO_KV8_READ(128); }
#undef NEKO_KV8_READ
  NEKO_CHECK_LAUNCH();
  return NEKO_OK;
}
