// Attention of T new rows per sequence over the 8-bit cache (layout: kv8.h).
//
//   out[s, i, hq] = sum_t softmax_t(scale * q[s, i, hq] . K[s, hq / G, t]) V[s, hq / G, t]   over the visible t of the row at position p = pos[s] + i:
//   start[s] <= t <= p   and   (window == 0, or t > p - window, or t < start[s] + sinks)
//
// Rows i >= n_new[s] are left as they are; a row that sees nothing is 0.  Codes are unpacked to bf16 (exact), scores, maxima, sums and the
// output accumulate in fp32; block scales never touch an operand: K's multiplies the scores, V's the probabilities.
#include "kv8.h"
#include <type_traits>

namespace {

constexpr float NEVER = -3.0e38f;       // a running maximum before any visible key (finite: no special cases)
// Sums of probabilities x values pass fp32's end long before their quotient does: values of 1.75 2^127 are kept by the cache.  Both kernels hold the
// values by a power of two `vref`, 1 unless a visible block's scale exceeds what the kernel's sums have room for; the quotient is formed before the
// power is put back.  Partial results are quotients too.
constexpr float VTOP_ROWS = 0x1p64f;    // 2^24 keys x 448 x 2^64 (probabilities at most 1)
constexpr float VTOP_TILE = 0x1p40f;    // the same x probabilities of at most 2^40: 2^113

struct AttnArgs {
  const uint8_t *k8, *v8;
  const float *ks, *vs;
  const bf16_t* q;
  bf16_t* out;
  long q_ss, q_st, o_ss, o_st;
  const int *pos, *n_new, *start;
  float *part_o, *part_ml;           // [S * H][splits][row tiles * rows per tile][hd], quotients, and [..][2], maximum and sum
  int S, H, G, cap, T, bshift, window, sinks, splits, rtiles;
  float scale_log2e;
};

// What the rows of one tile see of their sequence.  Key tiles of 64 positions: first those with sinks, then the window (or everything).
struct Span {
  int rows;          // rows of this call (n * G)
  int p0;            // position of row 0
  int first;         // first visible key
  int plast;         // last position of the tile's rows
  int pfirst;        // first position of the tile's rows
  int a0, na, b0, nt;
};
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
// (rows == 0: this row tile has nothing to do.  Every field is wave-uniform and in a scalar register: as a plain struct the compiler kept it in
// scratch, and the reload of a field inside the key loop waited for the whole prefetch)
__device__ __forceinline__ Span span_of(const AttnArgs& a, int s, int r0, int r1) {
  const int p = uni(a.pos[s]);
  const int given = a.n_new ? uni(a.n_new[s]) : a.T;
  const bool ok = p >= 0 && p < a.cap && given > 0;
  const int n = ok ? min(min(given, a.T), a.cap - p) : 0;
  Span sp;
  sp.rows = r0 < n * a.G ? n * a.G : 0;
  sp.p0 = p;
  sp.pfirst = p + r0 / a.G;
  sp.plast = p + max(min(r1, n * a.G) - 1, 0) / a.G;
  sp.first = a.start ? max(uni(a.start[s]), 0) : 0;
  const int lo = a.window > 0 ? max(sp.first, sp.pfirst - a.window + 1) : sp.first;
  const int sink_last = (int)min((long)sp.first + a.sinks - 1, (long)sp.plast);
  sp.b0 = lo >> 6;
  sp.a0 = sp.first >> 6;
  sp.na = a.window > 0 && a.sinks > 0 ? max(0, min((sink_last >> 6) + 1, sp.b0) - sp.a0) : 0;
  sp.nt = sp.first > sp.plast ? 0 : sp.na + (sp.plast >> 6) + 1 - sp.b0;
  return sp;
}
__device__ __forceinline__ int tile_of(const Span& sp, int i) { return i + (i < sp.na ? sp.a0 : sp.b0 - sp.na); }
// the keys a row at position p sees: [first, p], without (lowest, sinks_end) if there is a window.  No short cuts: selects, no branches.
struct Sight { int p, first, low, sinks_end; };
__device__ __forceinline__ Sight sight_of(const AttnArgs& a, const Span& sp, int p) {
  return Sight{p, sp.first, a.window > 0 ? p - a.window : -1, a.window > 0 ? (int)min((long)sp.first + a.sinks, 0x7fffffffL) : 0};
}
__device__ __forceinline__ bool visible(const Sight& v, int key) {
  return (key <= v.p) & (key >= v.first) & ((key > v.low) | (key < v.sinks_end));
}

// ---- few rows: a wave owns whole key tiles --------------------------------------------------------------------------------
// One workgroup of NW waves per (split, head, sequence, row tile).  A wave takes every NW-th 64-key tile of its split and keeps its own
// running maximum, sum and output for 16 NQ rows; the waves meet once at the end in LDS, the splits in a second kernel.  No LDS and no
// barrier in the loop: operands go from memory to registers in matrix-operand order.  S^T = K Q^T (a lane holds 4 keys of one row per
// 16 x 16 tile); the keys a matrix row stands for are chosen so that a lane's 16 scores of a 64-key tile are 16 CONSECUTIVE positions:
// matrix row r of tile t is key 16 (r / 4) + 4 t + r % 4.  They are then, as they stand, the operand of O^T = V^T P^T whose other
// operand is one 16-byte load of V's transposed tile, and they share one block scale.
// Bound by the cache's bytes where there are many: one token for each of 32 sequences of up to 8192 keys, 16 heads of 128 in int8: 139 us, 5.1 TB/s
// (a copy: 5.2); by the latency of positions -> queries and keys -> products -> the meeting of the waves where there are few: 7 us for 24 heads
// of 32 over 1000 keys.
constexpr int KT = 64;

template <int HD, int DT, int NQ, int NW>
__global__ __launch_bounds__(NW * 64, NQ == 1 || HD < 128 ? 2 : 1) void attn_kv8_rows_kernel(AttnArgs a) {
  constexpr int NC = HD / 16;                 // channel tiles
  constexpr int NK = HD / 32;                 // contraction steps of the scores
  constexpr int LDO = HD + 4;
  __shared__ float sm_o[NW][16][LDO];
  __shared__ float sm_ml[NW][16][2];
  __shared__ float sm_v[NW];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int split = blockIdx.x % a.splits, rt = blockIdx.x / a.splits;
  const int h = blockIdx.y, s = blockIdx.z;
  const Span sp = span_of(a, s, rt * NQ * 16, rt * NQ * 16 + NQ * 16);
  if (sp.rows == 0) return;
  const int per = (sp.nt + a.splits - 1) / a.splits;
  const int i_end = min(sp.nt, (split + 1) * per);
  const long head = (long)s * a.H + h;
  const uint8_t* kb = a.k8 + head * a.cap * HD;
  const uint8_t* vb = a.v8 + head * a.cap * HD;
  const float* ksb = a.ks + head * (a.cap >> a.bshift);
  const float* vsb = a.vs + head * (a.cap >> a.bshift);

  // queries: contraction slot (step, g, j) is channel 16 (4 (step / 2) + g) + 8 (step % 2) + j, for hd = 32 channel 8 g + j
  bf16x8_v qf[NQ][NK];
  Sight sight[NQ];                            // what the lane's row sees
#pragma unroll
  for (int iq = 0; iq < NQ; ++iq) {
    const int row = min(rt * NQ * 16 + iq * 16 + r, sp.rows - 1);
    const int t = row / a.G, gq = row - t * a.G;
    sight[iq] = sight_of(a, sp, sp.p0 + t);
    const bf16_t* qp = a.q + a.q_ss * s + a.q_st * t + (long)(h * a.G + gq) * HD;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const int ch = HD == 32 ? 8 * g : 16 * (4 * (k >> 1) + g) + 8 * (k & 1);
      qf[iq][k] = *reinterpret_cast<const bf16x8_v*>(qp + ch);
    }
  }
  f32x4 o[NQ][NC];
  float m[NQ], l[NQ];
#pragma unroll
  for (int iq = 0; iq < NQ; ++iq) {
    m[iq] = -INFINITY;
    l[iq] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[iq][c] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  constexpr int KW = HD == 32 ? 2 : HD / 16;  // dwords of K per lane and 16-key row tile (8 B | 16 B | 32 B)
  uint32_t kc[4][KW], kn[4][KW];
  uint4 vc[NC], vn[NC];
  float ksc = 0.f, vsc = 0.f, ksn = 0.f, vsn = 0.f;
  auto load = [&](int tile, uint32_t (&kk)[4][KW], uint4 (&vv)[NC], float& kscale, float& vscale) {
    const uint8_t* kp = kb + ((long)tile * KT + (r >> 2) * 16 + (r & 3)) * HD;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if constexpr (HD == 32) {
        const uint2 w = *reinterpret_cast<const uint2*>(kp + t * 4 * HD + g * 8);
        kk[t][0] = w.x; kk[t][1] = w.y;
      } else {
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
          const uint4 w = *reinterpret_cast<const uint4*>(kp + t * 4 * HD + (j * 4 + g) * 16);
          kk[t][4 * j] = w.x; kk[t][4 * j + 1] = w.y; kk[t][4 * j + 2] = w.z; kk[t][4 * j + 3] = w.w;
        }
      }
    }
    const uint8_t* vp = vb + ((long)tile * 4 + g) * (HD * 16) + r * 16;
#pragma unroll
    for (int c = 0; c < NC; ++c) vv[c] = *reinterpret_cast<const uint4*>(vp + c * 256);
    const int b = (tile * KT + g * 16) >> a.bshift;
    kscale = ksb[b];
    vscale = vsb[b];
  };
  float vref = 1.0f, vinv = 1.0f;             // the wave's (uniform)
  int it = split * per + wave;
  if (it < i_end) load(tile_of(sp, it), kc, vc, ksc, vsc);
  for (; it < i_end; it += NW) {
    const int tile = tile_of(sp, it);
    if (it + NW < i_end) load(tile_of(sp, it + NW), kn, vn, ksn, vsn);
    const int key0 = tile * KT + g * 16;      // the lane's 16 positions
    const bool plain = tile * KT >= sp.first && tile * KT + KT - 1 <= sp.pfirst && (a.window == 0 || tile * KT > sp.plast - a.window);
    if (!plain) {                             // positions outside [first, plast] hold whatever was left there: out of V before it is multiplied by 0
      const int lo = sp.first - key0, hi = sp.plast - key0;
      uint32_t bm[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        bm[d] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * d + e >= lo && 4 * d + e <= hi) bm[d] |= 0xffu << (8 * e);
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) { vc[c].x &= bm[0]; vc[c].y &= bm[1]; vc[c].z &= bm[2]; vc[c].w &= bm[3]; }
      if (lo > 15 || hi < 0) { vsc = 0.f; ksc = 0.f; }
    }
    const float sc = ksc * a.scale_log2e;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(vsc * vinv > VTOP_ROWS) != 0, 0)) {
      float top = fmaxf(vsc, __shfl_xor(vsc, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64)) * (1.0f / VTOP_ROWS);
      const float f = vref / top;
#pragma unroll
      for (int iq = 0; iq < NQ; ++iq)
#pragma unroll
        for (int c = 0; c < NC; ++c) o[iq][c] *= f;
      vref = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(top)));
      vinv = 1.0f / vref;
    }
    vsc *= vinv;
    bf16x8_v pf[NQ][2], pl[NQ][2];
    f32x4 st[NQ][4];
#pragma unroll
    for (int iq = 0; iq < NQ; ++iq)
#pragma unroll
      for (int t = 0; t < 4; ++t) st[iq][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const bf16x8_v kf = kv8_frag<DT>(kc[t][2 * k], kc[t][2 * k + 1]);
#pragma unroll
        for (int iq = 0; iq < NQ; ++iq) st[iq][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[iq][k], st[iq][t], 0, 0, 0);
      }
#pragma unroll
    for (int iq = 0; iq < NQ; ++iq) {
      float x[16];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[4 * t + i] = st[iq][t][i] * sc;
          if (!plain) x[4 * t + i] = visible(sight[iq], key0 + 4 * t + i) ? x[4 * t + i] : -INFINITY;
        }
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mn = fmaxf(m[iq], mx);
      const float ms = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m[iq] - ms);
      m[iq] = mn;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] = __builtin_amdgcn_exp2f(x[i] - ms);
        sum += x[i];
        x[i] *= vsc;
      }
      l[iq] = l[iq] * alpha + sum;
#pragma unroll
      for (int c = 0; c < NC; ++c) o[iq][c] *= alpha;
      // the probabilities enter the product as two bf16 (value and remainder, 16 bits together): the loop waits for memory, and a single
      // rounding would add as much again to the error as the output's own
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float y[8], z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[8 * u + e];
        pf[iq][u] = pack8_bf16(y);
        const uint4 w = __builtin_bit_cast(uint4, pf[iq][u]);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          z[2 * e] = y[2 * e] - __uint_as_float(ww[e] << 16);
          z[2 * e + 1] = y[2 * e + 1] - __uint_as_float(ww[e] & 0xffff0000u);
        }
        pl[iq][u] = pack8_bf16(z);
      }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const bf16x8_v v0 = kv8_frag<DT>(vc[c].x, vc[c].y), v1 = kv8_frag<DT>(vc[c].z, vc[c].w);
#pragma unroll
      for (int iq = 0; iq < NQ; ++iq) {
        o[iq][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, pf[iq][0], o[iq][c], 0, 0, 0);
        o[iq][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, pf[iq][1], o[iq][c], 0, 0, 0);
        o[iq][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, pl[iq][0], o[iq][c], 0, 0, 0);
        o[iq][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, pl[iq][1], o[iq][c], 0, 0, 0);
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int w = 0; w < KW; ++w) kc[t][w] = kn[t][w];
#pragma unroll
    for (int c = 0; c < NC; ++c) vc[c] = vn[c];
    ksc = ksn;
    vsc = vsn;
  }

  // the waves meet
  if (lane == 0) sm_v[wave] = vref;
#pragma unroll
  for (int iq = 0; iq < NQ; ++iq) {
    l[iq] += __shfl_xor(l[iq], 16, 64);
    l[iq] += __shfl_xor(l[iq], 32, 64);
    if (iq) __syncthreads();
#pragma unroll
    for (int c = 0; c < NC; ++c) *reinterpret_cast<f32x4*>(&sm_o[wave][r][c * 16 + g * 4]) = o[iq][c];
    if (g == 0) { sm_ml[wave][r][0] = m[iq]; sm_ml[wave][r][1] = l[iq]; }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * (HD / 4); e += NW * 64) {
      const int row16 = e / (HD / 4), c4 = (e % (HD / 4)) * 4;
      const int row = rt * NQ * 16 + iq * 16 + row16;
      if (row >= sp.rows) continue;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) mm = fmaxf(mm, sm_ml[w][row16][0]);
      const float ms = mm == -INFINITY ? 0.f : mm;
      float vr = sm_v[0];
#pragma unroll
      for (int w = 1; w < NW; ++w) vr = fmaxf(vr, sm_v[w]);
      const float vri = 1.0f / vr;
      float ll = 0.f;
      f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = __builtin_amdgcn_exp2f(sm_ml[w][row16][0] - ms);
        ll = fmaf(f, sm_ml[w][row16][1], ll);
        acc += *reinterpret_cast<const f32x4*>(&sm_o[w][row16][c4]) * (f * (sm_v[w] * vri));
      }
      acc *= ll == 0.f ? 0.f : 1.0f / ll;
      acc *= vr;
      if (a.splits == 1) {
        const int t = row / a.G, gq = row - t * a.G;
        uint2 pk;
        pk.x = pack_bf16x2(acc[0], acc[1]);
        pk.y = pack_bf16x2(acc[2], acc[3]);
        *reinterpret_cast<uint2*>(a.out + a.o_ss * s + a.o_st * t + (long)(h * a.G + gq) * HD + c4) = pk;
      } else {
        const long pr = (head * a.splits + split) * ((long)a.rtiles * NQ * 16) + row;
        *reinterpret_cast<f32x4*>(a.part_o + pr * HD + c4) = acc;
        if (c4 == 0) { a.part_ml[2 * pr] = mm; a.part_ml[2 * pr + 1] = ll; }
      }
    }
  }
}

// ---- many rows: key tiles through LDS -------------------------------------------------------------------------------------
// One workgroup of NW waves per (split, head, sequence, row tile of 32 NW rows); a wave owns 32 rows.  A 64-key tile is unpacked ONCE, on its way
// into LDS (codes x scale as bf16: exact), and read there by every wave as matrix operands; the codes of the tile after it are on their way
// meanwhile, one barrier per tile.  32 x 32 x 16 products: S^T = K Q^T, then O^T = V^T P^T with the probabilities as they stand -- LDS row r of a
// 32-key half tile holds key 16 ((r >> 2) & 1) + 4 (r >> 3) + (r & 3), so that a lane's 16 scores are 16 consecutive keys.
//   K image: rows of HD bf16, 16-byte pieces XORed with the row (16 lanes read 16 rows: all banks once);  V image: [8 keys][channel] pieces.
// The running reference of a row moves only when its probabilities outgrow 2^40 (fp32 sums and bf16 probabilities do not care about a common
// factor), so the common step takes no maximum.  Probabilities are rounded to bf16 once, and the sums are of the rounded ones: their errors are
// independent and average out like the values' own (measured 1.0-1.4 x the error of the rounded output); a second product for their low parts
// would cost 50 % of the matrix work.
// 4 sequences x 16 heads of 128, 1024 queries over 2976-4000 keys: 127-133 us in a row of calls (0.88-0.92 PFLOP/s), 140-150 one at a time (156 with a
// maximum a tile).  The products and their operand reads alone take 53 us, with the staging 62: what binds it are
// the vector instructions of the softmax (130 a tile and wave), which two waves of a SIMD in the same phase do not hide behind each other's
// products.  Opposite phases for the two halves of the workgroup, a barrier between the phases, took 151; softmax of one tile beside the products
// of another within a wave 155, and so with 64 rows a wave, one wave per SIMD, 176.
template <int HD>
__device__ __forceinline__ int kimg(int row, int piece) {
  constexpr int PC = HD / 8, SH = HD == 128 ? 0 : HD == 64 ? 1 : 2;
  return row * (HD * 2) + ((piece ^ ((row >> SH) & (PC - 1))) << 4);
}

template <int HD, int DT, int NW>
__global__ __launch_bounds__(NW * 64, 2) void attn_kv8_tile_kernel(AttnArgs a) {
  constexpr int NC = HD / 32, NK = HD / 16;
  constexpr int IMG = KT * HD * 2;                        // bytes of one image
  constexpr int UNITS = KT * HD / 16;                     // 16-byte pieces of K, and of V, in a tile
  constexpr int NT = NW * 64;
  constexpr int UPT = (UNITS + NT - 1) / NT;              // pieces per thread
  constexpr int RT = NW * 32;
  __shared__ __attribute__((aligned(16))) char kimgs[2][IMG];
  __shared__ __attribute__((aligned(16))) char vimgs[2][IMG];
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int r = lane & 31, hf = lane >> 5;
  // consecutive row tiles of a head on one XCD (they read the same keys), those with the most keys first
  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int split = id % a.splits, rt = a.rtiles - 1 - id / a.splits % a.rtiles;
  const int hs = id / (a.splits * a.rtiles), h = hs % a.H, s = hs / a.H;
  const Span sp = span_of(a, s, rt * RT, rt * RT + RT);
  if (sp.rows == 0) return;
  const int per = (sp.nt + a.splits - 1) / a.splits;
  const int i0 = split * per, n = min(sp.nt, i0 + per) - i0;      // this workgroup's tiles
  const long head = (long)s * a.H + h;
  const uint8_t* kb = a.k8 + head * a.cap * HD;
  const uint8_t* vb = a.v8 + head * a.cap * HD;
  const float* ksb = a.ks + head * (a.cap >> a.bshift);
  const float* vsb = a.vs + head * (a.cap >> a.bshift);

  const int row = rt * RT + wave * 32 + r;
  const int w0 = rt * RT + wave * 32;                     // the wave's first row
  const int rc = min(row, sp.rows - 1);                   // (lanes and waves behind the last row compute it again and write nothing)
  const int t = rc / a.G, gq = rc - t * a.G;
  const Sight sight = sight_of(a, sp, sp.p0 + t);
  const int wfirst = sp.p0 + min(w0, sp.rows - 1) / a.G, wlast = sp.p0 + min(w0 + 31, sp.rows - 1) / a.G;
  // the power of two the values are held by: from the scales of this workgroup's blocks, every wave for itself
  float vref = 1.0f, vinv = 1.0f;
  {
    const int bpt = KT >> a.bshift;                       // blocks of a tile
    float top = 0.f;
    for (int b = lane; b < max(n, 0) * bpt; b += 64) {
      const int blk = tile_of(sp, i0 + b / bpt) * bpt + b % bpt, at = blk << a.bshift;
      if (at <= sp.plast && at + (1 << a.bshift) > sp.first) top = fmaxf(top, vsb[blk]);
    }
    top = __uint_as_float(uni(__float_as_uint(wave_max(top))));
    if (top > VTOP_TILE) {
      vref = top * (1.0f / VTOP_TILE);
      vinv = 1.0f / vref;
    }
  }
  bf16x8_v qf[NK];
  {
    const bf16_t* qp = a.q + a.q_ss * s + a.q_st * t + (long)(h * a.G + gq) * HD + hf * 8;
#pragma unroll
    for (int k = 0; k < NK; ++k) qf[k] = *reinterpret_cast<const bf16x8_v*>(qp + k * 16);
  }
  f32x16 o[NC], sc[2];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[c][i] = 0.f;
  float m = NEVER, l = 0.f;
  bf16x8_v pf[4];
  // the queries are waited for here: left to the first product, that wait would stand in the key loop and cover the prefetch there too
#pragma unroll
  for (int k = 0; k < NK; ++k) asm volatile("" : "+v"(qf[k]));

  // ---- pieces of 16 bytes on their way in: UPT of a K tile, UPT of a V tile per thread ----
  uint4 kst[UPT], vst[UPT];
  float kss[UPT], vss[UPT];
  uint32_t off[UPT];
  int kblk[UPT], vblk[UPT];
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    const int u = min(tid + i * NT, UNITS - 1);
    off[i] = u * 16;
    kblk[i] = (u / (HD / 16)) >> a.bshift;
    vblk[i] = ((u / HD) * 16) >> a.bshift;
  }
  auto fetch_k = [&](int j) {
    if (j >= n) return;
    const int tile = tile_of(sp, i0 + j);
    const uint8_t* base = kb + (long)tile * (KT * HD);
    const float* sb = ksb + ((tile * KT) >> a.bshift);
#pragma unroll
    for (int i = 0; i < UPT; ++i) { kst[i] = *reinterpret_cast<const uint4*>(base + off[i]); kss[i] = sb[kblk[i]]; }
  };
  auto fetch_v = [&](int j) {
    if (j >= n) return;
    const int tile = tile_of(sp, i0 + j);
    const uint8_t* base = vb + (long)tile * (KT * HD);
    const float* sb = vsb + ((tile * KT) >> a.bshift);
#pragma unroll
    for (int i = 0; i < UPT; ++i) { vst[i] = *reinterpret_cast<const uint4*>(base + off[i]); vss[i] = sb[vblk[i]]; }
  };
  auto put = [&](char* img, int at0, int at1, const uint32_t (&w)[4], float sc8) {
    *reinterpret_cast<uint4*>(img + at0) = make_uint4(kv8_unpack2<DT, false>(w[0], sc8), kv8_unpack2<DT, true>(w[0], sc8),
                                                      kv8_unpack2<DT, false>(w[1], sc8), kv8_unpack2<DT, true>(w[1], sc8));
    *reinterpret_cast<uint4*>(img + at1) = make_uint4(kv8_unpack2<DT, false>(w[2], sc8), kv8_unpack2<DT, true>(w[2], sc8),
                                                      kv8_unpack2<DT, false>(w[3], sc8), kv8_unpack2<DT, true>(w[3], sc8));
  };
  // positions outside [first, plast] hold whatever was left there: zeros
  auto stage_k = [&](int j, char* img) {
    if (j >= n) return;
    const int tk = tile_of(sp, i0 + j) * KT;
    const bool edge = tk < sp.first || tk + KT - 1 > sp.plast;
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      const int u = tid + i * NT;
      if (UNITS % NT && u >= UNITS) break;
      uint32_t w[4] = {kst[i].x, kst[i].y, kst[i].z, kst[i].w};
      float sc8 = kss[i];
      const int key = u / (HD / 16), cc = u % (HD / 16);
      const int kk = key & 31;                            // its row in the half tile
      const int lr = (key & 32) + 8 * ((kk >> 2) & 3) + 4 * (kk >> 4) + (kk & 3);
      if (edge && (tk + key < sp.first || tk + key > sp.plast)) {
        w[0] = w[1] = w[2] = w[3] = 0;
        sc8 = 0.f;
      }
      put(img, kimg<HD>(lr, 2 * cc), kimg<HD>(lr, 2 * cc + 1), w, sc8);
    }
  };
  auto stage_v = [&](int j, char* img) {
    if (j >= n) return;
    const int tk = tile_of(sp, i0 + j) * KT;
    const bool edge = tk < sp.first || tk + KT - 1 > sp.plast;
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      const int u = tid + i * NT;
      if (UNITS % NT && u >= UNITS) break;
      uint32_t w[4] = {vst[i].x, vst[i].y, vst[i].z, vst[i].w};
      float sc8 = vss[i];
      if (__builtin_expect(vinv != 1.0f, 0)) {            // (the conversion reads a scale's exponent only: no subnormal ones)
        sc8 *= vinv;
        if (sc8 < 0x1p-126f) w[0] = w[1] = w[2] = w[3] = 0;
      }
      const int t16 = u / HD, ch = u % HD;
      if (edge) {
        const int lo = sp.first - (tk + t16 * 16), hi = sp.plast - (tk + t16 * 16);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          uint32_t bm = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * d + e >= lo && 4 * d + e <= hi) bm |= 0xffu << (8 * e);
          w[d] &= bm;
        }
        if (lo > 15 || hi < 0) sc8 = 0.f;
      }
      put(img, ((2 * t16) * HD + ch) * 16, ((2 * t16 + 1) * HD + ch) * 16, w, sc8);
    }
  };

  // Scores of tile j.  The mask is what the products start from, 0 or -inf: the scores are written by the products alone, in place.
  auto k_frag = [&](const char* img, int kt, int k) { return *reinterpret_cast<const bf16x8_v*>(img + kimg<HD>(kt * 32 + r, 2 * k + hf)); };
  auto first_scores = [&](int j, const char* img) {
    const int tk = tile_of(sp, i0 + j) * KT;
    const bool plain = tk >= sp.first && tk + KT - 1 <= wfirst && (a.window == 0 || tk > wlast - a.window);
    if (plain) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        f32x16 z;
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = 0.f;
        sc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_frag(img, kt, 0), qf[0], z, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        f32x16 z;
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = visible(sight, tk + kt * 32 + hf * 16 + i) ? 0.f : -INFINITY;
        sc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_frag(img, kt, 0), qf[0], z, 0, 0, 0);
      }
    }
  };
  auto more_scores = [&](const char* img) {
#pragma unroll
    for (int k = 1; k < NK; ++k)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) sc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_frag(img, kt, k), qf[k], sc[kt], 0, 0, 0);
  };
  auto output = [&](const char* img) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const bf16x8_v vf = *reinterpret_cast<const bf16x8_v*>(img + (((q >> 1) * 4 + 2 * hf + (q & 1)) * HD + c * 32 + r) * 16);
        o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[q], o[c], 0, 0, 0);
      }
  };

  // ---- probabilities against the running reference as it stands; a lane whose sum of 32 passes 2^40 (or is infinite: the first
  // visible keys) sends the wave back for the maximum.  Sums are of the rounded probabilities, two an instruction. ----
  auto softmax = [&]() {
    float sum;
    auto probabilities = [&]() {
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_exp2f(fmaf(sc[q >> 1][8 * (q & 1) + e], a.scale_log2e, -m));
        pf[q] = pack8_bf16(y);
        const uint4 w = __builtin_bit_cast(uint4, pf[q]);
        const bf16x2_t one = {(__bf16)1.0f, (__bf16)1.0f};
        s0 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w.x), one, s0, false);
        s1 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w.y), one, s1, false);
        s0 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w.z), one, s0, false);
        s1 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w.w), one, s1, false);
      }
      sum = s0 + s1;
    };
    probabilities();
    if (__builtin_amdgcn_ballot_w64(!(sum <= 0x1p40f))) {
      float mx = sc[0][0];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[kt][i]);
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
      mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * a.scale_log2e;        // scale > 0 (checked on entry)
      const float mn = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][i] *= alpha;
      probabilities();
    }
    l += sum;
  };

  if (n > 0) {
    fetch_k(0);
    fetch_v(0);
    stage_k(0, kimgs[0]);
    stage_v(0, vimgs[0]);
    fetch_k(1);
    fetch_v(1);
    __syncthreads();
    // step j, its parity known to the compiler: LDS addresses are registers + constants
    auto step = [&](int j, auto parity) {
      constexpr int p = parity;
      first_scores(j, kimgs[p]);
      more_scores(kimgs[p]);
      softmax();
      stage_k(j + 1, kimgs[p ^ 1]);                       // requested a whole step ago; its last readers are behind the barrier
      stage_v(j + 1, vimgs[p ^ 1]);
      fetch_k(j + 2);
      fetch_v(j + 2);
      output(vimgs[p]);
      __syncthreads();
    };
    int j = 0;
    for (; j + 1 < n; j += 2) {
      step(j, std::integral_constant<int, 0>{});
      step(j + 1, std::integral_constant<int, 1>{});
    }
    if (j < n) step(j, std::integral_constant<int, 0>{});
  }
  l += __shfl_xor(l, 32, 64);
  if (row >= sp.rows) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[c][i] = o[c][i] * inv * vref;
  if (a.splits == 1) {
    bf16_t* op = a.out + a.o_ss * s + a.o_st * t + (long)(h * a.G + gq) * HD;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint2 pk;
        pk.x = pack_bf16x2(o[c][4 * j], o[c][4 * j + 1]);
        pk.y = pack_bf16x2(o[c][4 * j + 2], o[c][4 * j + 3]);
        *reinterpret_cast<uint2*>(op + c * 32 + 8 * j + 4 * hf) = pk;
      }
  } else {
    const long pr = (head * a.splits + split) * ((long)a.rtiles * RT) + row;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 x = {o[c][4 * j], o[c][4 * j + 1], o[c][4 * j + 2], o[c][4 * j + 3]};
        *reinterpret_cast<f32x4*>(a.part_o + pr * HD + c * 32 + 8 * j + 4 * hf) = x;
      }
    if (hf == 0) { a.part_ml[2 * pr] = m; a.part_ml[2 * pr + 1] = l; }
  }
}

// the splits meet: HD / 4 lanes per row
template <int HD>
__global__ __launch_bounds__(256) void attn_kv8_merge_kernel(AttnArgs a, int rows_pad) {
  constexpr int LR = HD / 4;
  const int h = blockIdx.y, s = blockIdx.z;
  const int row = blockIdx.x * (256 / LR) + threadIdx.x / LR;
  const int c4 = (threadIdx.x % LR) * 4;
  const int p = a.pos[s];
  int n = min(a.n_new ? a.n_new[s] : a.T, a.T);
  if (p < 0 || p >= a.cap || n <= 0) return;
  n = min(n, a.cap - p);
  if (row >= n * a.G) return;
  const long base = ((long)s * a.H + h) * a.splits * rows_pad + row;
  float mm = -INFINITY;
  for (int i = 0; i < a.splits; ++i) mm = fmaxf(mm, a.part_ml[2 * (base + (long)i * rows_pad)]);
  const float ms = mm == -INFINITY ? 0.f : mm;
  auto share = [&](int i) {                               // split i's share of the row's sum, not yet divided by it
    const long pr = base + (long)i * rows_pad;
    return __builtin_amdgcn_exp2f(a.part_ml[2 * pr] - ms) * a.part_ml[2 * pr + 1];
  };
  float ll = 0.f;
#pragma unroll 4
  for (int i = 0; i < a.splits; ++i) ll += share(i);
  const float inv = ll == 0.f ? 0.f : 1.0f / ll;
  f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < a.splits; ++i) acc += *reinterpret_cast<const f32x4*>(a.part_o + (base + (long)i * rows_pad) * HD + c4) * (share(i) * inv);
  const int t = row / a.G, gq = row - t * a.G;
  uint2 pk;
  pk.x = pack_bf16x2(acc[0], acc[1]);
  pk.y = pack_bf16x2(acc[2], acc[3]);
  *reinterpret_cast<uint2*>(a.out + a.o_ss * s + a.o_st * t + (long)(h * a.G + gq) * HD + c4) = pk;
}

// How a call is cut: the kernel, its row tile and the number of splits of the key axis with the least estimated time
//   launch + (fixed + step * (64-key tiles of the longest wave)) * (1 + crowd * (workgroups per CU - 1)) + the merge of the partial results, if any
// in us, fitted (least squares of the logarithms) to 2000 measured calls: 8, 64, 256 key heads x sequences, 500 - 4000 keys, 16 - 384 rows, 1 - 32
// splits, each of the four kernels.  The cut taken is 2 % slower on average than the best measured one; a choice by the number of rows alone was
// 19 %, even with the best splits.  Both sides, 4000 keys: 64 rows of one sequence, 8 heads of 128: 13.4 us with 16 rows a wave, 17.9 with 32,
// 20.6 through LDS; 32 rows, 64 heads of 64: 18.3 | 19.1 | 22.9; 128 rows, 64 heads of 128: 75 | 73 | 39; 256 rows, 256 heads of 128: 164 with 128
// rows a workgroup, 145 with 256.
// Up to 64 rows stay in the register kernel, which keeps probabilities to 16 bits.
struct Plan { int rt, rtiles, splits; };
struct Cost { float fixed, step, crowd; };
constexpr Cost COST[3][4] = {{{0.12f, 1.34f, 1.0f}, {0.64f, 1.67f, 0.60f}, {1.68f, 0.77f, 0.42f}, {1.79f, 0.97f, 0.60f}},       // hd = 32
                             {{0.43f, 2.25f, 1.0f}, {0.79f, 2.09f, 0.78f}, {2.15f, 0.99f, 0.37f}, {1.28f, 1.24f, 1.0f}},        // 64
                             {{0.0f, 4.36f, 1.0f}, {2.39f, 3.96f, 1.0f}, {3.17f, 1.49f, 0.41f}, {1.19f, 1.87f, 1.0f}}};         // 128
Plan plan_of(int S, int H, int hd, int rows, int keys) {
  constexpr int RT[4] = {16, 32, 128, 256}, PER_WG[4] = {8, 4, 1, 1};       // rows of a workgroup; key tiles it works on at a time
  constexpr int SPLITS[12] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
  const int tiles = (keys + KT - 1) / KT, kernels = rows <= 64 ? 2 : 4;
  Plan p{};
  float best = 0.f;
  for (const int sp : SPLITS)
    for (int v = 0; v < kernels; ++v) {
      if (sp > 1 && (sp - 1) * PER_WG[v] >= tiles) continue;
      const Cost& c = COST[hd == 32 ? 0 : hd == 64 ? 1 : 2][v];
      const int rtiles = (rows + RT[v] - 1) / RT[v];
      const long wgs = (long)S * H * rtiles * sp;
      const int steps = ((tiles + sp - 1) / sp + PER_WG[v] - 1) / PER_WG[v];
      float t = (c.fixed + c.step * steps) * (1.0f + c.crowd * ((wgs + 255) / 256 - 1));
      if (sp > 1) t += 2.29f + 0.27f * sp + 0.15e-6f * 4 * (hd + 2) * wgs * RT[v];
      if (best == 0.f || t < best * 0.97f) { best = t; p = Plan{RT[v], rtiles, sp}; }
    }
  return p;
}
int keys_of(int cap, int T, int window, int sinks, int max_len) {
  long k = max_len > 0 && max_len < cap ? max_len : cap;
  if (window > 0 && (long)window + sinks + T + KT < k) k = (long)window + sinks + T + KT;
  return (int)k;
}

template <int HD, int DT>
int launch_rows(const AttnArgs& a, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.splits * p.rtiles), a.H, a.S);
  const dim3 flat((unsigned)(p.splits * p.rtiles) * a.H * a.S);
  if (p.rt == 256) hipLaunchKernelGGL((attn_kv8_tile_kernel<HD, DT, 8>), flat, dim3(512), 0, s, a);
  else if (p.rt == 128) hipLaunchKernelGGL((attn_kv8_tile_kernel<HD, DT, 4>), flat, dim3(256), 0, s, a);
  else if (p.rt == 16) hipLaunchKernelGGL((attn_kv8_rows_kernel<HD, DT, 1, 8>), grid, dim3(512), 0, s, a);
  else hipLaunchKernelGGL((attn_kv8_rows_kernel<HD, DT, 2, 4>), grid, dim3(256), 0, s, a);
  NEKO_CHECK_LAUNCH();
  if (p.splits > 1) {
    const int rows = a.T * a.G, per = 256 / (HD / 4);
    hipLaunchKernelGGL((attn_kv8_merge_kernel<HD>), dim3((rows + per - 1) / per, a.H, a.S), dim3(256), 0, s, a, p.rtiles * p.rt);
    NEKO_CHECK_LAUNCH();
  }
  return NEKO_OK;
}

}  // namespace

long neko_attn_kv8_ws_floats_impl(int S, int H, int G, int cap, int hd, int T, int window, int sinks, int max_len) {
  if (S <= 0 || H <= 0 || G <= 0 || T <= 0 || cap <= 0 || hd <= 0) return 0;
  const Plan p = plan_of(S, H, hd, T * G, keys_of(cap, T, window, sinks, max_len));
  return p.splits > 1 ? (long)S * H * p.splits * p.rtiles * p.rt * (hd + 2) : 0;
}

int neko_attn_kv8_impl(const uint8_t* k8, const uint8_t* v8, const float* ks, const float* vs, int dtype, int S, int H, int cap, int hd, int block,
                       const bf16_t* q, long q_ss, long q_st, bf16_t* out, long o_ss, long o_st, int G, int T, const int* pos, const int* n_new,
                       const int* start, int window, int sinks, float scale, int max_len, float* ws, long ws_floats, hipStream_t s) {
  if (!k8 || !v8 || !ks || !vs || !q || !out || !pos || G <= 0 || T <= 0 || window < 0 || sinks < 0 || !(scale > 0.f)) return NEKO_ERR_ARG;
  const int rc = neko_kv8_geometry(dtype, S, H, cap, hd, block);
  if (rc) return rc;
  if (T > cap || (long)T * G > (1 << 24)) return NEKO_ERR_ARG;
  if (((uintptr_t)q | (uintptr_t)out) & 15 || (q_ss | q_st | o_ss | o_st) & 7) return NEKO_ERR_ARG;
  {
    // rows and sequences in the order of their strides; every output row is written by its own workgroup, in no order
    const bool in_rows = S == 1 || (T > 1 && o_st <= o_ss);
    const long w = (long)H * G * hd * 2, n_lo = in_rows ? T : S, n_hi = in_rows ? S : T;
    const long q_lo = 2 * (in_rows ? q_st : q_ss), q_hi = 2 * (in_rows ? q_ss : q_st), o_lo = 2 * (in_rows ? o_st : o_ss), o_hi = 2 * (in_rows ? o_ss : o_st);
    if ((q_ss | q_st | o_ss | o_st) < 0 || !neko_rows_apart(w, n_lo, o_lo, n_hi, o_hi) || neko_rows_shared(q, q_lo, q_hi, out, o_lo, o_hi, w, n_lo, n_hi))
      return NEKO_ERR_ARG;
  }
  const Plan p = plan_of(S, H, hd, T * G, keys_of(cap, T, window, sinks, max_len));
  const long need = p.splits > 1 ? (long)S * H * p.splits * p.rtiles * p.rt * (hd + 2) : 0;
  if (need > ws_floats || (need && !ws)) return NEKO_ERR_ARG;
  if ((long)S * H * p.splits * p.rtiles > 0x7fffffffL) return NEKO_ERR_UNSUPPORTED;
  const int bshift = block == 16 ? 4 : block == 32 ? 5 : 6;
  AttnArgs a{k8, v8, ks, vs, q, out, q_ss, q_st, o_ss, o_st, pos, n_new, start, ws, nullptr, S, H, G, cap, T, bshift, window, sinks, p.splits, p.rtiles,
             scale * 1.4426950408889634f};
  a.part_ml = ws + (long)S * H * p.splits * p.rtiles * p.rt * hd;
#define NEKO_KV8_ATTN(HD) return dtype == 0 ? launch_rows<HD, 0>(a, p, s) : launch_rows<HD, 1>(a, p, s)
  if (hd == 32) NEKO_KV8_ATTN(32);
  if (hd == 64) NEKO_KV8_ATTN(64);
  NEKO_KV8_ATTN(128);
#undef NEKO_KV8_ATTN
}
