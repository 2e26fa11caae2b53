// Verification of drafted tokens (speculative decoding): which of n drafted tokens the target model keeps, and the token behind them.
//
// Sequence b holds K + 1 rows of target logits (row i: the distribution of the token at drafted position i; row n: behind the last draft) and
// n <= K drafted tokens x_i.  With p_i = softmax(target_i / tau), q_i = softmax(draft_i / tau) (no draft logits: q_i is 1 at x_i) and given
// uniform numbers u_i, r:
//     token i is kept while u_i q_i(x_i) < p_i(x_i);   a = number kept
//     next token: smallest v with  sum_{w <= v} f(w) > r sum_w f(w),   f = max(p_a - q_a, 0) if a < n (p_a where that is 0 everywhere), p_n otherwise
// tau = 0: x_i is kept while it is the target row's largest logit (lowest index among equals), the next token is the largest of row a.
//
// The answer is an index: a sum over 50 thousand tokens that ends next to the border picks another token in 32 bits once in a few hundred
// calls, so weights and sums are fp64 -- with an exponential of its own (pow2_64).
// Reads (2 K + 1) V logits once (HBM), then the two rows that are sampled from again (last-level cache).  Three launches: row pieces ->
// (maximum, sum); acceptance, redone by every workgroup from the pieces, and the sampled weights' sum per piece; the piece that holds the
// border and the token in it.  tau = 0 needs two.
// 64 sequences of three to seven drafts over 52305 fp32 logits: 58 us, of them 34 for the one pass over 147 MB (4.3 TB/s; the fp64 units at half
// their rate); a single sequence is three launches' latency.
#include "neko_kernels.h"

namespace {

constexpr int PIECE = 4096;                            // logits per workgroup
constexpr int VT = 256, VE = PIECE / VT;               // where every row is read: 16 a thread
// where one row is sampled from, latency is all there is: 8 a thread (64 sequences of three to seven drafts: 15.4 + 10.9 us; 16 a thread 17.1 + 13.6,
// 4 a thread 18.8 + 13.5)
constexpr int ST = 512, SE = PIECE / ST;
constexpr int MAXK = 63;                               // a lane per drafted token

struct Source;
struct VerifyArgs {
  const void *target, *draft;
  long t_sb, t_sr, d_sb, d_sr;
  const long long* tokens;
  const float *u, *r;
  const int* n_draft;
  int* accepted;
  long long* out;
  float* pm;          // [B][2K+1][pieces] maximum of the piece
  double* ps;         // sum of exp((l - piece maximum) / tau); tau = 0: the index of the maximum
  double* pw;         // [B][pieces][2] sums of the sampled weights: the residual's, the target's own
  Source* src; // [B]
  int B, K, V, pieces;
  double c, low;      // log2(e) / tau; the distance from the maximum where weights end, -1000 / c
  int greedy;
};

template <typename T> __device__ __forceinline__ float logit(const T* p, long i);
template <> __device__ __forceinline__ float logit<float>(const float* p, long i) { const float x = p[i]; return x == x ? x : -INFINITY; }
template <> __device__ __forceinline__ float logit<bf16_t>(const bf16_t* p, long i) { const float x = bf16_to_f32(p[i]); return x == x ? x : -INFINITY; }

template <typename T> __device__ __forceinline__ float raw_logit(const T* p, int i);
template <> __device__ __forceinline__ float raw_logit<float>(const float* p, int i) { return p[i]; }
template <> __device__ __forceinline__ float raw_logit<bf16_t>(const bf16_t* p, int i) { return bf16_to_f32(p[i]); }

// 2^(d c) for -1000 <= d c <= 1/2, fp64: d c = n + f, the polynomial of degree 9 that interpolates 2^f at the ten Chebyshev nodes of [-1/2, 1/2]
// (relative error 2e-14), n added to the exponent field.  Adding 1.5 2^52 leaves n in the sum's low word: no conversion and no ldexp; and the product
// is part of both multiply-adds, so it is never rounded
__device__ __forceinline__ double pow2_64(double d, double c) {
  constexpr double MAGIC = 6755399441055744.0;
  const double y = fma(d, c, MAGIC), f = fma(d, c, MAGIC - y);
  double p = 1.02059054137655955e-07;
  p = fma(p, f, 1.32596452448871106e-06);
  p = fma(p, f, 1.52526729248507372e-05);
  p = fma(p, f, 1.54034337512510097e-04);
  p = fma(p, f, 1.33335582007945925e-03);
  p = fma(p, f, 9.61812919393431262e-03);
  p = fma(p, f, 5.55041086646516704e-02);
  p = fma(p, f, 2.40226506956403407e-01);
  p = fma(p, f, 6.93147180559946174e-01);
  p = fma(p, f, 1.00000000000001354e+00);
  return __hiloint2double(__double2hiint(p) + (__double2loint(y) << 20), __double2loint(p));
}
// weight of logit l under the maximum m, c = log2(e) / tau: 2^((l - m) c), exactly 1 for the maximum at any temperature (c l - c m in one multiply-add
// is off by the rounding of c m), 0 below 2^-1000; an infinite maximum shares the mass among its equals
struct Weigh {
  double c, low;
  float m;
  bool inf;
  __device__ __forceinline__ Weigh(float m_, const VerifyArgs& a) : c(a.c), low(a.low), m(m_), inf(m_ == INFINITY || m_ == -INFINITY) {}
  __device__ __forceinline__ double operator()(float l) const {
    if (__builtin_expect(inf, 0)) return l == m && m == INFINITY ? 1.0 : 0.0;
    const double d = (double)l - (double)m;
    return d > low ? pow2_64(d, c) : 0.0;
  }
};
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ double wave_scan64(double v, int lane) {       // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ int drafted(const VerifyArgs& a, int b) { return min(max(a.n_draft ? a.n_draft[b] : a.K, 0), a.K); }

// ---- launch 1: every row piece -> maximum and sum (or the maximum's index) ----
// Bound by the vector unit: an element costs 20 instructions (15 of them fp64), so everything else stays out of the loop: whole pieces load and
// compare without bounds, and a NaN needs no test (the maximum ignores it, the lower bound of the exponent turns it into nothing).
template <typename T, bool GREEDY>
__global__ __launch_bounds__(VT) void verify_rows_kernel(VerifyArgs a) {
  __shared__ float sm[VT / 64];
  __shared__ double ss[VT / 64];
  __shared__ int si[VT / 64];
  const int piece = blockIdx.x, row = blockIdx.y, b = blockIdx.z;     // rows 0..K target, K+1..2K draft
  const int n = drafted(a, b);
  const bool is_draft = row > a.K;
  const int i = is_draft ? row - a.K - 1 : row;
  if (is_draft ? i >= n : i > n) return;                              // rows behind the drafted ones are not looked at
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = threadIdx.x;
  const int c0 = piece * PIECE;
  const T* z = (is_draft ? (const T*)a.draft + a.d_sb * b + a.d_sr * i : (const T*)a.target + a.t_sb * b + a.t_sr * i) + c0;
  const int left = a.V - c0;                                          // columns of this piece
  float x[VE];
  if (left >= PIECE) {
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = raw_logit<T>(z + e * VT, tid);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const int c = e * VT + tid;
      x[e] = raw_logit<T>(z, min(c, left - 1));
      if (c >= left) x[e] = -INFINITY;
    }
  }
  float m = x[0] == x[0] ? x[0] : -INFINITY;
  int at = tid;
#pragma unroll
  for (int e = 1; e < VE; ++e) {
    if (GREEDY) {
      if (x[e] > m) { m = x[e]; at = e * VT + tid; }
    } else {
      m = fmaxf(m, x[e]);
    }
  }
  const float wm = wave_max(m);
  if (lane == 0) sm[wave] = wm;
  __syncthreads();
  const float bm = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])))));
  const long o = ((long)b * (2 * a.K + 1) + row) * a.pieces + piece;
  if (GREEDY) {
    int idx = m == bm ? at : 0x7fffffff;                              // lowest index among equals
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) idx = min(idx, __shfl_xor(idx, d, 64));
    if (lane == 0) si[wave] = idx;
    __syncthreads();
    if (tid == 0) { a.pm[o] = bm; a.ps[o] = (double)(c0 + min(min(si[0], si[1]), min(si[2], si[3]))); }
    return;
  }
  double s = 0.0;
  if (bm == INFINITY || bm == -INFINITY) {
#pragma unroll
    for (int e = 0; e < VE; ++e) s += x[e] == bm && bm == INFINITY ? 1.0 : 0.0;
  } else {
    const double dm = (double)bm, low = a.low;
    // exponents stop at -1000: 2^-1000 beside the 1 of the maximum is nothing, and the exponent field does not run over
#pragma unroll
    for (int e = 0; e < VE; ++e) s += pow2_64(fmax((double)x[e] - dm, low), a.c);
  }
  s = wave_sum64(s);
  if (lane == 0) ss[wave] = s;
  __syncthreads();
  if (tid == 0) { a.pm[o] = bm; a.ps[o] = (ss[0] + ss[1]) + (ss[2] + ss[3]); }
}

// What is sampled from once `kept` are kept: target row and maximum and 1 / sum, and the draft row's that is taken off (or one token).
struct Source { float mp, mq; double ip, iq; int has_q; int x; };

template <typename T>
__device__ __forceinline__ double residual(float lp, float lq, int c, const Source& s, const Weigh& wp, const Weigh& wq, double& own) {
  own = wp(lp) * s.ip;
  if (s.has_q) return fmax(own - wq(lq) * s.iq, 0.0);
  return c == s.x ? 0.0 : own;
}

// ---- launch 2: acceptance (by every workgroup again, from the pieces), and the sums of the sampled weights of one piece ----
template <typename T>
__global__ __launch_bounds__(ST) void verify_accept_kernel(VerifyArgs a) {
  __shared__ double ss[ST / 64][2];
  __shared__ float row_m[2 * MAXK];
  __shared__ double row_s[2 * MAXK];
  __shared__ Source s_src;
  __shared__ int s_kept;
  const int piece = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = drafted(a, b);
  // what lane i of wave 0 needs to judge draft i, requested before the rows' statistics
  float u = 0.f, lx = 0.f, qx = 0.f;
  long long x = -1;
  if (tid < n) {
    x = a.tokens[(long)b * a.K + tid];
    u = a.u[(long)b * a.K + tid];
    const long long xc = min(max(x, 0LL), (long long)a.V - 1);
    lx = logit<T>((const T*)a.target + a.t_sb * b + a.t_sr * tid, xc);
    if (a.draft) qx = logit<T>((const T*)a.draft + a.d_sb * b + a.d_sr * tid, xc);
  }
  // rows 0..n of the target, then n of the draft: sixteen lanes each
  const int nrows = a.draft ? 2 * n + 1 : n + 1;
  for (int q = tid >> 4; q < nrows; q += ST / 16) {
    const int row = q <= n ? q : a.K + 1 + (q - n - 1);
    const long o = ((long)b * (2 * a.K + 1) + row) * a.pieces;
    float m = -INFINITY;
    for (int p = lane & 15; p < a.pieces; p += 16) m = fmaxf(m, a.pm[o + p]);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    const Weigh w(m, a);
    double s = 0.0;
    for (int p = lane & 15; p < a.pieces; p += 16) s += a.ps[o + p] * w(a.pm[o + p]);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) s += __shfl_xor(s, d, 64);
    if ((lane & 15) == 0) { row_m[q] = m; row_s[q] = s; }
  }
  __syncthreads();
  if (wave == 0) {                                                    // lane i judges draft i
    bool ok = false;
    if (lane < n && x >= 0 && x < a.V) {
      const double p = Weigh(row_m[lane], a)(lx) / row_s[lane];
      const double q = a.draft ? Weigh(row_m[n + 1 + lane], a)(qx) / row_s[n + 1 + lane] : 1.0;
      ok = (double)u * q < p;
    }
    const unsigned long long bad = ~__builtin_amdgcn_ballot_w64(ok);
    const int kept = min(n, (int)__builtin_ctzll(bad | (1ull << 63)));
    if (lane == 0) {
      Source s{row_m[kept], 0.f, row_s[kept] > 0.0 ? 1.0 / row_s[kept] : 0.0, 0.0, 0, -1};
      if (kept < n) {
        if (a.draft) {
          s.has_q = 1;
          s.mq = row_m[n + 1 + kept];
          s.iq = row_s[n + 1 + kept] > 0.0 ? 1.0 / row_s[n + 1 + kept] : 0.0;
        } else {
          const long long x = a.tokens[(long)b * a.K + kept];
          s.x = x >= 0 && x < a.V ? (int)x : -1;
        }
      }
      s_src = s;
      s_kept = kept;
      if (piece == 0) {
        a.accepted[b] = kept;
        a.src[b] = s;
      }
    }
  }
  __syncthreads();
  const int kept = s_kept;
  const Source src = s_src;
  const T* zp = (const T*)a.target + a.t_sb * b + a.t_sr * kept;
  const T* zq = src.has_q ? (const T*)a.draft + a.d_sb * b + a.d_sr * kept : zp;
  float lp[SE], lq[SE];
#pragma unroll
  for (int e = 0; e < SE; ++e) {
    const int c = min(piece * PIECE + e * ST + tid, a.V - 1);
    lp[e] = logit<T>(zp, c);
    lq[e] = logit<T>(zq, c);
  }
  const Weigh wp(src.mp, a), wq(src.mq, a);
  double sr = 0.0, so = 0.0;
#pragma unroll
  for (int e = 0; e < SE; ++e) {
    const int c = piece * PIECE + e * ST + tid;
    double own;
    const double res = residual<T>(lp[e], lq[e], c, src, wp, wq, own);
    if (c < a.V) { sr += res; so += own; }
  }
  sr = wave_sum64(sr);
  so = wave_sum64(so);
  if (lane == 0) { ss[wave][0] = sr; ss[wave][1] = so; }
  __syncthreads();
  if (tid == 0) {
    double* w = a.pw + ((long)b * a.pieces + piece) * 2;
    double t0 = 0.0, t1 = 0.0;
    for (int i = 0; i < ST / 64; ++i) { t0 += ss[i][0]; t1 += ss[i][1]; }
    w[0] = t0;
    w[1] = t1;
  }
}

__device__ __forceinline__ void write_tokens(const VerifyArgs& a, int b, int kept, long long next) {
  for (int i = threadIdx.x; i <= a.K; i += blockDim.x)
    a.out[(long)b * (a.K + 1) + i] = i < kept ? a.tokens[(long)b * a.K + i] : i == kept ? next : -1;
}

// greedy, launch 2: sixteen lanes find the best token of a row; then the chain
__global__ __launch_bounds__(VT) void verify_greedy_kernel(VerifyArgs a) {
  __shared__ int best[MAXK + 1];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int n = drafted(a, b);
  for (int q = tid >> 4; q <= n; q += VT / 16) {
    const long o = ((long)b * (2 * a.K + 1) + q) * a.pieces;
    float m = -INFINITY;
    int at = 0x7fffffff;
    for (int p = lane & 15; p < a.pieces; p += 16) {
      const float x = a.pm[o + p];
      const int i = (int)a.ps[o + p];
      if (x > m) { m = x; at = i; }
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      const float om = __shfl_xor(m, d, 64);
      const int oa = __shfl_xor(at, d, 64);
      if (om > m || (om == m && oa < at)) { m = om; at = oa; }
    }
    if ((lane & 15) == 0) best[q] = m == -INFINITY ? -1 : at;
  }
  __syncthreads();
  if (tid < 64) {
    const bool ok = lane < n && best[lane] >= 0 && best[lane] == a.tokens[(long)b * a.K + lane];
    const unsigned long long bad = ~__builtin_amdgcn_ballot_w64(ok);
    const int kept = min(n, (int)__builtin_ctzll(bad | (1ull << 63)));
    const long long next = best[kept];
    for (int i = lane; i <= a.K; i += 64) a.out[(long)b * (a.K + 1) + i] = i < kept ? a.tokens[(long)b * a.K + i] : i == kept ? next : -1;
    if (lane == 0) a.accepted[b] = kept;
  }
}

// ---- launch 3: the piece that holds the border, and the token in it ----
template <typename T>
__global__ __launch_bounds__(ST) void verify_sample_kernel(VerifyArgs a) {
  __shared__ double f[PIECE + PIECE / SE];                // a thread's consecutive weights, padded by one
  __shared__ double wsum[ST / 64];
  __shared__ int s_at, s_last;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int kept = a.accepted[b];
  const Source src = a.src[b];
  const double* w = a.pw + (long)b * a.pieces * 2;
  // every wave finds the piece: totals, then the first piece whose running sum passes the border
  double t0 = 0.0, t1 = 0.0;
  for (int p = lane; p < a.pieces; p += 64) { t0 += w[2 * p]; t1 += w[2 * p + 1]; }
  t0 = wave_sum64(t0);
  const int col = t0 > 0.0 ? 0 : 1;                       // nothing is left of p - q: the target's own distribution
  const double total = col ? wave_sum64(t1) : t0;
  if (!(total > 0.0)) {                                   // a row without a finite logit
    write_tokens(a, b, kept, -1);
    return;
  }
  const double border = (double)a.r[b] * total;
  int piece = -1;
  double before = 0.0, run0 = 0.0;
  for (int p0 = 0; p0 < a.pieces; p0 += 64) {
    const double x = p0 + lane < a.pieces ? w[2 * (p0 + lane) + col] : 0.0;
    const double incl = run0 + wave_scan64(x, lane);
    const unsigned long long some = __builtin_amdgcn_ballot_w64(x > 0.0), over = __builtin_amdgcn_ballot_w64(x > 0.0 && incl > border);
    // without a piece above the border (rounding, r next to 1) the last one with weight stands
    const int pick = over ? (int)__builtin_ctzll(over) : some ? 63 - (int)__builtin_clzll(some) : -1;
    if (pick >= 0) {
      piece = p0 + pick;
      before = __shfl(incl - x, pick, 64);
      if (over) break;
    }
    run0 = __shfl(incl, 63, 64);
  }
  const T* zp = (const T*)a.target + a.t_sb * b + a.t_sr * kept;
  const T* zq = src.has_q ? (const T*)a.draft + a.d_sb * b + a.d_sr * kept : zp;
  const Weigh wp(src.mp, a), wq(src.mq, a);
  float lp[SE], lq[SE];
#pragma unroll
  for (int e = 0; e < SE; ++e) {
    const int c = min(piece * PIECE + e * ST + tid, a.V - 1);
    lp[e] = logit<T>(zp, c);
    lq[e] = logit<T>(zq, c);
  }
#pragma unroll
  for (int e = 0; e < SE; ++e) {
    const int i = e * ST + tid, c = piece * PIECE + i;
    double own;
    const double res = residual<T>(lp[e], lq[e], c, src, wp, wq, own);
    f[i + i / SE] = c < a.V ? (col ? own : res) : 0.0;
  }
  if (tid == 0) { s_at = 0x7fffffff; s_last = -1; }
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < SE; ++e) sum += f[tid * (SE + 1) + e];
  const double incl = wave_scan64(sum, lane);
  if (lane == 63) wsum[wave] = incl;
  __syncthreads();
  double run = before + (incl - sum);
  for (int i = 0; i < wave; ++i) run += wsum[i];
  const int c0 = piece * PIECE + tid * SE;
  int at = 0x7fffffff, last = -1;
#pragma unroll
  for (int e = 0; e < SE; ++e) {
    const double x = f[tid * (SE + 1) + e];
    run += x;
    if (x > 0.0) {
      last = c0 + e;
      if (run > border && at == 0x7fffffff) at = c0 + e;
    }
  }
  if (at != 0x7fffffff) atomicMin(&s_at, at);
  if (last >= 0) atomicMax(&s_last, last);
  __syncthreads();
  write_tokens(a, b, kept, s_at != 0x7fffffff ? s_at : s_last);
}

template <typename T>
int launch(const VerifyArgs& a, hipStream_t s) {
  const int rows = a.greedy || !a.draft ? a.K + 1 : 2 * a.K + 1;
  if (a.greedy) hipLaunchKernelGGL((verify_rows_kernel<T, true>), dim3(a.pieces, rows, a.B), dim3(VT), 0, s, a);
  else hipLaunchKernelGGL((verify_rows_kernel<T, false>), dim3(a.pieces, rows, a.B), dim3(VT), 0, s, a);
  NEKO_CHECK_LAUNCH();
  if (a.greedy) {
    hipLaunchKernelGGL(verify_greedy_kernel, dim3(a.B), dim3(VT), 0, s, a);
  } else {
    hipLaunchKernelGGL((verify_accept_kernel<T>), dim3(a.pieces, a.B), dim3(ST), 0, s, a);
    NEKO_CHECK_LAUNCH();
    hipLaunchKernelGGL((verify_sample_kernel<T>), dim3(a.B), dim3(ST), 0, s, a);
  }
  NEKO_CHECK_LAUNCH();
  return NEKO_OK;
}

}  // namespace

long neko_verify_draft_ws_bytes_impl(int B, int K, int V) {
  if (B <= 0 || K <= 0 || V <= 0) return 0;
  const long pieces = ((long)V + PIECE - 1) / PIECE;
  return (long)B * pieces * ((2 * K + 1) * 12L + 16L) + (long)B * (long)sizeof(Source);
}

int neko_verify_draft_impl(const void* target, long t_sb, long t_sr, const void* draft, long d_sb, long d_sr, int is_bf16, int B, int K, int V,
                           const long long* tokens, const float* u, const float* r, const int* n_draft, float temperature, int* accepted,
                           long long* out, void* ws, long ws_bytes, hipStream_t s) {
  if (!target || !tokens || !accepted || !out || !ws || B <= 0 || K <= 0 || V <= 0) return NEKO_ERR_ARG;
  if (!(temperature >= 0.f && temperature <= 3.402823466e38f) || (temperature > 0.f && (!u || !r))) return NEKO_ERR_ARG;
  if (K > MAXK - 1 || B > 65535 || V > (1 << 30)) return NEKO_ERR_UNSUPPORTED;
  if ((uintptr_t)ws & 7 || ws_bytes < neko_verify_draft_ws_bytes_impl(B, K, V)) return NEKO_ERR_ARG;
  VerifyArgs a{};
  a.target = target; a.draft = draft; a.t_sb = t_sb; a.t_sr = t_sr; a.d_sb = d_sb; a.d_sr = d_sr;
  a.tokens = tokens; a.u = u; a.r = r; a.n_draft = n_draft; a.accepted = accepted; a.out = out;
  a.B = B; a.K = K; a.V = V; a.pieces = (int)(((long)V + PIECE - 1) / PIECE);
  const long cells = (long)B * (2 * K + 1) * a.pieces;
  a.ps = (double*)ws;
  a.pw = a.ps + cells;
  a.src = (Source*)(a.pw + 2L * B * a.pieces);
  a.pm = (float*)(a.src + B);
  a.greedy = temperature == 0.f;
  a.c = a.greedy ? 1.0 : 1.4426950408889634074 / (double)temperature;
  a.low = -1000.0 / a.c;
  return is_bf16 ? launch<bf16_t>(a, s) : launch<float>(a, s);
}
