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
// calls, so weights and sums are fp64 -- with an exponential of its own (exp64 below).
// Reads (2 K + 1) V logits once (HBM), then the two rows that are sampled from again (last-level cache).  Three launches: row pieces ->
// (maximum, sum); acceptance, redone by every workgroup from the pieces, and the sampled weights' sum per piece; the piece that holds the
// border and the token in it.  tau = 0 needs two.
#include "neko_kernels.h"

namespace {

constexpr int VT = 256, VE = 16, PIECE = VT * VE;      // 4096 logits per workgroup, 16 a thread
constexpr int MAXK = 63;                               // a lane per drafted token

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
  double* pw;         // [B][pieces] sums of the sampled weights
  int B, K, V, pieces;
  double inv_tau;
  int greedy;
};

template <typename T> __device__ __forceinline__ float logit(const T* p, long i);
template <> __device__ __forceinline__ float logit<float>(const float* p, long i) { const float x = p[i]; return x == x ? x : -INFINITY; }
template <> __device__ __forceinline__ float logit<bf16_t>(const bf16_t* p, long i) { const float x = bf16_to_f32(p[i]); return x == x ? x : -INFINITY; }

// e^x for x <= 0, fp64: x = n ln 2 + f (ln 2 as its nearest double and the rest, both steps fused), Taylor series of e^f to f^13 / 13!
// (|f| <= 0.3466: the next term is 4e-18), scaled by 2^n; below -708: 0
__device__ __forceinline__ double exp64(double x) {
  const double n = rint(x * 1.4426950408889634074);
  double f = fma(n, -0.693147180559945309417, x);
  f = fma(n, -2.3190468138462996e-17, f);
  double p = 1.0 / 6227020800.0;
  p = fma(p, f, 1.0 / 479001600.0);
  p = fma(p, f, 1.0 / 39916800.0);
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return x < -708.0 ? 0.0 : ldexp(p, (int)n);
}
// weight of logit l under maximum m: equal logits weigh 1 also where both are infinite
__device__ __forceinline__ double weight(float l, float m, double inv_tau) {
  if (l == m) return m == -INFINITY ? 0.0 : 1.0;
  return exp64(((double)l - (double)m) * inv_tau);
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ int drafted(const VerifyArgs& a, int b) { return min(max(a.n_draft ? a.n_draft[b] : a.K, 0), a.K); }

// ---- launch 1: every row piece -> maximum and sum (or the maximum's index) ----
template <typename T>
__global__ __launch_bounds__(VT) void verify_rows_kernel(VerifyArgs a) {
  __shared__ float sm[VT / 64];
  __shared__ double ss[VT / 64];
  __shared__ int si[VT / 64];
  const int piece = blockIdx.x, row = blockIdx.y, b = blockIdx.z;     // rows 0..K target, K+1..2K draft
  const int n = drafted(a, b);
  const bool is_draft = row > a.K;
  const int i = is_draft ? row - a.K - 1 : row;
  if (is_draft ? i >= n : i > n) return;                              // rows behind the drafted ones are not looked at
  const T* z = is_draft ? (const T*)a.draft + a.d_sb * b + a.d_sr * i : (const T*)a.target + a.t_sb * b + a.t_sr * i;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c0 = piece * PIECE;
  float x[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    const int c = c0 + e * VT + threadIdx.x;
    x[e] = logit<T>(z, min(c, a.V - 1));
    if (c >= a.V) x[e] = -INFINITY;
  }
  float m = x[0];
  int at = c0 + (int)threadIdx.x;
#pragma unroll
  for (int e = 1; e < VE; ++e)
    if (x[e] > m) { m = x[e]; at = c0 + e * VT + (int)threadIdx.x; }
  float wm = wave_max(m);
  if (lane == 0) sm[wave] = wm;
  __syncthreads();
  float bm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const long o = ((long)b * (2 * a.K + 1) + row) * a.pieces + piece;
  if (a.greedy) {
    int idx = m == bm ? at : 0x7fffffff;                              // lowest index among equals
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) idx = min(idx, __shfl_xor(idx, d, 64));
    if (lane == 0) si[wave] = idx;
    __syncthreads();
    if (threadIdx.x == 0) { a.pm[o] = bm; a.ps[o] = (double)min(min(si[0], si[1]), min(si[2], si[3])); }
    return;
  }
  double s = 0.0;
#pragma unroll
  for (int e = 0; e < VE; ++e) s += weight(x[e], bm, a.inv_tau);
  s = wave_sum64(s);
  if (lane == 0) ss[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) { a.pm[o] = bm; a.ps[o] = (ss[0] + ss[1]) + (ss[2] + ss[3]); }
}

// a row's maximum and sum from its pieces
__device__ __forceinline__ void row_stats(const VerifyArgs& a, int b, int row, float& m, double& s) {
  const long o = ((long)b * (2 * a.K + 1) + row) * a.pieces;
  m = -INFINITY;
  for (int p = 0; p < a.pieces; ++p) m = fmaxf(m, a.pm[o + p]);
  s = 0.0;
  for (int p = 0; p < a.pieces; ++p) s += a.ps[o + p] * weight(a.pm[o + p], m, a.inv_tau);
}

// lane i of a wave judges draft i; returns the number kept (every lane)
template <typename T>
__device__ __forceinline__ int accept(const VerifyArgs& a, int b, int n, int lane) {
  bool ok = false;
  if (lane < n) {
    float mp, mq;
    double sp, sq;
    row_stats(a, b, lane, mp, sp);
    const long long x = a.tokens[(long)b * a.K + lane];
    if (x >= 0 && x < a.V) {
      const double p = weight(logit<T>((const T*)a.target + a.t_sb * b + a.t_sr * lane, x), mp, a.inv_tau) / sp;
      double q = 1.0;
      if (a.draft) {
        row_stats(a, b, a.K + 1 + lane, mq, sq);
        q = weight(logit<T>((const T*)a.draft + a.d_sb * b + a.d_sr * lane, x), mq, a.inv_tau) / sq;
      }
      ok = (double)a.u[(long)b * a.K + lane] * q < p;
    }
  }
  const unsigned long long bad = ~__builtin_amdgcn_ballot_w64(ok);
  return min(n, __builtin_ctzll(bad | (1ull << 63)));
}

// What is sampled from once `kept` are kept: the target row, and the draft row that is taken off (if any).
template <typename T>
struct Source {
  const T *p, *q;
  long long x;        // without draft logits: the token that is taken off, or -1
  float mp, mq;
  double ip, iq;      // 1 / sum
  __device__ __forceinline__ Source(const VerifyArgs& a, int b, int n, int kept) {
    double s;
    p = (const T*)a.target + a.t_sb * b + a.t_sr * kept;
    row_stats(a, b, kept, mp, s);
    ip = s > 0.0 ? 1.0 / s : 0.0;
    q = nullptr;
    x = -1;
    mq = 0.f;
    iq = 0.0;
    if (kept < n) {
      if (a.draft) {
        q = (const T*)a.draft + a.d_sb * b + a.d_sr * kept;
        row_stats(a, b, a.K + 1 + kept, mq, s);
        iq = s > 0.0 ? 1.0 / s : 0.0;
      } else {
        x = a.tokens[(long)b * a.K + kept];
      }
    }
  }
  // residual weight and the target's own
  __device__ __forceinline__ double operator()(const VerifyArgs& a, int c, double& own) const {
    own = weight(logit<T>(p, c), mp, a.inv_tau) * ip;
    if (q) return fmax(own - weight(logit<T>(q, c), mq, a.inv_tau) * iq, 0.0);
    return c == x ? 0.0 : own;
  }
};

// ---- launch 2: acceptance, and per piece the sums of the sampled weights (greedy: everything) ----
template <typename T>
__global__ __launch_bounds__(VT) void verify_accept_kernel(VerifyArgs a) {
  __shared__ double ss[VT / 64][2];
  __shared__ int s_kept;
  const int piece = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = drafted(a, b);
  if (wave == 0) {
    const int kept = accept<T>(a, b, n, lane);
    if (lane == 0) s_kept = kept;
  }
  __syncthreads();
  const int kept = s_kept;
  const Source<T> src(a, b, n, kept);
  double sr = 0.0, so = 0.0;
  for (int e = 0; e < VE; ++e) {
    const int c = piece * PIECE + e * VT + (int)threadIdx.x;
    if (c < a.V) {
      double own;
      sr += src(a, c, own);
      so += own;
    }
  }
  sr = wave_sum64(sr);
  so = wave_sum64(so);
  if (lane == 0) { ss[wave][0] = sr; ss[wave][1] = so; }
  __syncthreads();
  if (threadIdx.x == 0) {
    double* w = a.pw + ((long)b * a.pieces + piece) * 2;
    w[0] = (ss[0][0] + ss[1][0]) + (ss[2][0] + ss[3][0]);
    w[1] = (ss[0][1] + ss[1][1]) + (ss[2][1] + ss[3][1]);
    if (piece == 0) a.accepted[b] = kept;
  }
}

__device__ __forceinline__ void write_tokens(const VerifyArgs& a, int b, int kept, long long next) {
  for (int i = threadIdx.x; i <= a.K; i += blockDim.x)
    a.out[(long)b * (a.K + 1) + i] = i < kept ? a.tokens[(long)b * a.K + i] : i == kept ? next : -1;
}

__global__ __launch_bounds__(64) void verify_greedy_kernel(VerifyArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const int n = drafted(a, b);
  long long best = -1;
  bool ok = false;
  if (lane <= n) {
    const long o = ((long)b * (2 * a.K + 1) + lane) * a.pieces;
    float m = -INFINITY;
    for (int p = 0; p < a.pieces; ++p)
      if (a.pm[o + p] > m) { m = a.pm[o + p]; best = (long long)a.ps[o + p]; }
    ok = lane < n && best >= 0 && best == a.tokens[(long)b * a.K + lane];
  }
  const unsigned long long bad = ~__builtin_amdgcn_ballot_w64(ok);
  const int kept = min(n, __builtin_ctzll(bad | (1ull << 63)));
  const long long next = __shfl(best, kept, 64);
  write_tokens(a, b, kept, next);
  if (lane == 0) a.accepted[b] = kept;
}

// ---- launch 3: the piece that holds the border, and the token in it ----
template <typename T>
__global__ __launch_bounds__(VT) void verify_sample_kernel(VerifyArgs a) {
  __shared__ double part[VT];
  __shared__ int s_at, s_last;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int n = drafted(a, b), kept = a.accepted[b];
  const double* w = a.pw + (long)b * a.pieces * 2;
  double total = 0.0;
  for (int p = 0; p < a.pieces; ++p) total += w[2 * p];
  const int col = total > 0.0 ? 0 : 1;                    // nothing is left of p - q: the target's own distribution
  if (col) {
    total = 0.0;
    for (int p = 0; p < a.pieces; ++p) total += w[2 * p + 1];
  }
  if (!(total > 0.0)) {                                   // a row without a finite logit
    write_tokens(a, b, kept, -1);
    return;
  }
  const double border = (double)a.r[b] * total;
  int piece = -1;
  double before = 0.0;
  for (int p = 0; p < a.pieces; ++p) {
    const double x = w[2 * p + col];
    if (x > 0.0) {
      if (piece >= 0) before += w[2 * piece + col];       // the last piece with weight stays where rounding leaves none above the border
      piece = p;
      if (before + x > border) break;
    }
  }
  const Source<T> src(a, b, n, kept);
  const int c0 = piece * PIECE + tid * VE;                // here a thread holds 16 consecutive tokens
  double f[VE], sum = 0.0;
  for (int e = 0; e < VE; ++e) {
    f[e] = 0.0;
    if (c0 + e < a.V) {
      double own;
      const double res = src(a, c0 + e, own);
      f[e] = col ? own : res;
    }
    sum += f[e];
  }
  part[tid] = sum;
  if (tid == 0) { s_at = 0x7fffffff; s_last = -1; }
  __syncthreads();
  for (int d = 1; d < VT; d <<= 1) {                      // inclusive scan
    const double v = tid >= d ? part[tid - d] : 0.0;
    __syncthreads();
    part[tid] += v;
    __syncthreads();
  }
  double run = before + (tid ? part[tid - 1] : 0.0);
  int at = 0x7fffffff, last = -1;
  for (int e = 0; e < VE; ++e) {
    run += f[e];
    if (f[e] > 0.0) {
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
  hipLaunchKernelGGL((verify_rows_kernel<T>), dim3(a.pieces, rows, a.B), dim3(VT), 0, s, a);
  NEKO_CHECK_LAUNCH();
  if (a.greedy) {
    hipLaunchKernelGGL(verify_greedy_kernel, dim3(a.B), dim3(64), 0, s, a);
  } else {
    hipLaunchKernelGGL((verify_accept_kernel<T>), dim3(a.pieces, a.B), dim3(VT), 0, s, a);
    NEKO_CHECK_LAUNCH();
    hipLaunchKernelGGL((verify_sample_kernel<T>), dim3(a.B), dim3(VT), 0, s, a);
  }
  NEKO_CHECK_LAUNCH();
  return NEKO_OK;
}

}  // namespace

long neko_verify_draft_ws_bytes_impl(int B, int K, int V) {
  if (B <= 0 || K <= 0 || V <= 0) return 0;
  const long pieces = (V + PIECE - 1) / PIECE;
  return (long)B * pieces * ((2 * K + 1) * 12L + 16L) + 16;
}

int neko_verify_draft_impl(const void* target, long t_sb, long t_sr, const void* draft, long d_sb, long d_sr, int is_bf16, int B, int K, int V,
                           const long long* tokens, const float* u, const float* r, const int* n_draft, float temperature, int* accepted,
                           long long* out, void* ws, long ws_bytes, hipStream_t s) {
  if (!target || !tokens || !accepted || !out || !ws || B <= 0 || K <= 0 || V <= 0) return NEKO_ERR_ARG;
  if (!(temperature >= 0.f) || (temperature > 0.f && (!u || !r))) return NEKO_ERR_ARG;
  if (K > MAXK - 1 || B > 65535) return NEKO_ERR_UNSUPPORTED;
  if ((uintptr_t)ws & 7 || ws_bytes < neko_verify_draft_ws_bytes_impl(B, K, V)) return NEKO_ERR_ARG;
  VerifyArgs a{};
  a.target = target; a.draft = draft; a.t_sb = t_sb; a.t_sr = t_sr; a.d_sb = d_sb; a.d_sr = d_sr;
  a.tokens = tokens; a.u = u; a.r = r; a.n_draft = n_draft; a.accepted = accepted; a.out = out;
  a.B = B; a.K = K; a.V = V; a.pieces = (V + PIECE - 1) / PIECE;
  const long cells = (long)B * (2 * K + 1) * a.pieces;
  a.ps = (double*)ws;
  a.pw = a.ps + cells;
  a.pm = (float*)(a.pw + 2L * B * a.pieces);
  a.greedy = temperature == 0.f;
  a.inv_tau = a.greedy ? 1.0 : 1.0 / (double)temperature;
  return is_bf16 ? launch<bf16_t>(a, s) : launch<float>(a, s);
}
