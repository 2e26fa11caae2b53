// Distillation from a teacher's top logits: loss and gradient of every row in one pass over the student's logits.
//
//   t   = softmax over the row's k teacher logits / tau    (entries with an index outside [0, V) or a logit of -inf: none)
//   s   = softmax(z / tau) over the V student logits
//   loss_row = (1 - hard) tau^2 sum_j t_j (log t_j - log s[idx_j])  +  hard (logsumexp(z) - z[target])
//   dlogits  = weight [ (1 - hard) tau (s - sum_j t_j e_{idx_j})  +  hard (softmax(z) - e_target) ]          columns V .. Vpad-1: 0
//   weight == 0: loss 0, gradient 0.  A row without a teacher entry has no soft term, target < 0 no hard term.
//
// Bound by HBM: V logits in, V gradients out (the softmax needs the whole row before the first gradient, so the row stays in registers
// between the two: up to 1024 threads x 13 pieces of 16 B; longer rows are read again, from the last-level cache).  8192 rows of 52305 bf16 logits
// at two temperatures, a tenth of them of weight 0: 368 us, 1.63 GB at 4.4 TB/s (a copy reaches 5.2).  The k + 1 sparse places are
// written a second time behind the dense pass, with the dense term formed again from the logit that the thread kept: equal indices add up in
// registers (every holder writes the same sum), so no atomics and one rounding per element.  Sums are fp32 of positive terms: a thread adds its
// pieces' one after the other (13 pieces of 8 bf16: 104; of a row that is read again, as many as it has, 152 in 150000 bf16 logits), then six levels
// of lanes, then up to sixteen waves.  dlogits may be z.
#include "neko_kernels.h"

namespace {

constexpr int KMAX = 1024;

struct DistillArgs {
  const void* z;
  void* dz;
  long ldz, ldd;
  int V, Vpad, k;
  const float* t_val;
  const int* t_idx;
  const float* weight;
  const long long* target;
  float* loss_row;
  float tau, hard;
};

template <typename T> struct Piece;
template <> struct Piece<bf16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& r, float (&x)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[2 * e] = __uint_as_float(w[e] << 16); x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[8]) {
    return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
  // keeps the first `n` values (n < 8), the others become -inf
  static __device__ __forceinline__ uint4 mask(const uint4& r, int n) {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e >= n) w[e >> 1] = (e & 1) ? ((w[e >> 1] & 0x0000ffffu) | 0xff800000u) : ((w[e >> 1] & 0xffff0000u) | 0x0000ff80u);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // the largest bit pattern as a signed 16-bit integer, two values an instruction: the largest value if that is not negative
  struct Max {
    typedef __attribute__((ext_vector_type(2))) short s16x2;
    s16x2 v = {-32768, -32768};
    __device__ __forceinline__ void add(const uint4& r) {
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) v = __builtin_elementwise_max(v, __builtin_bit_cast(s16x2, w[e]));
    }
    __device__ __forceinline__ float value() const {                   // -1 where no value >= 0 was seen (a NaN of either sign stays one or is found later)
      const short x = v.x > v.y ? v.x : v.y;
      return x < 0 ? -1.0f : __uint_as_float((uint32_t)(unsigned short)x << 16);
    }
    static __device__ __forceinline__ bool is_exact(float m) { return !(m < 0.f); }
  };
  static __device__ __forceinline__ float one(const bf16_t* p) { return bf16_to_f32(*p); }
  static __device__ __forceinline__ bf16_t store(float x) { return f32_to_bf16(x); }
};
template <> struct Piece<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& r, float (&x)[4]) {
    x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
  static __device__ __forceinline__ uint4 mask(const uint4& r, int n) {
    const uint32_t ni = 0xff800000u;
    return make_uint4(n > 0 ? r.x : ni, n > 1 ? r.y : ni, n > 2 ? r.z : ni, ni);
  }
  struct Max {
    float v = -INFINITY;
    __device__ __forceinline__ void add(const uint4& r) {
      v = fmaxf(v, fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w))));
    }
    __device__ __forceinline__ float value() const { return v; }
    static __device__ __forceinline__ bool is_exact(float) { return true; }
  };
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ float store(float x) { return x; }
};

// NCH > 0: the row lives in NCH pieces per thread, as it came (unpacked again in every pass: an unpacked bf16 row would be twice the registers
// and half the workgroups per CU); 0: it is read again for every use.
// TWO: labels at temperature 1 beside a teacher at another, two exponentials per element and pass.  The factor of a gradient term is folded into
// its exponent (2^(c (x - m) + log2 of the factor); -inf for a term that the row does not have): per element 0.5-1 issue slots for the
// maximum, 8 (14 with TWO) for the sums, 8.5 (13.5) for the gradient, an exponential counting four.
// two workgroups of 1024 per CU where the row leaves room (64 registers): one loads while the other computes
template <typename T, int NT, int NCH, bool TWO>
__global__ __launch_bounds__(NT, NCH <= 7 ? 8 : NT == 512 ? 6 : 4) void distill_kernel(DistillArgs a) {
  using P = Piece<T>;
  constexpr int N = P::N, NW = NT / 64;
  constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
  __shared__ float red[3][NW];
  __shared__ int2 s_e[KMAX];                           // teacher entries: index (-1: none), probability
  __shared__ float s_z[KMAX];                          // the student's logit there
  __shared__ float s_teacher[2];                       // sum t log t; 1 if there is a teacher
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* z = (const T*)a.z + (long)row * a.ldz;
  T* dz = a.dz ? (T*)a.dz + (long)row * a.ldd : nullptr;
  const float w = a.weight[row];
  const int nch = a.Vpad / N;
  if (w == 0.f) {                                      // block-uniform
    if (tid == 0 && a.loss_row) a.loss_row[row] = 0.f;
    if (dz)
      for (int c = tid; c < nch; c += NT) reinterpret_cast<uint4*>(dz)[c] = make_uint4(0, 0, 0, 0);
    return;
  }
  const float soft_w = 1.0f - a.hard;
  const long long y = a.target ? a.target[row] : -1;
  const bool has_y = a.hard > 0.f && y >= 0 && y < a.V;

  // every load of the row is in flight before anything looks at one (clamped, unconditional)
  constexpr int NR = NCH > 0 ? NCH : 1;
  uint4 reg[NR];
  auto load = [&](int i) {                             // the piece of thread tid, round i; columns >= V are -inf
    const int c = tid + i * NT;
    uint4 r = reinterpret_cast<const uint4*>(z)[min(c, nch - 1)];
    return r;
  };
  const int full = a.V / (NT * N);                     // rounds without a column >= V (uniform)
  auto fence_cols = [&](int i, uint4 r) {
    const int c = tid + i * NT;
    if (i >= full && (c + 1) * N > a.V) r = P::mask(r, max(a.V - c * N, 0));
    return r;
  };
  if constexpr (NCH > 0) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) reg[i] = load(i);
  }
  auto keep_packed = [&]() {                           // without this the compiler keeps the unpacked values of the last pass
    if constexpr (NCH > 0) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) asm volatile("" : "+v"(reg[i].x), "+v"(reg[i].y), "+v"(reg[i].z), "+v"(reg[i].w));
    }
  };
  const int rounds = NCH > 0 ? NCH : (nch + NT - 1) / NT;
  // the student's logits at the teacher's entries and at the label, read before anything is overwritten
  const float zy = has_y ? P::one(z + y) : 0.f;
  if (soft_w != 0.f) {
#pragma unroll 1
    for (int j = tid; j < a.k; j += NT) {
      const int ix = a.t_idx[(long)row * a.k + j];
      s_z[j] = P::one(z + (ix >= 0 && ix < a.V ? ix : 0));
    }
  }

  // the teacher's entries (wave 0): index, probability
  if (soft_w != 0.f) {
    if (wave == 0) {
      const float it = 1.0f / a.tau;
      float tm = -INFINITY;
#pragma unroll 1
      for (int j = lane; j < a.k; j += 64) {
        const int ix = a.t_idx[(long)row * a.k + j];
        const float v = ix >= 0 && ix < a.V ? a.t_val[(long)row * a.k + j] : -INFINITY;
        s_e[j] = make_int2(v == -INFINITY ? -1 : ix, __float_as_int(v));
        tm = fmaxf(tm, v);
      }
      tm = wave_max(tm);
      const bool any = tm != -INFINITY;
      float ts = 0.f;
#pragma unroll 1
      for (int j = lane; j < a.k; j += 64)
        if (s_e[j].x >= 0) ts += __expf((__int_as_float(s_e[j].y) - tm) * it);
      ts = wave_sum(ts);
      const float inv = any ? 1.0f / ts : 0.f, lts = logf(ts);
      float acc = 0.f;
#pragma unroll 1
      for (int j = lane; j < a.k; j += 64) {
        float t = 0.f;
        if (s_e[j].x >= 0) {
          const float lt = (__int_as_float(s_e[j].y) - tm) * it;
          t = __expf(lt) * inv;
          if (t > 0.f) acc += t * (lt - lts);          // sum t log t
        }
        s_e[j].y = __float_as_int(t);
      }
      acc = wave_sum(acc);
      if (lane == 0) { s_teacher[0] = acc; s_teacher[1] = any ? 1.f : 0.f; }
    }
  } else if (tid == 0) {
    s_teacher[0] = 0.f;
    s_teacher[1] = 0.f;
  }

  // maximum
  typename P::Max mx;
#pragma unroll
  for (int i = 0; i < rounds; ++i) {
    if constexpr (NCH > 0) { reg[i] = fence_cols(i, reg[i]); mx.add(reg[i]); }
    else mx.add(fence_cols(i, load(i)));
  }
  float m = wave_max(mx.value());
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
  m = red[0][0];
#pragma unroll
  for (int i = 1; i < NW; ++i) m = fmaxf(m, red[0][i]);
  if (!P::Max::is_exact(m)) {                          // bf16, no value >= 0 in the row: its largest by value
    __syncthreads();
    m = -INFINITY;
#pragma unroll 1
    for (int i = 0; i < rounds; ++i) {
      float x[N];
      P::get(fence_cols(i, load(i)), x);
#pragma unroll
      for (int e = 0; e < N; ++e) m = fmaxf(m, x[e]);
    }
    m = wave_max(m);
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = red[0][0];
#pragma unroll
    for (int i = 1; i < NW; ++i) m = fmaxf(m, red[0][i]);
  }

  // sums: c1 serves the teacher's temperature (and the labels where that is 1 or there is no teacher), LOG2E the labels' with TWO
  const bool soft = soft_w != 0.f && s_teacher[1] != 0.f;
  const float c1 = soft_w != 0.f ? LOG2E / a.tau : LOG2E;
  // exponents are (x - m) c: exactly 0 for the maximum, whatever its size (c x - c m in one multiply-add is off by the rounding of c m, which a row
  // of the type's lowest values or a tiny tau makes larger than any exponent fp32 can hold)
  float s1 = 0.f, s2 = 0.f;
  keep_packed();
#pragma unroll
  for (int i = 0; i < rounds; ++i) {
    float x[N];
    if constexpr (NCH > 0) P::get(reg[i], x);
    else P::get(fence_cols(i, load(i)), x);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = x[e] - m;
      s1 += __builtin_amdgcn_exp2f(d * c1);
      if (TWO) s2 += __builtin_amdgcn_exp2f(d * LOG2E);
    }
  }
  s1 = wave_sum(s1);
  if (TWO) s2 = wave_sum(s2);
  if (lane == 0) { red[1][wave] = s1; red[2][wave] = s2; }
  __syncthreads();
  s1 = s2 = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) { s1 += red[1][i]; s2 += red[2][i]; }
  const float sum_soft = s1, sum_hard = TWO ? s2 : s1;
  const float fs = soft ? soft_w * a.tau / sum_soft : 0.f, fh = has_y ? a.hard / sum_hard : 0.f;

  if (wave == 0 && a.loss_row) {
    float acc = 0.f;
    if (soft)
#pragma unroll 1
      for (int j = lane; j < a.k; j += 64) {
        const float t = __int_as_float(s_e[j].y);
        if (t > 0.f) acc += t * (s_z[j] - m);
      }
    acc = wave_sum(acc);
    if (lane == 0) {
      float loss = 0.f;
      // tau^2 (sum t log t + log sum - sum t (z - m) / tau), with one tau multiplied through: neither tau^2 nor (z - m) / tau is formed, which a
      // small tau takes out of fp32
      if (soft) loss += soft_w * a.tau * (a.tau * (s_teacher[0] + LN2 * log2f(sum_soft)) - acc);
      if (has_y) loss += a.hard * LN2 * (log2f(sum_hard) - (zy - m) * (TWO ? LOG2E : c1));
      a.loss_row[row] = loss;
    }
  }
  if (!dz) return;
  keep_packed();
  // bf16 results: the factor of a term goes into its exponent, the sign of the weight into the packing.  fp32 results multiply (an exponent of 40
  // is held to 2^-19 only)
  constexpr bool FOLD = sizeof(T) == 2;
  const float f1 = w * (TWO ? fs : fs + fh), f2 = w * fh;
  const float e1 = __log2f(fabsf(f1)), e2 = __log2f(fabsf(f2));
  const bool neg = FOLD && w < 0.f;
#pragma unroll
  for (int i = 0; i < rounds; ++i) {
    const int c = tid + i * NT;
    float x[N];
    if constexpr (NCH > 0) P::get(reg[i], x);
    else P::get(fence_cols(i, load(i)), x);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = x[e] - m;
      float g = __builtin_amdgcn_exp2f(FOLD ? fmaf(d, c1, e1) : d * c1);
      if (!FOLD) g *= f1;
      if (TWO) {
        const float g2 = __builtin_amdgcn_exp2f(FOLD ? fmaf(d, LOG2E, e2) : d * LOG2E);
        g = FOLD ? g + g2 : fmaf(g2, f2, g);
      }
      x[e] = g;
    }
    if (neg) {
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = -x[e];
    }
    if (c < nch) {
      typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_v;
      const uint4 o = P::put(x);
      __builtin_nontemporal_store((u32x4_v){o.x, o.y, o.z, o.w}, reinterpret_cast<u32x4_v*>(dz) + c);
    }
  }
  // the sparse results replace the dense ones: the dense terms once more, minus everything the teacher and the label have at this place
  auto sparse = [&](int c, float x) {
    float t = 0.f, g = 0.f;
    if (soft) {
#pragma unroll 4
      for (int i = 0; i < a.k; ++i) {
        const int2 e = s_e[i];
        t += e.x == c ? __int_as_float(e.y) : 0.f;
      }
      g += w * (fs * __builtin_amdgcn_exp2f((x - m) * c1) - soft_w * a.tau * t);
    }
    if (has_y) g += w * (fh * __builtin_amdgcn_exp2f((x - m) * (TWO ? LOG2E : c1)) - (c == (int)y ? a.hard : 0.f));
    return P::store(g);
  };
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // the dense values are written: a store behind the barrier to the same place comes second
  __syncthreads();
  if (soft) {
#pragma unroll 1
    for (int j = tid; j < a.k; j += NT)
      if (s_e[j].x >= 0) dz[s_e[j].x] = sparse(s_e[j].x, s_z[j]);
  }
  if (has_y && tid == NT - 1) dz[y] = sparse((int)y, zy);
}

// Threads and rounds (pieces of 16 B a thread) by the pieces of a row: as many rounds as the row has, or little more -- a round computes whether the
// row reaches it or not (a test per round cost more: it kept the rounds from overlapping) -- and workgroups as small as the registers allow, so that
// several rows per CU fill each other's gaps.  A few of the variants at two temperatures in bf16 (512 threads, 11 to 14 rounds) keep 2 to 11 registers
// in scratch (12-40 B a lane; one temperature, 1024 x 7: 2), and still are the fastest for their rows.  Measured in bf16 | fp32, us (in and out 0.37 | 0.37 GB at 700
// pieces, 0.68 | 0.68 at 1300, 1.07 | 1.57 at 3000, 1.07 | 2.15 above):
//   700 pieces:  256 threads 76 | 73, 512 threads 112 | 98          1300: 512 x 4 155 | 136, 1024 x 4 276 | 234        3000: 512 x 6 193 | 303, 1024 x 4 227 | 316
//   5000: 1024 x 5 190 | 379, 512 x 10 200 | 397; at two temperatures in bf16, where registers for two rows more pay, 512 x 10 211, 1024 x 5 214
//   6544: 1024 x 7 194 | 372, 512 x 13 206 | 401; two temperatures in bf16 512 x 13 234, 1024 x 7 247
//   8000: 1024 x 8 283 | 462, read again 302 | 564               13000: 1024 x 13 254 | 395, read again 313 | 591
template <typename T, bool TWO>
void start(const DistillArgs& a, int R, int nch, hipStream_t s) {
#define NEKO_DISTILL(NT, NCH)                                                                     \
  {                                                                                               \
    hipLaunchKernelGGL((distill_kernel<T, NT, NCH, TWO>), dim3(R), dim3(NT), 0, s, a);            \
    return;                                                                                       \
  }
  if (nch <= 256) NEKO_DISTILL(256, 1)
  if (nch <= 2 * 256) NEKO_DISTILL(256, 2)
  if (nch <= 4 * 256) NEKO_DISTILL(256, 4)
  if (nch <= 4 * 512) NEKO_DISTILL(512, 4)
  if (nch <= 6 * 512) NEKO_DISTILL(512, 6)
  if constexpr (TWO && sizeof(T) == 2) {
    if (nch <= 8 * 512) NEKO_DISTILL(512, 8)
    if (nch <= 9 * 512) NEKO_DISTILL(512, 9)
    if (nch <= 10 * 512) NEKO_DISTILL(512, 10)
    if (nch <= 11 * 512) NEKO_DISTILL(512, 11)
    if (nch <= 12 * 512) NEKO_DISTILL(512, 12)
    if (nch <= 13 * 512) NEKO_DISTILL(512, 13)
    if (nch <= 14 * 512) NEKO_DISTILL(512, 14)
  } else {
    if (nch <= 4 * 1024) NEKO_DISTILL(1024, 4)
    if (nch <= 5 * 1024) NEKO_DISTILL(1024, 5)
    if (nch <= 6 * 1024) NEKO_DISTILL(1024, 6)
    if (nch <= 7 * 1024) NEKO_DISTILL(1024, 7)
  }
  if (nch <= 8 * 1024) NEKO_DISTILL(1024, 8)
  if (nch <= 9 * 1024) NEKO_DISTILL(1024, 9)
  if (nch <= 11 * 1024) NEKO_DISTILL(1024, 11)
  if (nch <= 13 * 1024) NEKO_DISTILL(1024, 13)
  NEKO_DISTILL(1024, 0)
#undef NEKO_DISTILL
}

template <typename T>
int launch(const DistillArgs& a, int R, hipStream_t s) {
  const int nch = a.Vpad / Piece<T>::N;
  if (a.hard > 0.f && a.hard < 1.f && a.tau != 1.0f) start<T, true>(a, R, nch, s);
  else start<T, false>(a, R, nch, s);
  NEKO_CHECK_LAUNCH();
  return NEKO_OK;
}

}  // namespace

int neko_distill_topk_impl(const void* z, long ldz, int is_bf16, int R, int V, int Vpad, const float* t_val, const int* t_idx, int k, const float* weight,
                           float tau, const long long* target, float hard, float* loss_row, void* dlogits, long ldd, hipStream_t s) {
  if (!z || !weight || R <= 0 || V <= 0 || Vpad < V || (!loss_row && !dlogits)) return NEKO_ERR_ARG;
  if (!(tau >= 1.17549435e-38f && tau <= 3.402823466e38f) || !(hard >= 0.f && hard <= 1.f) || (hard > 0.f && !target) || (hard < 1.f && (!t_val || !t_idx || k <= 0))) return NEKO_ERR_ARG;
  if (k > KMAX || Vpad > (1 << 30)) return NEKO_ERR_UNSUPPORTED;        // (columns and a workgroup's width add up in 32 bits)
  const int n = is_bf16 ? 8 : 4;
  if (Vpad % n || ldz % n || ldz < Vpad || (uintptr_t)z & 15) return NEKO_ERR_ARG;
  if (dlogits && (ldd % n || ldd < Vpad || (uintptr_t)dlogits & 15)) return NEKO_ERR_ARG;
  const long width = (long)Vpad * (is_bf16 ? 2 : 4), size = is_bf16 ? 2 : 4;
  if (dlogits && neko_rows_shared(z, ldz * size, 0, dlogits, ldd * size, 0, width, R, 1)) return NEKO_ERR_ARG;
  DistillArgs a{z, dlogits, ldz, ldd, V, Vpad, k, t_val, t_idx, weight, target, loss_row, tau, hard};
  return is_bf16 ? launch<bf16_t>(a, R, s) : launch<float>(a, R, s);
}
