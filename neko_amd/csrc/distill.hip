// Distillation from a teacher's top logits: loss and gradient of every row in one pass over the student's logits.
//
//   t   = softmax over the row's k teacher logits / tau    (entries with an index outside [0, V) or a logit of -inf: none)
//   s   = softmax(z / tau) over the V student logits
//   loss_row = (1 - hard) tau^2 sum_j t_j (log t_j - log s[idx_j])  +  hard (logsumexp(z) - z[target])
//   dlogits  = weight [ (1 - hard) tau (s - sum_j t_j e_{idx_j})  +  hard (softmax(z) - e_target) ]          columns V .. Vpad-1: 0
//   weight == 0: loss 0, gradient 0.  A row without a teacher entry has no soft term, target < 0 no hard term.
//
// Bound by HBM: V logits in, V gradients out (the softmax needs the whole row before the first gradient, so the row stays in registers
// between the two: 1024 threads x up to 16 pieces of 16 B; longer rows are read again, from the last-level cache).  The k + 1 sparse places are
// written a second time behind the dense pass, with the dense term formed again from the logit that the thread kept: equal indices add up in
// registers (every holder writes the same sum), so no atomics and one rounding per element.  Sums are fp32 of at most 52 K positive terms in
// a tree (a thread's 56, then lanes, then waves).  dlogits may be z.
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
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ float store(float x) { return x; }
};

// NCH > 0: the row lives in NCH pieces per thread; 0: it is read again for every use
template <typename T, int NT, int NCH>
__global__ __launch_bounds__(NT) void distill_kernel(DistillArgs a) {
  using P = Piece<T>;
  constexpr int N = P::N, NW = NT / 64;
  constexpr float LOG2E = 1.44269504088896340736f;
  __shared__ float red[3][NW];
  __shared__ float s_t[KMAX];
  __shared__ int s_i[KMAX];
  __shared__ float s_teacher[2];                       // soft loss without the student's normaliser; 1 if there is a teacher
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
  if constexpr (NCH > 0) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) reg[i] = reinterpret_cast<const uint4*>(z)[min(tid + i * NT, nch - 1)];
  }
  // between the passes the row stays packed: without this the compiler keeps every unpacked value instead (twice the registers, spills)
  auto keep_packed = [&]() {
    if constexpr (NCH > 0) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) asm volatile("" : "+v"(reg[i].x), "+v"(reg[i].y), "+v"(reg[i].z), "+v"(reg[i].w));
    }
  };
  // the piece of thread tid, round i, as fp32; columns >= V are -inf
  auto piece = [&](int i, float (&x)[N]) {
    const int c = tid + i * NT;
    P::get(NCH > 0 ? reg[NCH > 0 ? i : 0] : reinterpret_cast<const uint4*>(z)[min(c, nch - 1)], x);
    if ((c + 1) * N > a.V) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (c * N + e >= a.V) x[e] = -INFINITY;
    }
  };
  const int rounds = NCH > 0 ? NCH : (nch + NT - 1) / NT;

  // the teacher's entries (wave 0): index, probability, and the student's logit there, read before anything is overwritten
  if (soft_w != 0.f) {
    if (wave == 0) {
      const float it = 1.0f / a.tau;
      float tm = -INFINITY;
      for (int j = lane; j < a.k; j += 64) {
        const int ix = a.t_idx[(long)row * a.k + j];
        const float v = ix >= 0 && ix < a.V ? a.t_val[(long)row * a.k + j] : -INFINITY;
        s_i[j] = v == -INFINITY ? -1 : ix;
        s_t[j] = v;
        tm = fmaxf(tm, v);
      }
      tm = wave_max(tm);
      const bool any = tm != -INFINITY;
      float ts = 0.f;
      for (int j = lane; j < a.k; j += 64)
        if (s_i[j] >= 0) ts += __expf((s_t[j] - tm) * it);
      ts = wave_sum(ts);
      const float inv = any ? 1.0f / ts : 0.f, lts = logf(ts);
      float acc = 0.f;
      for (int j = lane; j < a.k; j += 64) {
        float t = 0.f;
        if (s_i[j] >= 0) {
          const float lt = (s_t[j] - tm) * it;
          t = __expf(lt) * inv;
          if (t > 0.f) acc += t * (lt - lts);          // sum t log t
        }
        s_t[j] = t;
      }
      acc = wave_sum(acc);
      if (lane == 0) { s_teacher[0] = acc; s_teacher[1] = any ? 1.f : 0.f; }
    }
  } else if (tid == 0) {
    s_teacher[0] = 0.f;
    s_teacher[1] = 0.f;
  }

  // maximum
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < rounds; ++i) {
    float x[N];
    piece(i, x);
#pragma unroll
    for (int e = 0; e < N; ++e) m = fmaxf(m, x[e]);
  }
  m = wave_max(m);
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
  m = red[0][0];
#pragma unroll
  for (int i = 1; i < NW; ++i) m = fmaxf(m, red[0][i]);

  // sums, at the temperature and (for the labels) without it
  const bool soft = soft_w != 0.f && s_teacher[1] != 0.f;
  const float c_soft = LOG2E / a.tau;
  const bool two = has_y && a.tau != 1.0f && soft;
  const float c_one = soft ? c_soft : LOG2E;
  float s1 = 0.f, s2 = 0.f;
  keep_packed();
#pragma unroll
  for (int i = 0; i < rounds; ++i) {
    float x[N];
    piece(i, x);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = x[e] - m;
      s1 += __builtin_amdgcn_exp2f(d * c_one);
      if (two) s2 += __builtin_amdgcn_exp2f(d * LOG2E);
    }
  }
  s1 = wave_sum(s1);
  if (two) s2 = wave_sum(s2);
  if (lane == 0) { red[1][wave] = s1; red[2][wave] = s2; }
  // the sparse places of this thread: teacher entries, then the label
  __syncthreads();
  s1 = s2 = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) { s1 += red[1][i]; s2 += red[2][i]; }
  const float sum_soft = s1, sum_hard = two ? s2 : s1;
  const float gs = soft ? w * soft_w * a.tau / sum_soft : 0.f;      // dense terms: gs 2^(c_soft d) + gh 2^(LOG2E d)
  const float gh = has_y ? w * a.hard / sum_hard : 0.f;

  if (wave == 0 && a.loss_row) {
    float acc = 0.f;
    if (soft)
      for (int j = lane; j < a.k; j += 64)
        if (s_t[j] > 0.f) acc += s_t[j] * (P::one(z + s_i[j]) - m);
    acc = wave_sum(acc);
    if (lane == 0) {
      float loss = 0.f;
      if (soft) loss += soft_w * a.tau * a.tau * (s_teacher[0] - acc / a.tau + logf(sum_soft));
      if (has_y) loss += a.hard * (logf(sum_hard) - (P::one(z + y) - m));
      a.loss_row[row] = loss;
    }
  }
  if (!dz) return;
  // this thread's sparse results (their logits are read before the dense pass overwrites them in place)
  constexpr int MAXJ = (KMAX + NT) / NT;               // k + 1 entries over NT threads
  float fix[MAXJ];
  int at[MAXJ];
#pragma unroll
  for (int q = 0; q < MAXJ; ++q) {
    const int j = tid + q * NT;
    at[q] = -1;
    fix[q] = 0.f;
    if (j < a.k && soft) at[q] = s_i[j];
    if (j == a.k && has_y) at[q] = (int)y;
    if (at[q] >= 0) {
      const float d = P::one(z + at[q]) - m;
      float t = 0.f;
      if (soft)
        for (int i = 0; i < a.k; ++i) t += s_i[i] == at[q] ? s_t[i] : 0.f;
      float g = 0.f;
      if (soft) g += w * soft_w * a.tau * (__builtin_amdgcn_exp2f(d * c_soft) / sum_soft - t);
      if (has_y) g += w * a.hard * (__builtin_amdgcn_exp2f(d * LOG2E) / sum_hard - (at[q] == (int)y ? 1.f : 0.f));
      fix[q] = g;
    }
  }
  __syncthreads();                                      // every sparse logit is read
  keep_packed();
#pragma unroll
  for (int i = 0; i < rounds; ++i) {
    const int c = tid + i * NT;
    float x[N];
    piece(i, x);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = x[e] - m;
      float g = 0.f;
      if (soft && has_y && !two) g = __builtin_amdgcn_exp2f(d * LOG2E) * (gs + gh);       // one temperature: one exponential
      else {
        if (soft) g = __builtin_amdgcn_exp2f(d * c_soft) * gs;
        if (has_y) g = fmaf(__builtin_amdgcn_exp2f(d * LOG2E), gh, g);
      }
      x[e] = c * N + e < a.V ? g : 0.f;
    }
    if (c < nch) reinterpret_cast<uint4*>(dz)[c] = P::put(x);
  }
  __syncthreads();                                      // the dense values are written
#pragma unroll
  for (int q = 0; q < MAXJ; ++q)
    if (at[q] >= 0) dz[at[q]] = P::store(fix[q]);
}

template <typename T>
int launch(const DistillArgs& a, int R, hipStream_t s) {
  const int nch = a.Vpad / Piece<T>::N;
#define NEKO_DISTILL(NT, NCH) hipLaunchKernelGGL((distill_kernel<T, NT, NCH>), dim3(R), dim3(NT), 0, s, a)
  if (nch <= 256) NEKO_DISTILL(256, 1);                 // short vocabularies: small workgroups, several rows per CU
  else if (nch <= 1024) NEKO_DISTILL(256, 4);
  else if (nch <= 4 * 1024) NEKO_DISTILL(1024, 4);
  else if (nch <= 7 * 1024) NEKO_DISTILL(1024, 7);
  else if (nch <= 13 * 1024) NEKO_DISTILL(1024, 13);
  else NEKO_DISTILL(1024, 0);
#undef NEKO_DISTILL
  NEKO_CHECK_LAUNCH();
  return NEKO_OK;
}

}  // namespace

int neko_distill_topk_impl(const void* z, long ldz, int is_bf16, int R, int V, int Vpad, const float* t_val, const int* t_idx, int k, const float* weight,
                           float tau, const long long* target, float hard, float* loss_row, void* dlogits, long ldd, hipStream_t s) {
  if (!z || !weight || R <= 0 || V <= 0 || Vpad < V || (!loss_row && !dlogits)) return NEKO_ERR_ARG;
  if (!(tau > 0.f) || !(hard >= 0.f && hard <= 1.f) || (hard > 0.f && !target) || (hard < 1.f && (!t_val || !t_idx || k <= 0))) return NEKO_ERR_ARG;
  if (k > KMAX) return NEKO_ERR_UNSUPPORTED;
  const int n = is_bf16 ? 8 : 4;
  if (Vpad % n || ldz % n || ldz < Vpad || (uintptr_t)z & 15) return NEKO_ERR_ARG;
  if (dlogits && (ldd % n || ldd < Vpad || (uintptr_t)dlogits & 15)) return NEKO_ERR_ARG;
  DistillArgs a{z, dlogits, ldz, ldd, V, Vpad, k, t_val, t_idx, weight, target, loss_row, tau, hard};
  return is_bf16 ? launch<bf16_t>(a, R, s) : launch<float>(a, R, s);
}
