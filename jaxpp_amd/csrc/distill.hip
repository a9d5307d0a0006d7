// The loss of a student's logits against a teacher's top logits, and its gradient.
//
//   p = softmax(teacher / T) over the listed ids,  q = softmax(z / T) over the vocabulary
//   row_loss = w T^2 sum_k p_k (log p_k - log q_k),   dz = scale w T (q - p)
//
// HBM-bound: the logits are read, their gradient is written.  One workgroup per row: the running maximum and
// sum of the softmax in one pass over the row, q in a second (which finds the row in the caches); the few listed
// places are written last, each by one thread, so the sums do not depend on timing.
#include <math.h>

#include <algorithm>

#include "common.h"

namespace {

constexpr int kMaxListed = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DistillParams {
  const void* z;
  const int32_t* ids;
  const float* teacher;
  const float* weight;
  float* row_loss;
  void* dz;
  long ld, ldd;
  int vocab, k;
  float temperature, scale;
};

template <class E>
__device__ __forceinline__ float load1(const E* p) {
  if constexpr (sizeof(E) == 2) return bf16_to_f32(*p);
  else return *p;
}
template <class E>
__device__ __forceinline__ void store1(E* p, float v) {
  if constexpr (sizeof(E) == 2) *p = f32_to_bf16(v);
  else *p = v;
}
template <class E>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[16 / sizeof(E)]) {
  if constexpr (sizeof(E) == 2) {
    unpack8(v, f);
  } else {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
}
template <class E>
__device__ __forceinline__ uint4 pack(const float (&f)[16 / sizeof(E)]) {
  if constexpr (sizeof(E) == 2)
    return pack8(f);
  else
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

// over a workgroup of T threads; every thread gets the result.  `red`: T / 64 floats of LDS.
template <int T, class F>
__device__ __forceinline__ float reduce(float v, float* red, F&& f) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < T / 64; ++i) v = f(v, red[i]);
  return v;
}

// exp2((z - m) c): m is at least z, or -inf where every z so far is
__device__ __forceinline__ float weight_of(float z, float m, float c) {
  return z == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((z - m) * c);
}

template <class E, int T>
__global__ __launch_bounds__(T) void distill_kernel(DistillParams p) {
  constexpr int N = 16 / sizeof(E);
  __shared__ float red[T / 64], prob[kMaxListed], listed[kMaxListed];
  __shared__ int id[kMaxListed];
  const int tid = threadIdx.x;
  const long row = blockIdx.x;
  const E* z = (const E*)p.z + row * p.ld;
  E* dz = p.dz ? (E*)p.dz + row * p.ldd : nullptr;
  auto add = [](float a, float b) { return a + b; };
  auto most = [](float a, float b) { return fmaxf(a, b); };
  const float w = p.weight ? p.weight[row] : 1.f;
  const float c = kLog2e / p.temperature;

  // the teacher's side
  float tmax = -INFINITY;
  for (int k = tid; k < p.k; k += T) {
    const int at = p.ids[row * p.k + k];
    const bool in = at >= 0 && at < p.vocab;
    const float t = in ? p.teacher[row * p.k + k] : -INFINITY;
    id[k] = in ? at : -1;
    prob[k] = t;
    listed[k] = in ? load1(z + at) : 0.f;
    tmax = t > tmax || t != t ? t : tmax;
  }
  tmax = reduce<T>(tmax, red, most);
  float tsum = 0.f;
  for (int k = tid; k < p.k; k += T) tsum += weight_of(prob[k], tmax, c);
  tsum = reduce<T>(tsum, red, add);
  bool live = w != 0.f && tmax != -INFINITY;

  // the row from its first 16-byte boundary on: `head` elements before it, whole units, `tail` elements behind
  const int head = min((int)((16 - ((uintptr_t)z & 15)) & 15) / (int)sizeof(E), p.vocab);
  const int units = (p.vocab - head) / N, tail = p.vocab - head - units * N;
  const uint4* zu = (const uint4*)(z + head);
  const int edge = tid < head ? tid : tid - head < tail ? head + units * N + tid - head : -1;   // this thread's single element

  float m = -INFINITY, s = 0.f;
  if (live) {
    float ez = edge >= 0 ? load1(z + edge) : -INFINITY;
    m = ez;
    s = ez == -INFINITY ? 0.f : 1.f;
    for (int u = tid; u < units; u += T) {
      float f[N];
      unpack<E>(zu[u], f);
      float um = f[0];
#pragma unroll
      for (int e = 1; e < N; ++e) um = fmaxf(um, f[e]);
      if (um > m) {
        s *= weight_of(m, um, c);
        m = um;
      }
#pragma unroll
      for (int e = 0; e < N; ++e) s += weight_of(f[e], m, c);
    }
    const float all = reduce<T>(m, red, most);
    s = reduce<T>(s * weight_of(m, all, c), red, add);
    m = all;
    live = m != -INFINITY;
  }
  if (!live) {
    if (tid == 0) p.row_loss[row] = 0.f;
    if (dz)
      for (int i = tid; i < p.vocab; i += T) store1(dz + i, 0.f);
    return;
  }

  float loss = 0.f;
  for (int k = tid; k < p.k; k += T) {
    const float pk = weight_of(prob[k], tmax, c) / tsum;
    if (pk > 0.f || pk != pk) {
      const float lp = kLn2 * (c * (prob[k] - tmax) - log2f(tsum));
      loss += pk * (lp - kLn2 * (c * (listed[k] - m) - log2f(s)));
    }
  }
  loss = reduce<T>(loss, red, add);
  if (tid == 0) p.row_loss[row] = loss * (w * p.temperature * p.temperature);
  if (!dz) return;

  const float coef = p.scale * w * p.temperature, part = coef / s;
  const bool together = (((uintptr_t)dz - (uintptr_t)z) & 15) == 0;
  if (edge >= 0) store1(dz + edge, weight_of(load1(z + edge), m, c) * part);
  for (int u = tid; u < units; u += T) {
    float f[N];
    unpack<E>(zu[u], f);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = weight_of(f[e], m, c) * part;
    if (together) {
      ((uint4*)(dz + head))[u] = pack<E>(f);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) store1(dz + head + u * N + e, f[e]);
    }
  }
  __syncthreads();
  // the listed places: the first of an id's entries writes for all of them
  for (int k = tid; k < p.k; k += T) {
    if (id[k] < 0) continue;
    float pk = 0.f;
    bool first = true;
    for (int i = 0; i < p.k; ++i)
      if (id[i] == id[k]) {
        first = first && i >= k;
        pk += weight_of(prob[i], tmax, c) / tsum;
      }
    if (first) store1(dz + id[k], weight_of(listed[k], m, c) * part - coef * pk);
  }
}

__global__ __launch_bounds__(1024) void distill_sum_kernel(const float* row_loss, long rows, float scale, float* loss) {
  __shared__ float red[16];
  float s = 0.f;
  for (long i = threadIdx.x; i < rows; i += 1024) s += row_loss[i];
  s = reduce<1024>(s, red, [](float a, float b) { return a + b; });
  if (threadIdx.x == 0) *loss = s * scale;
}

template <class E>
void launch(hipStream_t st, const DistillParams& p, long rows) {
  if (p.vocab <= 8192)
    hipLaunchKernelGGL((distill_kernel<E, 256>), dim3((unsigned)rows), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((distill_kernel<E, 1024>), dim3((unsigned)rows), dim3(1024), 0, st, p);
}

}  // namespace

extern "C" int jpp_distill_loss(void* stream, const jpp_distill_args* a) {
  const char* who = "distill_loss";
  JPP_REQUIRE(a, "%s: null operand", who);
  JPP_REQUIRE(a->dtype == JPP_DTYPE_BF16 || a->dtype == JPP_DTYPE_F32, "%s: dtype %d", who, a->dtype);
  JPP_REQUIRE(a->rows >= 0 && a->rows < (1 << 22) && a->vocab > 0 && a->vocab < (int64_t)1 << 30, "%s: %lld x %lld logits", who,
              (long long)a->rows, (long long)a->vocab);
  JPP_REQUIRE(a->k >= 1 && a->k <= kMaxListed, "%s: k %d (1 to %d)", who, a->k, kMaxListed);
  JPP_REQUIRE(a->temperature > 0.f && isfinite(a->temperature) && isfinite(kLog2e / a->temperature),
              "%s: temperature %g", who, (double)a->temperature);
  hipStream_t st = (hipStream_t)stream;
  if (a->rows == 0) return a->loss ? jpp_fill_u32(a->loss, 0, 1, stream) : JPP_OK;
  JPP_REQUIRE(a->logits && a->ids && a->teacher && a->row_loss, "%s: null operand", who);
  JPP_REQUIRE(a->ld >= a->vocab && (!a->dlogits || a->ldd >= a->vocab), "%s: leading dimension too small", who);
  JPP_REQUIRE(((uintptr_t)a->logits | (uintptr_t)a->dlogits) % 16 == 0, "%s: logits and dlogits must be 16-byte aligned", who);
  JPP_REQUIRE(a->dlogits != a->logits || a->ldd == a->ld, "%s: dlogits over logits with another leading dimension", who);
  DistillParams p = {a->logits, a->ids, a->teacher, a->weight, a->row_loss, a->dlogits, (long)a->ld, (long)a->ldd,
                     (int)a->vocab, a->k, a->temperature, a->scale};
  const double n = (double)a->rows * a->vocab, es = a->dtype == JPP_DTYPE_F32 ? 4 : 2;
  ProbeScope probe(st, "distill_loss", 0, es * n * (a->dlogits ? 2 : 1));
  if (a->dtype == JPP_DTYPE_F32) launch<float>(st, p, a->rows);
  else launch<bf16_t>(st, p, a->rows);
  JPP_LAUNCH_CHECK();
  if (a->loss) {
    hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, st, a->row_loss, (long)a->rows, a->scale, a->loss);
    JPP_LAUNCH_CHECK();
  }
  return JPP_OK;
}
