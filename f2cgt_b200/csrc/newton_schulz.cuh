// What the Newton-Schulz kernels share (newton_schulz.cu, newton_schulz_small.cu).
#pragma once
#include "tcgen05.cuh"

namespace f2c {
namespace ns {

using namespace t5;

constexpr int kMaxList = 64;
constexpr int kScaleLog = 10;                // norms are brought to 2^10

// ---------------------------------------------------------------- what is read and written
struct Matrices {  // of one shape: a stack, or a list
  const void* g;
  void* out;              // the result; optimiser: the weights
  float* momentum;        // null: g is orthogonalised itself
  f2c_muon_matrix list[kMaxList];
  int listed;
  int64_t size;           // elements of a matrix
  float mu, keep, lr;     // w <- keep w - lr sqrt(max(1, rows / cols)) X
  int nesterov;
  template <typename T> __device__ __forceinline__ const T* grad(int z) const { return listed ? (const T*)list[z].grad : (const T*)g + z * size; }
  template <typename T> __device__ __forceinline__ T* result(int z) const { return listed ? (T*)list[z].weight : (T*)out + z * size; }
  __device__ __forceinline__ float gain(int64_t rows, int64_t cols) const { return lr * sqrtf(fmaxf(1.0f, (float)rows / (float)cols)); }
  __device__ __forceinline__ float* moment(int z) const { return listed ? list[z].momentum : nullptr; }
};

// Types whose matrices are held in pairs of half precision throughout (newton_schulz.cu).
template <typename T> constexpr bool is_wide = true;
template <> constexpr bool is_wide<__nv_bfloat16> = false;

// Factors of a step, for a matrix.
struct Factors {
  float gram, poly_b, poly_c, apply, own;  // As = gram Xs Xs^T; Rs = poly_c As^2 + poly_b As; the next Xs = own Xs + apply Rs Xs
};

struct Steps {
  int count;
  float co[3 * F2C_MAX_NS_STEPS];
  float top[F2C_MAX_NS_STEPS + 1];   // no singular value is larger in front of step t, if none was larger than one at first
  float factor[F2C_MAX_NS_STEPS];    // and none is multiplied by more
  float eps;
  uint32_t tries;                    // of a role's bounded waits; 0: no MMA or tensor copy is issued (product_kernel: and the waits run out)
};

__device__ __forceinline__ float power2(int e) { return __int_as_float((127 + min(max(e, -126), 127)) << 23); }
// 2^e is the smallest power that is not below v > 0 (v not subnormal)
__device__ __forceinline__ int log2_above(float v) {
  const uint32_t bits = __float_as_uint(v);
  return (int)(bits >> 23) - 127 + ((bits & 0x7fffffu) != 0u ? 1 : 0);
}

template <typename T, int V> struct alignas(V * sizeof(T)) Chunk { T v[V]; };

// u of V elements from i on
template <typename T, int V, bool UPDATE>
__device__ __forceinline__ void direction(const Matrices& s, int z, int64_t i, float (&u)[V]) {
  const Chunk<T, V> g = *reinterpret_cast<const Chunk<T, V>*>(s.template grad<T>(z) + i);
  float* momentum = s.moment(z);
  if (momentum == nullptr) {
#pragma unroll
    for (int e = 0; e < V; ++e) u[e] = to_float(g.v[e]);
    return;
  }
  Chunk<float, V> m = *reinterpret_cast<const Chunk<float, V>*>(momentum + i);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if (UPDATE) m.v[e] = fmaf(s.mu, m.v[e], to_float(g.v[e]));
    u[e] = s.nesterov ? fmaf(s.mu, m.v[e], to_float(g.v[e])) : m.v[e];
  }
  if (UPDATE) *reinterpret_cast<Chunk<float, V>*>(momentum + i) = m;
}

// Powers of two: X = u 2^up brings a norm to [2^10, 2^11).
__device__ __forceinline__ int scale_up(double norm) {
  if (!(norm <= 1e300 && norm > 0.0)) return kScaleLog + 1;
  const int e = (__double2hiint(norm) >> 20) - 1022;  // norm < 2^e
  return kScaleLog + 1 - e;
}

// The steps' factors for a matrix of that norm; without steps, `apply` of the first is the result's.
__device__ __forceinline__ void make_factors(const Steps& st, double norm, int up, Factors* table) {
  const double by = 1.0 / (norm + (double)st.eps);
  float kappa = (float)(by * __hiloint2double((1023 - up) << 20, 0));  // X = kappa Xs; 2^-up
  float bound = (float)(norm * by);
  for (int t = 0; t < st.count; ++t) {
    const float a = st.co[3 * t], b = st.co[3 * t + 1], c = st.co[3 * t + 2];
    const int lead = bound > 1e-37f && bound <= 64.0f ? log2_above(bound) : 0;
    const int a_log = min(kScaleLog - 2 * lead, 100);  // As = 2^a_log A
    Factors f;
    if (c != 0.0f) {
      f.gram = power2(a_log) * kappa * kappa;
      f.poly_b = b * power2(kScaleLog - a_log);
      f.poly_c = c * power2(kScaleLog - a_log) * power2(-a_log);
    } else {  // R itself
      f.gram = b * power2(kScaleLog) * kappa * kappa;
      f.poly_b = f.poly_c = 0.0f;
    }
    bound = fminf(st.top[t + 1], bound * st.factor[t]);
    const bool last = t + 1 == st.count;
    const float next = last ? 1.0f : power2((bound > 1e-37f && bound <= 64.0f ? log2_above(bound) : 0) - kScaleLog);
    f.apply = kappa * power2(-kScaleLog) / next;
    f.own = a * (kappa / next);
    kappa = next;
    table[t] = f;
  }
  if (st.count == 0) table[0].apply = kappa;
}

// Matrices of which the smaller side has up to 128 and the larger up to 256 elements, of any shapes (`list`, or a stack of rows x cols): one launch.
bool is_small(int64_t rows, int64_t cols);
int small(const char* op, const Matrices& s, int count, int64_t rows, int64_t cols, int dtype, const Steps& st, cudaStream_t stream);

}  // namespace ns
}  // namespace f2c
