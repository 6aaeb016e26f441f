// Newton-Schulz steps on stacks of matrices (f2c_orthogonalize) and the optimiser step around them (f2c_muon_step):
//   X = G / (|G|_F + eps);   A = X X^T,  B = a I + b A + c A^2,  X <- B X   for every step.
//
// Matrices with more rows than columns are worked on transposed.  Values, sums and norms in single precision, the norm's sum in double.
#include <math.h>

#include "common.cuh"

namespace f2c {
namespace ns {

constexpr int kThreads = 256, kTile = 64, kStep = 16, kParts = 64;

struct Source {     // what a matrix is read from, and what its result does
  const void* g;
  void* out;        // orthogonalize: the result; muon: the weights
  float* momentum;  // null: g is orthogonalised itself
  float mu, keep, gain;  // w <- keep w - gain X
  int nesterov;
};

// u of element i, and the momentum's update
template <typename T>
__device__ __forceinline__ float update(const Source& s, int64_t i) {
  const float g = to_float(((const T*)s.g)[i]);
  if (s.momentum == nullptr) return g;
  const float m = fmaf(s.mu, s.momentum[i], g);
  s.momentum[i] = m;
  return s.nesterov ? fmaf(s.mu, m, g) : m;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) load_kernel(const Source s, float* x, double* parts, int64_t rows, int64_t cols) {
  dependency_wait();
  release_dependents();
  const int64_t size = rows * cols, base = (int64_t)blockIdx.y * size;
  double sum = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < size; i += (int64_t)kParts * kThreads) {
    const float u = update<T>(s, base + i);
    sum += (double)u * u;
    x[base + (rows <= cols ? i : i % cols * rows + i / cols)] = u;
  }
  __shared__ double sums[kThreads];
  sums[threadIdx.x] = sum;
  __syncthreads();
  for (int o = kThreads / 2; o > 0; o >>= 1) {
    if (threadIdx.x < o) sums[threadIdx.x] += sums[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) parts[blockIdx.y * kParts + blockIdx.x] = sums[0];
}

__global__ void __launch_bounds__(kThreads) scale_kernel(float* x, const double* parts, int64_t size, float eps) {
  dependency_wait();
  release_dependents();
  double sum = 0.0;
  for (int i = 0; i < kParts; ++i) sum += parts[blockIdx.y * kParts + i];
  // a matrix that is not finite becomes NaN
  const float by = sum <= 1e300 ? (float)(1.0 / (sqrt(sum) + (double)eps)) : __int_as_float(0x7fffffff);
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < size; i += (int64_t)kParts * kThreads) x[blockIdx.y * size + i] *= by;
}

// D [p, q] = c L R + b C + a I with L [p, k] and R [k, q] (R given as [q, k] when turned)
__global__ void __launch_bounds__(kThreads) product_kernel(const float* l, const float* r, const float* add, float* d, int p, int q, int k, int turned,
                                                           float c, float b, float a) {
  dependency_wait();
  release_dependents();
  __shared__ float ls[kStep][kTile + 1], rs[kStep][kTile + 1];
  l += (int64_t)blockIdx.z * p * k;
  r += (int64_t)blockIdx.z * q * k;
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16, row0 = blockIdx.x * kTile, col0 = blockIdx.y * kTile;
  float acc[4][4] = {};
  for (int t0 = 0; t0 < k; t0 += kStep) {
    for (int e = tid; e < kTile * kStep; e += kThreads) {
      const int x = e / kStep, t = e % kStep, y = e % kTile, u = e / kTile;
      ls[t][x] = row0 + x < p && t0 + t < k ? l[(int64_t)(row0 + x) * k + t0 + t] : 0.0f;
      if (turned) rs[t][x] = col0 + x < q && t0 + t < k ? r[(int64_t)(col0 + x) * k + t0 + t] : 0.0f;
      else rs[u][y] = col0 + y < q && t0 + u < k ? r[(int64_t)(t0 + u) * q + col0 + y] : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kStep; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(ls[t][ty + 16 * i], rs[t][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int x = row0 + ty + 16 * i, y = col0 + tx + 16 * j;
      if (x >= p || y >= q) continue;
      const int64_t at = ((int64_t)blockIdx.z * p + x) * q + y;
      float v = c * acc[i][j];
      if (add != nullptr) v += b * add[at];
      d[at] = x == y ? v + a : v;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) store_kernel(const Source s, const float* x, int64_t rows, int64_t cols) {
  dependency_wait();
  release_dependents();
  const int64_t size = rows * cols, base = (int64_t)blockIdx.y * size;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < size; i += (int64_t)kParts * kThreads) {
    const float v = x[base + (rows <= cols ? i : i % cols * rows + i / cols)];
    T* o = (T*)s.out + base + i;
    *o = from_float<T>(s.momentum == nullptr ? v : s.keep * to_float(*o) - s.gain * v);
  }
}

static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

struct Shape {
  int64_t batch, rows, cols;
  int64_t p() const { return rows < cols ? rows : cols; }
  int64_t q() const { return rows < cols ? cols : rows; }
};

static int64_t workspace(const Shape& s) {
  return 2 * round256(4 * s.batch * s.rows * s.cols) + 2 * round256(4 * s.batch * s.p() * s.p()) + round256(8 * s.batch * kParts);
}

static int run(const char* op, const Source& src, int dtype, const Shape& s, const float* co, int steps, float eps, char* ws, cudaStream_t st) {
  float* x = (float*)ws;
  float* x2 = (float*)(ws += round256(4 * s.batch * s.rows * s.cols));
  float* a = (float*)(ws += round256(4 * s.batch * s.rows * s.cols));
  float* b = (float*)(ws += round256(4 * s.batch * s.p() * s.p()));
  double* parts = (double*)(ws + round256(4 * s.batch * s.p() * s.p()));
  const dim3 grid(kParts, (unsigned)s.batch);
  const int p = (int)s.p(), q = (int)s.q();
  auto* load = dtype == F2C_F32 ? load_kernel<float> : dtype == F2C_F16 ? load_kernel<__half> : load_kernel<__nv_bfloat16>;
  auto* store = dtype == F2C_F32 ? store_kernel<float> : dtype == F2C_F16 ? store_kernel<__half> : store_kernel<__nv_bfloat16>;
  launch_dependent(load, grid, kThreads, 0, st, src, x, parts, s.rows, s.cols);
  launch_dependent(scale_kernel, grid, kThreads, 0, st, x, (const double*)parts, s.rows * s.cols, eps);
  const unsigned tp = (unsigned)ceil_div(p, kTile), tq = (unsigned)ceil_div(q, kTile), z = (unsigned)s.batch;
  for (int t = 0; t < steps; ++t, co += 3) {
    launch_dependent(product_kernel, dim3(tp, tp, z), kThreads, 0, st, (const float*)x, (const float*)x, (const float*)nullptr, a, p, p, q, 1, 1.0f, 0.0f, 0.0f);
    launch_dependent(product_kernel, dim3(tp, tp, z), kThreads, 0, st, (const float*)a, (const float*)a, (const float*)a, b, p, p, p, 1, co[2], co[1], co[0]);
    launch_dependent(product_kernel, dim3(tp, tq, z), kThreads, 0, st, (const float*)b, (const float*)x, (const float*)nullptr, x2, p, q, p, 0, 1.0f, 0.0f, 0.0f);
    float* swap = x;
    x = x2;
    x2 = swap;
  }
  launch_dependent(store, grid, kThreads, 0, st, src, (const float*)x, s.rows, s.cols);
  return check_launch(op);
}

// Singular values start in [0, 1].  What keeps the half-precision operands in range: no step may take one out of [0, 7.9], nor multiply by more than 60.
static int check(const char* op, int dtype, const float* co, int steps, float eps) {
  F2C_REQUIRE(is_float_dtype(dtype), F2C_ERR_UNSUPPORTED, "%s: matrices must be float32, float16 or bfloat16", op);
  F2C_REQUIRE(steps >= 0 && steps <= F2C_MAX_NS_STEPS, F2C_ERR_LIMIT, "%s: 0 to %d steps", op, F2C_MAX_NS_STEPS);
  F2C_REQUIRE(steps == 0 || co, F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(eps >= 0.0f && eps <= 3.4028235e38f, F2C_ERR_INVALID, "%s: eps must not be negative", op);
  double top = 1.0;
  for (int t = 0; t < steps; ++t, co += 3) {
    double factor = 0.0, next = 0.0;
    for (int i = 0; i <= 1024; ++i) {
      const double v = top * i / 1024, f = fabs(co[0] + v * v * (co[1] + v * v * co[2]));
      if (!(f <= factor)) factor = f;
      if (!(v * f <= next)) next = v * f;
    }
    F2C_REQUIRE(factor <= 60.0 && next <= 7.9, F2C_ERR_LIMIT, "%s: the coefficients of step %d let the matrix grow too far", op, t);
    top = next;
  }
  return F2C_OK;
}

static int check_shape(const char* op, const Shape& s) {
  F2C_REQUIRE(s.batch >= 0 && s.rows >= 0 && s.cols >= 0, F2C_ERR_INVALID, "%s: negative size", op);
  F2C_REQUIRE(s.batch <= 65535 && s.rows <= 65536 && s.cols <= 65536, F2C_ERR_LIMIT, "%s: at most 65535 matrices of 65536 rows and columns", op);
  return F2C_OK;
}

}  // namespace ns
}  // namespace f2c

using namespace f2c;

extern "C" int64_t f2c_orthogonalize_workspace(int, int64_t batch, int64_t rows, int64_t cols) {
  return batch < 1 || rows < 1 || cols < 1 ? 0 : ns::workspace(ns::Shape{batch, rows, cols});
}

extern "C" int f2c_orthogonalize(const void* g, void* out, int dtype, int64_t batch, int64_t rows, int64_t cols, const float* coefficients_host,
                                 int steps, float eps, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "orthogonalize";
  const ns::Shape s{batch, rows, cols};
  if (const int rc = ns::check_shape(op, s)) return rc;
  if (const int rc = ns::check(op, dtype, coefficients_host, steps, eps)) return rc;
  if (batch == 0 || rows == 0 || cols == 0) return F2C_OK;
  F2C_REQUIRE(g && out, F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= ns::workspace(s), F2C_ERR_INVALID,
              "%s: workspace too small or not 256-byte aligned", op);
  return ns::run(op, ns::Source{g, out, nullptr, 0, 0, 0, 0}, dtype, s, coefficients_host, steps, eps, (char*)workspace, (cudaStream_t)stream);
}

extern "C" int64_t f2c_muon_workspace(const f2c_muon_matrix* list_host, int count, int) {
  int64_t most = 0;
  for (int i = 0; list_host != nullptr && i < count; ++i) {
    const ns::Shape s{1, list_host[i].rows, list_host[i].cols};
    if (s.rows < 1 || s.cols < 1) continue;
    const int64_t bytes = ns::workspace(s);
    most = bytes > most ? bytes : most;
  }
  return most;
}

extern "C" int f2c_muon_step(const f2c_muon_matrix* list_host, int count, int dtype, float lr, float momentum, int nesterov, float decay,
                             const float* coefficients_host, int steps, float eps, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "muon_step";
  F2C_REQUIRE(count >= 0 && (count == 0 || list_host), F2C_ERR_INVALID, "%s: bad list", op);
  if (const int rc = ns::check(op, dtype, coefficients_host, steps, eps)) return rc;
  for (int i = 0; i < count; ++i) {
    const f2c_muon_matrix& m = list_host[i];
    if (const int rc = ns::check_shape(op, ns::Shape{1, m.rows, m.cols})) return rc;
    F2C_REQUIRE(m.rows == 0 || m.cols == 0 || (m.weight && m.grad && m.momentum), F2C_ERR_INVALID, "%s: null pointer", op);
  }
  const int64_t need = f2c_muon_workspace(list_host, count, dtype);
  F2C_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), F2C_ERR_INVALID,
              "%s: workspace too small or not 256-byte aligned", op);
  for (int i = 0; i < count; ++i) {
    const f2c_muon_matrix& m = list_host[i];
    if (m.rows == 0 || m.cols == 0) continue;
    const double gain = (double)lr * sqrt(m.rows > m.cols ? (double)m.rows / (double)m.cols : 1.0);
    const ns::Source src{m.grad, m.weight, m.momentum, momentum, (float)(1.0 - (double)lr * decay), (float)gain, nesterov};
    if (const int rc = ns::run(op, src, dtype, ns::Shape{1, m.rows, m.cols}, coefficients_host, steps, eps, (char*)workspace, (cudaStream_t)stream)) return rc;
  }
  return F2C_OK;
}
