// What the 8-bit products share between their files (int8_quantize.cu, int8_mm.cu).
#pragma once
#include "common.cuh"

namespace f2c {
namespace i8 {

constexpr int kMaxK = 131071;                 // 128 * 128 * k stays below 2^31: the int32 sum is exact
constexpr int64_t kMaxRows = (1ll << 31) - 4096;

// Rows in floating point: the columns of x1, then those of x2.
struct Rows {
  const void *x1, *x2;
  int64_t ld1, ld2, k1, k2, m;
  int dtype;
};

int check_rows(const char* op, const Rows& r);
int quantize(const Rows& r, int8_t* codes, int64_t ldq, float* scales, cudaStream_t st);

}  // namespace i8
}  // namespace f2c
