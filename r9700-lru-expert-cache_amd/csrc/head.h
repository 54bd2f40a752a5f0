// The head's kernel for few rows (gemm_head.hip), launched also by the dense GEMM's entry point.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rlu {
namespace head {

// Waves that split K there, 0 where it does not take K.
int sk_of(int K);

// y [M, n] (rows ldy apart) = qx [M, K] x wq [n up to a multiple of 128, K]^T, sk_of(K) > 0. Above 64
// rows each launch row takes 64 of them and reads the weights again.
int rows(const uint8_t* qx, const float* xs, const uint8_t* wq, const float* ws, uint16_t* y,
         long long ldy, int M, int n, int K, hipStream_t st);

}  // namespace head
}  // namespace rlu
