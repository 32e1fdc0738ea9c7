// Quantisation of activations token by token (RockQuantizeParams in kernel_params.h): every row becomes int8 with one
// scale of its own, the form rock_token_gemm_i8_* takes its first operand in.
//
//   top = max_k |x_k| ;  scale = top / 127 ;  q_k = roundeven(127 x_k / top)
//
// A row is read once: its 16-byte pieces stay in registers between the maximum and the rounding (up to eight per lane;
// longer rows are read again, from L2).  One wave per row, or the four waves of a block where the rows are few or long.
// Bound by HBM: 24576 x 4096 f16 in 57.8 us, 302 MB at 5.2 TB/s (a copy reaches 5.05); one row of 4096 takes 3.2 us.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "kernel_params.h"
#include "mfma_gfx950.h"

#ifndef ROCK_KERNEL
#define ROCK_KERNEL -1
#endif
#define RK_SELECTED(n) (ROCK_KERNEL < 0 || ROCK_KERNEL == (n))

namespace rkq {

typedef uint16_t v2us __attribute__((ext_vector_type(2)));
constexpr int kPieces = 8;

template <int DT> struct Piece { // 16 bytes of a row
  static constexpr int ES = DT == ROCK_F32 ? 4 : 2, N = 16 / ES;
};

// piece number c of a row, elements behind its end as zeros; rows may start at any multiple of the element size
template <int DT> __device__ __forceinline__ v4i load_piece(const char *row, int c, int cols) {
  constexpr int ES = Piece<DT>::ES, N = Piece<DT>::N;
  v4i v = {0, 0, 0, 0};
  const int left = cols - c * N;
  if (left >= N) {
    __builtin_memcpy(&v, row + (int64_t)c * 16, 16);
  } else if (left > 0) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < left) {
        if constexpr (ES == 4)
          v[e] = ((const int *)row)[c * N + e];
        else
          v[e >> 1] |= (int)((uint32_t)((const uint16_t *)row)[c * N + e] << (16 * (e & 1)));
      }
  }
  return v;
}

// The largest magnitude, as bits of the element type: ordered like the values, an infinity and a NaN above all of them.
// 16-bit types keep two running maxima in one register.
template <int DT> __device__ __forceinline__ uint32_t max_bits(uint32_t top, const v4i &v) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int word = v[d];
    if constexpr (DT == ROCK_F32) {
      top = max(top, (uint32_t)word & 0x7fffffffu);
    } else {
      const v2us a = __builtin_bit_cast(v2us, (uint32_t)word & 0x7fff7fffu), b = __builtin_bit_cast(v2us, top);
      top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(a, b));
    }
  }
  return top;
}
template <int DT> __device__ __forceinline__ float widen_bits(uint32_t bits) {
  if constexpr (DT == ROCK_F32)
    return __builtin_bit_cast(float, bits);
  else if constexpr (DT == ROCK_BF16)
    return __builtin_bit_cast(float, bits << 16);
  else
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}
template <int DT> __device__ __forceinline__ float element(const v4i &v, int e) {
  const int word = v[DT == ROCK_F32 ? e : e >> 1];
  if constexpr (DT == ROCK_F32)
    return __builtin_bit_cast(float, word);
  else
    return widen_bits<DT>(((uint32_t)word >> (16 * (e & 1))) & 0xffffu);
}

// roundeven(127 x / top).  x * (127 / top) in f32 is off by less than 2e-5, so only a value within 1e-4 of a half is
// rounded from the quotient itself, in 64 bits (where 127 x is exact and a quotient of 31 by 24 bits that is not a
// half is further from it than the rounding).  `exact`: 127 / top is not a usable f32.
template <int DT> __device__ __forceinline__ void quantize_piece(const v4i &v, float top, float inv, bool exact,
                                                                 uint32_t (&out)[2]) {
  constexpr int N = Piece<DT>::N;
  float q[N], near = 1.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float t = element<DT>(v, e) * inv;
    q[e] = __builtin_rintf(t);
    near = fminf(near, 0.5f - __builtin_fabsf(t - q[e]));
  }
  if (exact || near < 1e-4f) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      q[e] = (float)__builtin_rint(127.0 * (double)element<DT>(v, e) / (double)top);
  }
#pragma unroll
  for (int w = 0; w < N / 4; ++w) {
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      word |= ((uint32_t)(int)q[4 * w + e] & 0xffu) << (8 * e);
    out[w] = word;
  }
}
template <int DT> __device__ __forceinline__ void store_piece(int8_t *row, int c, int cols, const uint32_t (&w)[2]) {
  constexpr int N = Piece<DT>::N;
  const int left = cols - c * N;
  if (left >= N) {
    __builtin_memcpy(row + (int64_t)c * N, w, N);
  } else if (left > 0) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < left)
        row[(int64_t)c * N + e] = (int8_t)(w[e >> 2] >> (8 * (e & 3)));
  }
}

template <int DT>
__device__ __forceinline__ void body(const void *x, int8_t *q, float *scale, const RockQuantizeParams &p) {
  constexpr int N = Piece<DT>::N;
  __shared__ uint32_t wave_top[4];
  const int lanes = p.lanes_per_row, sub = threadIdx.x & (lanes - 1);
  const int64_t row = lanes == 64 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
  if (row >= p.rows)
    return; // (a whole wave; blocks whose waves share a row have one each)
  const char *src = (const char *)x + row * p.cols * Piece<DT>::ES;
  int8_t *dst = q + row * p.cols;
  const int pieces = (p.cols + N - 1) / N;
  const bool resident = pieces <= kPieces * lanes; // uniform
  v4i v[kPieces];
  uint32_t top = 0;
  if (resident) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      v[i] = load_piece<DT>(src, sub + i * lanes, p.cols);
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      top = max_bits<DT>(top, v[i]);
  } else {
    for (int c = sub; c < pieces; c += lanes)
      top = max_bits<DT>(top, load_piece<DT>(src, c, p.cols));
  }
  if constexpr (DT != ROCK_F32)
    top = max(top & 0xffffu, top >> 16);
#pragma unroll
  for (int d = 32; d; d >>= 1)
    top = max(top, __shfl_xor(top, d));
  if (lanes == 256) {
    if ((threadIdx.x & 63) == 0)
      wave_top[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(wave_top[0], wave_top[1]), max(wave_top[2], wave_top[3]));
  }
  constexpr uint32_t kInf = DT == ROCK_F32 ? 0x7f800000u : DT == ROCK_BF16 ? 0x7f80u : 0x7c00u;
  const bool finite = top < kInf, zero = top == 0;
  const float m = widen_bits<DT>(top);
  if (sub == 0)
    scale[row] = finite ? m / 127.0f : __builtin_nanf("");
  const bool exact = finite && m < 0x1p-100f; // 127 / m overflows or m is subnormal
  const float inv = zero || !finite || exact ? 0.0f : 127.0f / m;
  auto emit = [&](int c, const v4i &piece) __attribute__((always_inline)) {
    uint32_t w[2] = {0, 0};
    if (finite && !zero) // uniform over the row; else zeros (an infinity times 0 would not be)
      quantize_piece<DT>(piece, m, inv, exact, w);
    store_piece<DT>(dst, c, p.cols, w);
  };
  if (resident) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      if (sub + i * lanes < pieces)
        emit(sub + i * lanes, v[i]);
  } else {
    for (int c = sub; c < pieces; c += lanes)
      emit(c, load_piece<DT>(src, c, p.cols));
  }
}

} // namespace rkq

// one code object per kernel: see relayout_kernels.hip
#if RK_SELECTED(0)
extern "C" __global__ __launch_bounds__(256) void rock_quantize_tokens_f32(const void *x, void *q, void *scale,
                                                                            RockQuantizeParams p) {
  rkq::body<ROCK_F32>(x, (int8_t *)q, (float *)scale, p);
}
#endif
#if RK_SELECTED(1)
extern "C" __global__ __launch_bounds__(256) void rock_quantize_tokens_f16(const void *x, void *q, void *scale,
                                                                            RockQuantizeParams p) {
  rkq::body<ROCK_F16>(x, (int8_t *)q, (float *)scale, p);
}
#endif
#if RK_SELECTED(2)
extern "C" __global__ __launch_bounds__(256) void rock_quantize_tokens_bf16(const void *x, void *q, void *scale,
                                                                             RockQuantizeParams p) {
  rkq::body<ROCK_BF16>(x, (int8_t *)q, (float *)scale, p);
}
#endif
