// Rows of fp16 / bf16 to 8-bit integers with one scale per row (sk_quantize_i8): the activations
// (one scale per token) or the weights (one per output channel) of sk_gemm_i8.
//
//   a = max_k |x[k]|     scale = a / 127     q[k] = 127 x[k] / a rounded to the nearest integer
//
// One pass over the data: a row is read once, 16 bytes per thread and load, kept in registers
// as it came (16-bit pairs) while its maximum is found, then divided and written.  The bits of
// |x| order like the numbers do, so the maximum is one packed integer instruction per pair, and
// NaN and infinity are whatever ends up at or above the infinity's pattern.
//
// The rounding goes by the exact quotient Q = 127 x / a, halves to even.  x and a are numbers of at
// most 11 bits, X and A times powers of two, so 2 |Q| = 254 |X| 2^i / A is either an odd number or
// at least 1 / (254 * 2047) away from any, relatively (1.9e-6): with an odd n, 254 |X| 2^i - n A is a
// whole number of units in the last place of 254 X or of n A, and zero only if 127 divides n A.  So
// unless 127 divides A, the one half that can occur is n = 127, x = a / 2, and it goes to 64: the
// quotient is taken a little too large, t = x r with r = (127 / a)(1 + 2^-20), and three roundings
// (1.8e-7) neither lose that half nor reach another one; rounding t rounds Q.  Rows whose A is a
// multiple of 127 (one in 127), and those whose a is so small that 127 / a overflows, are rounded
// in exact arithmetic: with b = a 2^-e (between 1 and 4) and x' = x 2^-e (exact; what underflows
// rounds to zero anyway) rounding x' (127 / b) rounds Q, except where Q is a half: there it may fall
// on either side, and the remainder 127 x' - q b, which fp32 holds exactly (18 bits less 18 bits
// of the same place), is plus or minus b / 2.  An odd q is then moved to the even side.
//
// Bound: memory (2 bytes read, 1 written per element; about four instructions per element).
// Measured: 8192 x 11008 of normally distributed bf16 46.7 us, 5.8 TB/s (a copy: 6.6); 16 x 4096
// 1.6 us, a launch.  Tried: looking again at the elements near a half instead of at whole rows (57 us:
// some warp of nearly every row has one, and the row's CTA waits for it); 512 threads a row 65 us,
// 128 threads 62; registers capped for five CTAs an SM are 3 % ahead of no cap, for six no better.
#include "sk_common.cuh"

namespace {

// 8 consecutive elements of a row, as packed pairs.  VEC: the rows allow 16-byte loads.  (Ordinary loads,
// and X is not `const __restrict__`: see skptx::griddep_wait.)
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int k, int K) {
  if (VEC && k + 8 <= K) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(row + k));
    return v;
  }
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (k + j < K) w[j >> 1] |= static_cast<uint32_t>(row[k + j]) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool VEC>
__device__ __forceinline__ void store8(int8_t* row, int k, int K, uint2 q) {
  if (VEC && k + 8 <= K) {
    *reinterpret_cast<uint2*>(row + k) = q;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (k + j < K) row[k + j] = static_cast<int8_t>((j < 4 ? q.x >> (8 * j) : q.y >> (8 * (j - 4))) & 0xFFu);
}

__device__ __forceinline__ uint32_t max_abs(uint32_t m, const uint4& v) {
  m = __vmaxu2(m, v.x & 0x7FFF7FFFu);
  m = __vmaxu2(m, v.y & 0x7FFF7FFFu);
  m = __vmaxu2(m, v.z & 0x7FFF7FFFu);
  return __vmaxu2(m, v.w & 0x7FFF7FFFu);
}

template <bool BF16>
__device__ __forceinline__ float widen(uint32_t bits16) {
  if constexpr (BF16) return __uint_as_float(bits16 << 16);
  else return __half2float(__ushort_as_half(static_cast<unsigned short>(bits16)));
}

template <bool BF16>
__device__ __forceinline__ float widen_high(uint32_t pair) {
  if constexpr (BF16) return __uint_as_float(pair & 0xFFFF0000u);
  else return widen<false>(pair >> 16);
}

struct RowScale {
  float q;            // (127 / a)(1 + 2^-20)
  float pow2, b, r;   // 2^-e, a * 2^-e, 127 / b
};

constexpr float ROUND = 12582912.f;   // 1.5 * 2^23: adding it leaves the nearest integer in the low bits

// One element, exactly: 127 x / a to the nearest integer, halves to even; the low byte holds it.
template <bool BF16>
__device__ __forceinline__ uint32_t quantize1(uint32_t bits16, const RowScale& s) {
  const float x = widen<BF16>(bits16) * s.pow2;
  const float m = __fmaf_rn(x, s.r, ROUND);
  const float q = m - ROUND;
  const float rem = __fmaf_rn(-q, s.b, 127.f * x);
  uint32_t u = __float_as_uint(m);
  if (2.f * fabsf(rem) == s.b && (u & 1u) != 0u) u = __float_as_uint(m + (rem > 0.f ? 1.f : -1.f));
  return u;
}

__device__ __forceinline__ uint2 pack8(const uint32_t (&u)[8]) {
  uint2 q;
  q.x = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
  q.y = __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410);
  return q;
}

template <bool BF16>
__device__ __forceinline__ uint2 quantize8_exactly(const uint4& v, const RowScale& s) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t u[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) u[j] = quantize1<BF16>(w[j >> 1] >> (16 * (j & 1)) & 0xFFFFu, s);
  return pack8(u);
}

template <bool BF16>
__device__ __forceinline__ uint2 quantize8(const uint4& v, const RowScale& s) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t u[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = (j & 1) ? widen_high<BF16>(w[j >> 1]) : widen<BF16>(w[j >> 1] & 0xFFFFu);
    u[j] = __float_as_uint(__fmaf_rn(x, s.q, ROUND));   // (one rounding: that of t to an integer)
  }
  return pack8(u);
}

// G threads take a row, `rows` of them a CTA.  NV > 0: the row fits NV vectors of 8 per thread
// and stays in registers; NV = 0: rows longer than that are read twice (the second time mostly
// from L2).
template <bool BF16, bool VEC, int G, int NV>
__global__ void __launch_bounds__(G < 128 ? 128 : G, G == 256 ? 5 : 1)
sk_quantize_i8_kernel(const uint16_t* X, int M, int K, int ldx, int8_t* __restrict__ Q, int ldq, float* __restrict__ scale) {
  constexpr int THREADS = G < 128 ? 128 : G;
  constexpr int WARPS = THREADS / 32;
  __shared__ uint32_t part[WARPS];
  const int tid = threadIdx.x % G;
  const long long row = static_cast<long long>(blockIdx.x) * (THREADS / G) + threadIdx.x / G;
  skptx::griddep_launch_dependents();
  skptx::griddep_wait();
  if (row >= M) return;   // (whole warps only: G is a multiple of 32; with G > 32 a CTA has one row)
  const uint16_t* x = X + row * ldx;
  uint4 v[NV > 0 ? NV : 1];
  uint32_t m = 0u;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = (i * G + tid) * 8;
      v[i] = k < K ? load8<VEC>(x, k, K) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) m = max_abs(m, v[i]);
  } else {
    for (long long k = tid * 8; k < K; k += G * 8) m = max_abs(m, load8<VEC>(x, static_cast<int>(k), K));
  }
  m = __reduce_max_sync(0xffffffffu, max(m & 0xFFFFu, m >> 16));
  if constexpr (G > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    m = (threadIdx.x & 31) < WARPS ? part[threadIdx.x & 31] : 0u;
    m = __reduce_max_sync(0xffffffffu, m);
  }
  constexpr uint32_t INF = BF16 ? 0x7F80u : 0x7C00u;
  const bool finite = m < INF;
  const float a = widen<BF16>(m);
  if (tid == 0) scale[row] = finite ? __fdiv_rn(a, 127.f) : __uint_as_float(0x7FC00000u);
  RowScale s;
  bool exactly = false;
  if (finite && m != 0u) {
    const int e = 254 - static_cast<int>(__float_as_uint(a) >> 23);
    s.pow2 = __uint_as_float(static_cast<uint32_t>(e > 1 ? e : 1) << 23);
    s.b = a * s.pow2;
    s.r = __fdiv_rn(127.f, s.b);
    s.q = __fdiv_rn(127.f, a) * (1.f + 0x1p-20f);
    constexpr int MANT = BF16 ? 7 : 10;
    const uint32_t A = (m & ((1u << MANT) - 1u)) | (m >> MANT ? 1u << MANT : 0u);
    exactly = A % 127u == 0u || a < 0x1p-100f;
  } else {
    s.q = 0.f; s.pow2 = 0.f; s.b = 1.f; s.r = 0.f;
  }
  int8_t* q = Q + row * ldq;
  if (exactly) {
    // (not unrolled, from memory again: rare)
    for (long long k = tid * 8; k < K; k += G * 8)
      store8<VEC>(q, static_cast<int>(k), K, quantize8_exactly<BF16>(load8<VEC>(x, static_cast<int>(k), K), s));
    return;
  }
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = (i * G + tid) * 8;
      if (!finite) v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (k < K) store8<VEC>(q, k, K, quantize8<BF16>(v[i], s));
    }
  } else {
    for (long long k = tid * 8; k < K; k += G * 8) {
      uint4 w = load8<VEC>(x, static_cast<int>(k), K);
      if (!finite) w = make_uint4(0u, 0u, 0u, 0u);
      store8<VEC>(q, static_cast<int>(k), K, quantize8<BF16>(w, s));
    }
  }
}

template <bool BF16, bool VEC, int G, int NV>
cudaError_t launch(const uint16_t* X, int M, int K, int ldx, int8_t* Q, int ldq, float* scale, bool pdl,
                   cudaStream_t stream) {
  constexpr int THREADS = G < 128 ? 128 : G;
  const int grid = (M + THREADS / G - 1) / (THREADS / G);
  return sk_launch(sk_quantize_i8_kernel<BF16, VEC, G, NV>, grid, THREADS, 0, stream, 1, pdl, X, M, K, ldx, Q, ldq,
                   scale);
}

template <bool BF16, bool VEC>
cudaError_t dispatch(const uint16_t* X, int M, int K, int ldx, int8_t* Q, int ldq, float* scale, bool pdl,
                     cudaStream_t stream) {
  const int vecs = K / 8 + ((K & 7) != 0);
  if (vecs <= 32 * 4) return launch<BF16, VEC, 32, 4>(X, M, K, ldx, Q, ldq, scale, pdl, stream);
  if (vecs <= 256 * 2) return launch<BF16, VEC, 256, 2>(X, M, K, ldx, Q, ldq, scale, pdl, stream);
  if (vecs <= 256 * 4) return launch<BF16, VEC, 256, 4>(X, M, K, ldx, Q, ldq, scale, pdl, stream);
  if (vecs <= 256 * 6) return launch<BF16, VEC, 256, 6>(X, M, K, ldx, Q, ldq, scale, pdl, stream);
  if (vecs <= 1024 * 4) return launch<BF16, VEC, 1024, 4>(X, M, K, ldx, Q, ldq, scale, pdl, stream);
  return launch<BF16, VEC, 1024, 0>(X, M, K, ldx, Q, ldq, scale, pdl, stream);
}

}  // namespace

extern "C" int sk_quantize_i8(const void* X, int M, int K, int ldx, int flags, void* Q, int ldq, float* scale,
                              void* stream) {
  if (!X || !Q || !scale) return SK_ERR_ARG;
  if (M <= 0 || K <= 0 || ldx < K || ldq < K) return SK_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(X) & 1u) != 0 || (reinterpret_cast<uintptr_t>(scale) & 3u) != 0) return SK_ERR_ALIGN;
  sk_problem any;
  memset(&any, 0, sizeof(any));
  int sms = 0, dev_sms = 0;
  const int st = sk_resolve_grid(&any, &sms, &dev_sms);   // (refuses other architectures)
  if (st != SK_OK) return st;
  const bool vec = (reinterpret_cast<uintptr_t>(X) & 15u) == 0 && (ldx & 7) == 0 &&
                   (reinterpret_cast<uintptr_t>(Q) & 7u) == 0 && (ldq & 7) == 0;
  const bool bf16 = (flags & SK_FLAG_BF16) != 0, pdl = (flags & SK_FLAG_PDL) != 0;
  const uint16_t* x = static_cast<const uint16_t*>(X);
  int8_t* q = static_cast<int8_t*>(Q);
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (bf16)
    e = vec ? dispatch<true, true>(x, M, K, ldx, q, ldq, scale, pdl, cs)
            : dispatch<true, false>(x, M, K, ldx, q, ldq, scale, pdl, cs);
  else
    e = vec ? dispatch<false, true>(x, M, K, ldx, q, ldq, scale, pdl, cs)
            : dispatch<false, false>(x, M, K, ldx, q, ldq, scale, pdl, cs);
  return e == cudaSuccess ? SK_OK : sk_set_cuda_error(e);
}
