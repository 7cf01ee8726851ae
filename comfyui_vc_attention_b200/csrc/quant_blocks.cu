// E4M3 quantisation with one scale for each block of 128 columns.
//
//   s = max(max |x|, 1e-30) / 448 over the block,   code = E4M3(x / s)
// Blocks are 1 x 128 (activations: one scale per row) or 128 x 128 (weights).
// A NaN in a block makes its scale, and so the whole block, NaN.
//
// A few lanes hold one 128-column row segment in registers as loaded: the
// maximum is taken on the 16-bit pairs.  Both quotients are Markstein's
// correction of a product with the reciprocal (see DivBy), so the scales and
// codes are those of IEEE divisions; the one of x / s runs on packed fp32
// pairs, scaled up first in blocks of tiny values (kDivMin).  Bound by HBM, the
// elements read once: 16384 x 14336 bf16 in 116-132 us (5.4-6.1 TB/s), square
// blocks of 14336 x 5376 in 44 us (5.2 TB/s).
#include <string>

#include "kernels.cuh"
#include "tc_math.cuh"

namespace vcattn {
namespace {

constexpr int kBlk = 128;
constexpr int kThreads = 256;

struct QuantArgs {
  const void* x;
  int64_t ldx;
  uint8_t* codes;
  int64_t ldc;
  float* scale;
  int64_t ssm, ssk;   // scale strides over row blocks and column blocks
  int64_t M;
  int K, kb;
  int64_t segs;       // 1 x 128 blocks: M * kb
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The correction's remainder x - q0 s is a multiple of ulp(q0) ulp(s).  Codes
// other than 0 have quotients of 2^-10 and more, so from this scale on that is
// 2^-147 or more and the remainder exact; below it (wrong codes next to ties
// from a maximum of 2^-99 down) x and s are multiplied by 2^64 first, exactly.
// (The division itself took 3.4 times as long on blocks of zeros.)
constexpr float kDivMin = 0x1p-90f, kDivUp = 0x1p64f;

// Eight consecutive columns as loaded: 16-bit pairs, or fp32.
template <int DT> struct Cols8 {
  uint32_t u[4];
  __device__ __forceinline__ float max_abs() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max_pair(m, u[i] & 0x7fff7fffu);
    if constexpr (DT == VCATTN_DTYPE_BF16) return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
    return max_nan(f.x, f.y);
  }
  // Per half, NaN if either is.
  static __device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
    if constexpr (DT == VCATTN_DTYPE_BF16) {
      const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
      return *reinterpret_cast<const uint32_t*>(&r);
    } else {
      const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
      return *reinterpret_cast<const uint32_t*>(&r);
    }
  }
  __device__ __forceinline__ void pair(int i, float& x, float& y) const {
    if constexpr (DT == VCATTN_DTYPE_BF16) {
      x = __uint_as_float(u[i] << 16);
      y = __uint_as_float(u[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x = f.x;
      y = f.y;
    }
  }
  // All columns times kDivUp.  (Blocks of f16 that small hold zeros alone.)
  __device__ __forceinline__ void scale_up() {
    if constexpr (DT == VCATTN_DTYPE_BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x, y;
        pair(i, x, y);
        const __nv_bfloat162 r = __floats2bfloat162_rn(x * kDivUp, y * kDivUp);
        u[i] = *reinterpret_cast<const uint32_t*>(&r);
      }
    }
  }
  __device__ __forceinline__ void load(const void* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w;
  }
  __device__ __forceinline__ void load_some(const void* p, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = 2 * i < n ? static_cast<const uint16_t*>(p)[2 * i] : 0u;
      if (2 * i + 1 < n) u[i] |= static_cast<uint32_t>(static_cast<const uint16_t*>(p)[2 * i + 1]) << 16;
    }
  }
};
template <> struct Cols8<VCATTN_DTYPE_F32> {
  float v[8];
  __device__ __forceinline__ float max_abs() const {
    float m = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(v[i]));
    return m;
  }
  __device__ __forceinline__ void pair(int i, float& x, float& y) const {
    x = v[2 * i];
    y = v[2 * i + 1];
  }
  __device__ __forceinline__ void scale_up() {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= kDivUp;
  }
  __device__ __forceinline__ void load(const void* p) {
    const float4 a = static_cast<const float4*>(p)[0], b = static_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void load_some(const void* p, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? static_cast<const float*>(p)[i] : 0.f;
  }
};

// Eight columns from c on of one row (columns past K, or all if !in, read as 0).
template <int DT, bool VEC>
__device__ __forceinline__ void load_cols(const QuantArgs& a, bool in, int64_t row, int c, Cols8<DT>& v) {
  const int n = in ? a.K - c : 0;
  const void* p = static_cast<const typename Elem<DT>::T*>(a.x) + (n > 0 ? row * a.ldx + c : 0);
  if (VEC && n >= 8) v.load(p);
  else v.load_some(p, n);
}

// max(amax, 1e-30) / 448: Markstein's quotient with the constant's reciprocal.
__device__ __forceinline__ float block_scale(float amax) {
  amax = max_nan(amax, kTiny);
  constexpr float y = 1.0f / kE4M3Max;
  const float q0 = __fmul_rn(amax, y);
  const float q = __fmaf_rn(__fmaf_rn(-q0, kE4M3Max, amax), y, q0);
  return amax < INFINITY ? q : amax;
}

// The divisor of a block's values and its reciprocal.
template <int DT, int N>
__device__ __forceinline__ float divisor(float s, Cols8<DT> (&v)[N], float& y) {
  if (s < kDivMin) {
#pragma unroll
    for (int u = 0; u < N; ++u) v[u].scale_up();
    s *= kDivUp;
  }
  y = __frcp_rn(s);
  return s;
}

__device__ __forceinline__ uint32_t codes2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// Codes of eight columns (the columns past K are not written).
template <int DT>
__device__ __forceinline__ void store_codes(const QuantArgs& a, int64_t row, int c, const Cols8<DT>& v, float s, float y) {
  uint32_t w[4];
  if (s < INFINITY) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x0, x1;
      v.pair(i, x0, x1);
      float q0 = x0, q1 = x1;
      tc::mul2(q0, q1, y, y);
      tc::fma2(x0, x1, q0, q1, -s, -s);   // the remainder
      tc::fma2(q0, q1, x0, x1, y, y);
      w[i] = codes2(q0, q1);
    }
  } else {   // an infinite or NaN block: the divisions themselves
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x0, x1;
      v.pair(i, x0, x1);
      w[i] = codes2(__fdiv_rn(x0, s), __fdiv_rn(x1, s));
    }
  }
  const uint2 b = make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
  uint8_t* p = a.codes + row * a.ldc + c;
  if (c + 8 <= a.K) {   // ldc and the base are multiples of 16
    *reinterpret_cast<uint2*>(p) = b;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < a.K) p[i] = static_cast<uint8_t>(((i < 4 ? b.x : b.y) >> (8 * (i & 3))) & 0xffu);
  }
}

// 1 x 128 blocks: kLanes lanes per block, each with every kLanes-th chunk of
// eight columns, so that the block's scale and its reciprocal are computed by
// few lanes for many elements each (16384 x 14336: 16 lanes 163 us, 8 lanes
// 126, 4 lanes 116).
constexpr int kLanes = 4;
constexpr int kChunks = 16 / kLanes;

template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) quant_rows_blocks_kernel(const QuantArgs a) {
  const int l = threadIdx.x % kLanes;
  const int64_t seg = static_cast<int64_t>(blockIdx.x) * (kThreads / kLanes) + threadIdx.x / kLanes;
  // (a 64-bit division takes longer than the rest of the block)
  int64_t row;
  if (a.segs < (int64_t{1} << 31)) row = static_cast<uint32_t>(seg) / static_cast<uint32_t>(a.kb);
  else row = seg / a.kb;
  const int blk = static_cast<int>(seg - row * a.kb);
  Cols8<DT> v[kChunks];
#pragma unroll
  for (int u = 0; u < kChunks; ++u) load_cols<DT, VEC>(a, seg < a.segs, row, blk * kBlk + (u * kLanes + l) * 8, v[u]);
  float m = v[0].max_abs();
#pragma unroll
  for (int u = 1; u < kChunks; ++u) m = max_nan(m, v[u].max_abs());
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (seg >= a.segs) return;
  float s = block_scale(m), y;
  if (l == 0) a.scale[row * a.ssm + blk * a.ssk] = s;
  s = divisor(s, v, y);
#pragma unroll
  for (int u = 0; u < kChunks; ++u) store_codes<DT>(a, row, blk * kBlk + (u * kLanes + l) * 8, v[u], s, y);
}

// 128 x 128 blocks: one CTA per block, eight rows of eight columns per thread.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) quant_square_blocks_kernel(const QuantArgs a) {
  __shared__ float wmax[kThreads / 32];
  const int64_t mb = blockIdx.x / a.kb;
  const int blk = static_cast<int>(blockIdx.x - mb * a.kb);
  const int c = blk * kBlk + (threadIdx.x & 15) * 8;
  const int64_t r0 = mb * kBlk + (threadIdx.x >> 4);
  Cols8<DT> v[8];
  float m = 0.f;
#pragma unroll
  for (int u = 0; u < 8; ++u) load_cols<DT, VEC>(a, r0 + 16 * u < a.M, r0 + 16 * u, c, v[u]);
#pragma unroll
  for (int u = 0; u < 8; ++u) m = max_nan(m, v[u].max_abs());
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) wmax[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) m = max_nan(m, wmax[w]);
  float s = block_scale(m), y;
  if (threadIdx.x == 0) a.scale[mb * a.ssm + blk * a.ssk] = s;
  s = divisor(s, v, y);
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (r0 + 16 * u < a.M) store_codes<DT>(a, r0 + 16 * u, c, v[u], s, y);
}

template <int DT, bool VEC>
cudaError_t launch(const QuantArgs& a, int rows, cudaStream_t st) {
  if (rows == 1) {
    const int64_t per = kThreads / kLanes;
    quant_rows_blocks_kernel<DT, VEC><<<static_cast<unsigned>((a.segs + per - 1) / per), kThreads, 0, st>>>(a);
  } else {
    const int64_t n = (a.M + kBlk - 1) / kBlk * a.kb;
    quant_square_blocks_kernel<DT, VEC><<<static_cast<unsigned>(n), kThreads, 0, st>>>(a);
  }
  return cudaGetLastError();
}

int arg_error(const char* msg) {
  return record_error(VCATTN_ERR_ARG, (std::string("vcattn_quantize_blocks: ") + msg).c_str());
}

}  // namespace
}  // namespace vcattn

extern "C" VCATTN_API int vcattn_quantize_blocks(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx,
                                                 int block_rows, uint8_t* codes, int64_t ldc, float* scale,
                                                 int64_t scale_sm, int64_t scale_sk, void* stream) {
  using namespace vcattn;
  clear_error();
  if (fault_injected("vcattn_quantize_blocks"))
    return record_error(VCATTN_ERR_INJECTED, "vcattn_quantize_blocks: injected fault");
  if (dtype != VCATTN_DTYPE_BF16 && dtype != VCATTN_DTYPE_F16 && dtype != VCATTN_DTYPE_F32)
    return arg_error("unsupported dtype");
  if (block_rows != 1 && block_rows != kBlk) return arg_error("block_rows must be 1 or 128");
  if (M < 0 || K < 0 || M > (int64_t{1} << 36) || K > (int64_t{1} << 30)) return arg_error("size out of range");
  if (M == 0 || K == 0) return VCATTN_OK;
  if (!x || !codes || !scale) return arg_error("null pointer");
  if (ldx < K || ldc < K) return arg_error("row stride below the row length");
  if ((reinterpret_cast<uintptr_t>(codes) & 15u) || ldc % 16) return arg_error("code rows must be 16-byte aligned");
  QuantArgs a{};
  a.x = x; a.ldx = ldx; a.codes = codes; a.ldc = ldc; a.scale = scale; a.ssm = scale_sm; a.ssk = scale_sk;
  a.M = M; a.K = static_cast<int>(K);
  a.kb = static_cast<int>((K + kBlk - 1) / kBlk);
  a.segs = M * a.kb;
  if (a.segs >= (int64_t{1} << 36)) return arg_error("size out of range");
  const int es = dtype == VCATTN_DTYPE_F32 ? 4 : 2;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (ldx * es) % 16 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == VCATTN_DTYPE_BF16)
    e = vec ? launch<VCATTN_DTYPE_BF16, true>(a, block_rows, st) : launch<VCATTN_DTYPE_BF16, false>(a, block_rows, st);
  else if (dtype == VCATTN_DTYPE_F16)
    e = vec ? launch<VCATTN_DTYPE_F16, true>(a, block_rows, st) : launch<VCATTN_DTYPE_F16, false>(a, block_rows, st);
  else
    e = vec ? launch<VCATTN_DTYPE_F32, true>(a, block_rows, st) : launch<VCATTN_DTYPE_F32, false>(a, block_rows, st);
  if (e != cudaSuccess)
    return record_error(VCATTN_ERR_CUDA, (std::string("vcattn_quantize_blocks: ") + cudaGetErrorString(e)).c_str());
  return VCATTN_OK;
}
