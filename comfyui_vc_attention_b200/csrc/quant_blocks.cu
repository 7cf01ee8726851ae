// E4M3 quantisation with one scale for each block of 128 columns.
//
//   s = max(max |x|, 1e-30) / 448 over the block,   code = E4M3(x / s)
// Blocks are 1 x 128 (activations: one scale per row) or 128 x 128 (weights).
// A NaN in a block makes its scale, and so the whole block, NaN.
//
// Sixteen lanes hold one 128-column row segment, eight columns each.  Bound by
// HBM: the elements are read once and stay in registers over the maximum and
// the conversion.
#include <string>

#include "kernels.cuh"

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

// Eight columns from c on of one row (columns past K read as 0).
template <int DT, bool VEC>
__device__ __forceinline__ void load_cols(const QuantArgs& a, int64_t row, int c, float (&v)[8]) {
  using T = typename Elem<DT>::T;
  const T* p = static_cast<const T*>(a.x) + row * a.ldx + c;
  if (VEC && c + 8 <= a.K) {
    if constexpr (DT == VCATTN_DTYPE_F32) {
      const float4 f = load4<DT>(p, 0), g = load4<DT>(p, 4);
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
      v[4] = g.x; v[5] = g.y; v[6] = g.z; v[7] = g.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const uint32_t r[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == VCATTN_DTYPE_BF16) {
          v[2 * i] = __uint_as_float(r[i] << 16);
          v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < a.K ? Elem<DT>::load(p + i) : 0.f;
  }
}

__device__ __forceinline__ float max8(const float (&v)[8]) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(v[i]));
  return m;
}

__device__ __forceinline__ float block_scale(float amax) { return __fdiv_rn(max_nan(amax, kTiny), kE4M3Max); }

// Codes of eight columns (the columns past K are not written).  The quotient
// is DivBy's; an infinite or NaN scale takes the division itself.
__device__ __forceinline__ void store_codes(const QuantArgs& a, int64_t row, int c, const float (&v)[8], float s) {
  float q[8];
  if (s < INFINITY) {
    const DivBy by(s);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = by(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = __fdiv_rn(v[i], s);
  }
  const uint2 w = make_uint2(e4m3x4(q[0], q[1], q[2], q[3]), e4m3x4(q[4], q[5], q[6], q[7]));
  uint8_t* p = a.codes + row * a.ldc + c;
  if (c + 8 <= a.K) {   // ldc and the base are multiples of 16
    *reinterpret_cast<uint2*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < a.K) p[i] = static_cast<uint8_t>((i < 4 ? w.x >> (8 * i) : w.y >> (8 * (i - 4))) & 0xffu);
  }
}

// 1 x 128 blocks: half a warp per block, kSegs blocks per half-warp in flight.
constexpr int kSegs = 4;

template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) quant_rows_blocks_kernel(const QuantArgs a) {
  const int l = threadIdx.x & 15;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * (kThreads / 16) + (threadIdx.x >> 4)) * kSegs;
  float v[kSegs][8];
  int64_t row[kSegs];
  int blk[kSegs];
  {
    int64_t r = first / a.kb;
    int b = static_cast<int>(first - r * a.kb);
#pragma unroll
    for (int u = 0; u < kSegs; ++u) {
      row[u] = r;
      blk[u] = b;
      if (++b == a.kb) {
        b = 0;
        ++r;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kSegs; ++u) {
    if (first + u < a.segs) load_cols<DT, VEC>(a, row[u], blk[u] * kBlk + l * 8, v[u]);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
  }
#pragma unroll
  for (int u = 0; u < kSegs; ++u) {
    float m = max8(v[u]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (first + u < a.segs) {
      const float s = block_scale(m);
      if (l == 0) a.scale[row[u] * a.ssm + blk[u] * a.ssk] = s;
      store_codes(a, row[u], blk[u] * kBlk + l * 8, v[u], s);
    }
  }
}

// 128 x 128 blocks: one CTA per block, eight rows of eight columns per thread.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) quant_square_blocks_kernel(const QuantArgs a) {
  __shared__ float wmax[kThreads / 32];
  const int64_t mb = blockIdx.x / a.kb;
  const int blk = static_cast<int>(blockIdx.x - mb * a.kb);
  const int c = blk * kBlk + (threadIdx.x & 15) * 8;
  const int64_t r0 = mb * kBlk + (threadIdx.x >> 4);
  float v[8][8];
  float m = 0.f;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    if (r0 + 16 * u < a.M) load_cols<DT, VEC>(a, r0 + 16 * u, c, v[u]);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
  }
#pragma unroll
  for (int u = 0; u < 8; ++u) m = max_nan(m, max8(v[u]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) wmax[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) m = max_nan(m, wmax[w]);
  const float s = block_scale(m);
  if (threadIdx.x == 0) a.scale[mb * a.ssm + blk * a.ssk] = s;
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (r0 + 16 * u < a.M) store_codes(a, r0 + 16 * u, c, v[u], s);
}

template <int DT, bool VEC>
cudaError_t launch(const QuantArgs& a, int rows, cudaStream_t st) {
  if (rows == 1) {
    const int64_t per = (kThreads / 16) * kSegs;
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
  if (M < 0 || K < 0 || K > (int64_t{1} << 30)) return arg_error("size out of range");
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
