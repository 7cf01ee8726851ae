// RMS norm of every query / key head and the position rotation, one pass.
//
//   y = x * rsqrt(mean_d x^2 + eps) * w            (per head row of D channels)
//   (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s)   on the first `rot` channels
// with j = i + rot/2 (half layout) or j = i + 1, i even (interleaved).
//
// A row is spread over LPR lanes in chunks of eight channels (16-byte loads for
// 16-bit types): one chunk per lane in the interleaved layout, two in the half
// layout, where they are partners, so no channel crosses lanes (with one chunk
// and a shuffle the half layout took 201 us where this takes 170).  Since the
// norm is one factor per row, w, cos and sin fold into two coefficients per
// channel, out_e = r * (x_e cw_e + x_p sw_e) with p the partner channel; a warp
// makes them for one token and applies them to its heads, whose rows it has
// loaded before.  Bound by HBM, every element read once and written once: a
// 16384-token clip of 56 + 56 heads x 128 bf16 in 154 us interleaved (6.1 TB/s)
// and 182 us in the half layout (170 into the same buffers again and again),
// whose two chunks per lane take 92 registers.
#include <string>

#include "kernels.cuh"
#include "tc_math.cuh"

namespace vcattn {
namespace {

constexpr int kWarpsPerCta = 4;
// Rows loaded per lane before the first use (16384 x 112 rows of 128 bf16, 96
// rotated: 2, 3 and 4 rows in the half layout take 175, 170 and 183 us).
template <bool HALF> constexpr int kRowsInFlight = HALF ? 3 : 4;

struct RopeArgs {
  const void* x[2];
  void* y[2];
  int64_t xsb[2], xsh[2], xsn[2], ysb[2], ysh[2], ysn[2];
  const float* w[2];
  int heads[2];
  const float *cos, *sin;
  int64_t tsb, tsn;
  int B, N, D, rot;
  float eps, inv_d;
  int norm;
  int chunk_heads, chunks_q, chunks;   // heads per warp, and warps per token
  int token_major;                     // consecutive warps share a token (its heads are adjacent in memory)
  uint32_t items;
};

// Eight consecutive elements of a row, as loaded.
template <int DT> struct Raw8 {
  uint4 u;
  __device__ __forceinline__ void load(const void* base, int64_t off) {
    u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + off);
  }
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void values(float (&v)[8]) const {
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
  static __device__ __forceinline__ void store(void* base, int64_t off, const float (&v)[8]) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == VCATTN_DTYPE_BF16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        r[i] = *reinterpret_cast<const uint32_t*>(&b);
      } else {
        const __half2 b = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        r[i] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + off) = make_uint4(r[0], r[1], r[2], r[3]);
  }
};
template <> struct Raw8<VCATTN_DTYPE_F32> {
  float4 a, b;
  __device__ __forceinline__ void load(const void* base, int64_t off) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + off);
    a = p[0];
    b = p[1];
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  static __device__ __forceinline__ void store(void* base, int64_t off, const float (&v)[8]) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + off);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
};

__device__ __forceinline__ void load8f(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

template <int DT, int LPR, bool HALF>
__global__ void __launch_bounds__(kWarpsPerCta * 32) qk_norm_rope_kernel(const RopeArgs a) {
  constexpr int RPW = 32 / LPR;   // rows (heads) side by side in a warp
  constexpr int CH = HALF ? 2 : 1, U = kRowsInFlight<HALF>;
  const uint32_t item = blockIdx.x * kWarpsPerCta + (threadIdx.x >> 5);
  if (item >= a.items) return;    // whole warps
  const int lane = threadIdx.x & 31, sub = lane / LPR, l = lane % LPR;
  const uint32_t tokens = static_cast<uint32_t>(a.B) * a.N;
  const uint32_t tok = a.token_major ? item / a.chunks : item % tokens;
  const int chunk = a.token_major ? item % a.chunks : item / tokens;
  const int b = tok / a.N, n = tok % a.N;
  const int t = chunk < a.chunks_q ? 0 : 1;   // q or k
  const int h0 = (t ? chunk - a.chunks_q : chunk) * a.chunk_heads;
  const int h1 = min(h0 + a.chunk_heads, a.heads[t]);

  // This lane's first channels: in the half layout chunk l of the first
  // rotated half and its partner, then the channels past `rot` in two halves.
  const int row_chunks = a.D / 8;
  const int pairs = HALF ? a.rot / 16 : 0;
  const int rest = HALF ? (row_chunks - 2 * pairs + 1) / 2 : row_chunks;
  const bool partner = l < pairs;
  int e[CH];
  bool live[CH];
  e[0] = 8 * (partner ? l : pairs + l);                    // (2 pairs + (l - pairs))
  live[0] = l < pairs + rest;
  if constexpr (HALF) {
    e[1] = 8 * (partner ? pairs + l : pairs + rest + l);
    live[1] = live[0] && e[1] < a.D;
  }

  const int64_t xoff = b * a.xsb[t] + n * a.xsn[t], yoff = b * a.ysb[t] + n * a.ysn[t];
  Raw8<DT> raw[U][CH];
#pragma unroll
  for (int u = 0; u < U; ++u) {   // in flight while the coefficients are made
    const int h = h0 + u * RPW + sub;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      if (live[j] && h < h1) raw[u][j].load(a.x[t], xoff + h * a.xsh[t] + e[j]);
      else raw[u][j].zero();
    }
  }

  float cw[CH][8], sw[CH][8];
  bool turned[CH];
  const int64_t trow = b * a.tsb + n * a.tsn;
#pragma unroll
  for (int j = 0; j < CH; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i) cw[j][i] = 1.f;
    if (live[j] && a.w[t] != nullptr) load8f(a.w[t] + e[j], cw[j]);
    turned[j] = HALF ? partner : live[j] && e[j] < a.rot;
  }
  if constexpr (HALF) {
    if (partner) {
      float c[8], s[8];
      load8f(a.cos + trow + e[0], c);
      load8f(a.sin + trow + e[0], s);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sw[0][i] = -cw[1][i] * s[i];
        sw[1][i] = cw[0][i] * s[i];
        cw[0][i] *= c[i];
        cw[1][i] *= c[i];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      if (turned[j]) {
        const float4 c = *reinterpret_cast<const float4*>(a.cos + trow + e[j] / 2);
        const float4 s = *reinterpret_cast<const float4*>(a.sin + trow + e[j] / 2);
        const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sw[j][2 * i] = -cw[j][2 * i + 1] * ss[i];
          sw[j][2 * i + 1] = cw[j][2 * i] * ss[i];
          cw[j][2 * i] *= cc[i];
          cw[j][2 * i + 1] *= cc[i];
        }
      }
    }
  }

#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * RPW + sub;
    float v[CH][8];
#pragma unroll
    for (int j = 0; j < CH; ++j) raw[u][j].values(v[j]);
    float r = 1.f;
    if (a.norm) {
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int j = 0; j < CH; ++j)
#pragma unroll
        for (int i = 0; i < 8; i += 2) tc::fma2(s0, s1, v[j][i], v[j][i + 1], v[j][i], v[j][i + 1]);
      s0 += s1;
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
      r = rsqrtf(fmaf(s0, a.inv_d, a.eps));
    }
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        out[i] = v[j][i];
        out[i + 1] = v[j][i + 1];
        tc::mul2(out[i], out[i + 1], cw[j][i], cw[j][i + 1]);
        // (the channels past `rot` take no partner: its value may be infinite)
        if (turned[j]) {
          const float p0 = HALF ? v[CH - 1 - j][i] : v[j][i + 1], p1 = HALF ? v[CH - 1 - j][i + 1] : v[j][i];
          tc::fma2(out[i], out[i + 1], p0, p1, sw[j][i], sw[j][i + 1]);
        }
        tc::mul2(out[i], out[i + 1], r, r);
      }
      if (live[j] && h < h1) Raw8<DT>::store(a.y[t], yoff + h * a.ysh[t] + e[j], out);
    }
  }
}

// Lanes of a row when each has `chunks` chunks.
int lanes_per_row(int D, int chunks) { return (D <= 64 ? 8 : D <= 128 ? 16 : 32) / chunks; }

template <int DT, int LPR, bool HALF>
cudaError_t launch_rows(RopeArgs a, cudaStream_t st) {
  a.chunk_heads = 32 / LPR * kRowsInFlight<HALF>;
  a.chunks_q = (a.heads[0] + a.chunk_heads - 1) / a.chunk_heads;
  a.chunks = a.chunks_q + (a.heads[1] + a.chunk_heads - 1) / a.chunk_heads;
  const int64_t items = static_cast<int64_t>(a.B) * a.N * a.chunks;
  if (items >= (int64_t{1} << 31)) return cudaErrorInvalidValue;
  a.items = static_cast<uint32_t>(items);
  const unsigned ctas = (a.items + kWarpsPerCta - 1) / kWarpsPerCta;
  qk_norm_rope_kernel<DT, LPR, HALF><<<ctas, kWarpsPerCta * 32, 0, st>>>(a);
  return cudaGetLastError();
}

template <int DT>
cudaError_t launch_dtype(const RopeArgs& a, bool half, cudaStream_t st) {
  switch (lanes_per_row(a.D, half ? 2 : 1)) {
    case 4: return launch_rows<DT, 4, true>(a, st);
    case 8: return half ? launch_rows<DT, 8, true>(a, st) : launch_rows<DT, 8, false>(a, st);
    case 16: return half ? launch_rows<DT, 16, true>(a, st) : launch_rows<DT, 16, false>(a, st);
    default: return launch_rows<DT, 32, false>(a, st);
  }
}

int arg_error(const char* msg) {
  return record_error(VCATTN_ERR_ARG, (std::string("vcattn_qk_norm_rope: ") + msg).c_str());
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool view_fits(const vcattn_bhnd* v, int es) {
  const int64_t q = 16 / es;
  return v != nullptr && v->data != nullptr && aligned(v->data) && v->sb % q == 0 && v->sh % q == 0 && v->sn % q == 0;
}

}  // namespace
}  // namespace vcattn

extern "C" VCATTN_API int vcattn_qk_norm_rope(const vcattn_bhnd* q, const vcattn_bhnd* k, int dtype, int B, int Hq,
                                              int Hk, int N, int D, const float* q_weight, const float* k_weight,
                                              const float* cos_table, const float* sin_table, int64_t table_sb,
                                              int64_t table_sn, int rot, int flags, float eps,
                                              const vcattn_bhnd* q_out, const vcattn_bhnd* k_out, void* stream) {
  using namespace vcattn;
  clear_error();
  if (fault_injected("vcattn_qk_norm_rope"))
    return record_error(VCATTN_ERR_INJECTED, "vcattn_qk_norm_rope: injected fault");
  if (dtype != VCATTN_DTYPE_BF16 && dtype != VCATTN_DTYPE_F16 && dtype != VCATTN_DTYPE_F32)
    return arg_error("unsupported dtype");
  if (B < 0 || Hq < 0 || Hk < 0 || N < 0) return arg_error("negative size");
  if (D < 8 || D > 256 || D % 8) return arg_error("D must be a multiple of 8 up to 256");
  if (rot < 0 || rot > D || rot % 16) return arg_error("rot must be a multiple of 16 up to D");
  if (flags & ~(VCATTN_ROPE_INTERLEAVED | VCATTN_ROPE_NORM)) return arg_error("unknown flag");
  const int64_t heads = static_cast<int64_t>(Hq) + Hk;
  if (static_cast<int64_t>(B) * N == 0 || heads == 0) return VCATTN_OK;
  const int es = dtype == VCATTN_DTYPE_F32 ? 4 : 2;
  if ((Hq > 0 && (!view_fits(q, es) || !view_fits(q_out, es))) || (Hk > 0 && (!view_fits(k, es) || !view_fits(k_out, es))))
    return arg_error("q, k and the outputs must be 16-byte aligned with strides of 16-byte multiples");
  if (rot > 0 && (!cos_table || !sin_table || !aligned(cos_table) || !aligned(sin_table) || table_sb % 4 || table_sn % 4))
    return arg_error("the tables must be 16-byte aligned with strides of 16-byte multiples");
  if (!aligned(q_weight) || !aligned(k_weight)) return arg_error("the weights must be 16-byte aligned");
  RopeArgs a{};
  const vcattn_bhnd* in[2] = {q, k};
  const vcattn_bhnd* out[2] = {q_out, k_out};
  a.heads[0] = Hq;
  a.heads[1] = Hk;
  for (int t = 0; t < 2; ++t) {
    if (a.heads[t] == 0) continue;
    a.x[t] = in[t]->data;
    a.y[t] = const_cast<void*>(out[t]->data);
    a.xsb[t] = in[t]->sb; a.xsh[t] = in[t]->sh; a.xsn[t] = in[t]->sn;
    a.ysb[t] = out[t]->sb; a.ysh[t] = out[t]->sh; a.ysn[t] = out[t]->sn;
  }
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.cos = cos_table; a.sin = sin_table; a.tsb = table_sb; a.tsn = table_sn;
  a.B = B; a.N = N; a.D = D; a.rot = rot;
  a.eps = eps;
  a.inv_d = 1.0f / static_cast<float>(D);
  a.norm = (flags & VCATTN_ROPE_NORM) ? 1 : 0;
  const int t0 = Hq > 0 ? 0 : 1;
  a.token_major = a.xsh[t0] <= a.xsn[t0];
  // (a warp takes four heads or more, so this bounds its count of groups)
  if (static_cast<int64_t>(B) * N > ((int64_t{1} << 31) - 1) / heads) return arg_error("2^31 head rows or more");
  const bool half = !(flags & VCATTN_ROPE_INTERLEAVED);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == VCATTN_DTYPE_BF16  ? launch_dtype<VCATTN_DTYPE_BF16>(a, half, st)
                        : dtype == VCATTN_DTYPE_F16 ? launch_dtype<VCATTN_DTYPE_F16>(a, half, st)
                                                    : launch_dtype<VCATTN_DTYPE_F32>(a, half, st);
  if (e != cudaSuccess)
    return record_error(VCATTN_ERR_CUDA, (std::string("vcattn_qk_norm_rope: ") + cudaGetErrorString(e)).c_str());
  return VCATTN_OK;
}
