// Packed attention on the 5th-generation tensor cores, for the sequences whose
// queries cost more in 64-row register-MMA tiles over a KV head's group (from 17
// queries on with one query head per KV head, from 33 with four).
//
//   O = softmax(scale q k^T + mask) v,  one pass over the keys with a running
//   reference m and sum l per row (fp32)
//
// One CTA = 256 query rows (two 128-row halves) of one sequence and head; 12
// warps in 3 warpgroups:
//   warp 0       TMA producer: Q once, then K and V tiles of 128 keys in a ring
//   warp 1       MMA issuer and tensor-memory owner
//   warps 2-3    V tiles that hold rows the CTA must not use (see below)
//   warps 4-7    softmax of the first half, thread = query row = TMEM lane
//   warps 8-11   softmax of the second half
// TMEM columns: S of the halves [0,128) [128,256), O [256,384) [384,512); P
// (16 bits) goes over the first 64 columns of its own S and feeds the P V
// product from tensor memory.  MMAs complete in issue order, so per half the
// issuer runs  P V (tile j), S (tile j + 1)  as P of tile j comes in
// (two parts of 64 keys), and while the softmax of one half works the tensor
// pipe runs the other half's two products.  When S of tile j is complete, so is the P V
// product of tile j - 1: the softmax thread may rescale its row of O without a
// hand-off.  It does so only when the row's maximum outgrows m by more than kGrow
// (in powers of two): m is a reference, not the maximum, P stays bounded, and
// the division by l at the end cancels it exactly.
//
// Rows of a V tile past the sequence's end belong to another sequence (or to
// nobody) and have P = 0; warps 2-3 overwrite them with zeros, since 0 times
// an infinite value is NaN.  Where the causal mask ends inside a tile they
// look for infinite or NaN values, which enter the product as 0; the rows
// that see them add their share at the end.
// Bound by the power cap on long sequences (16384 x 16384, 14 heads x 128:
// 1.82 ms, 1.06 PFLOP/s, three quarters of the sustained cuBLAS rate; 1.58 ms
// in short runs, of which 2^x takes 0.13 and the whole softmax 0.23; 14 heads x
// 64 1.38 ms, where the 2^x alone are 0.81), by item set-up and output on short
// ones (causal prompts of 4097 queries 161 us).  Every wait is bounded.
#include "attn_packed.cuh"

#include <cuda.h>
#include <algorithm>
#include <mutex>

#include "launch.cuh"
#include "tc_common.cuh"
#include "tc_math.cuh"

namespace vcattn {

__device__ tc::DevStatus g_attn_packed_status;

namespace {

using namespace tc;

constexpr int kHalf = 128;      // query rows of a softmax warpgroup
constexpr int kKeys = 128;      // keys per tile
constexpr int kThreads = 384;
constexpr uint32_t kColS = 0, kColO = 256;
// A row's reference m starts kRaise (log2) below its first maximum, and follows
// when the maximum outgrows that by kGrow more.  bf16 holds every P = 2^(s - m)
// below 2^8 to its eight bits.  f16 has steps of 2^-24 below 2^-14, so P uses
// its range up to 2^15, and the reference follows closer: a probability is off
// by 2^-11 of itself or by 2^-36 of the row's largest.  (With 8 and 0, 65536
// keys 18 nats below the first lost 2.8 % of the output; 8192 x 8192, 8 heads x
// 128, 229 us with 4, 245 with 2 and 13.)
template <int DT> constexpr float kRaise = DT == VCATTN_DTYPE_F16 ? 11.f : 0.f;
template <int DT> constexpr float kGrow = DT == VCATTN_DTYPE_F16 ? 4.f : 8.f;

template <int D> struct Cfg {
  static constexpr int kStages = D == 128 ? 4 : 8;
  static constexpr int kBlocks = D / 64;               // 64-channel blocks of a tile (128-byte swizzled rows)
  static constexpr int kBlockBytes = kKeys * 128;
  static constexpr int kTileBytes = kBlocks * kBlockBytes;
};

template <int D> struct PackedSmem {
  alignas(1024) uint8_t q[2][Cfg<D>::kTileBytes];
  alignas(1024) uint8_t kv[Cfg<D>::kStages][Cfg<D>::kTileBytes];   // tile i: K of step i / 2 (i even) or V
  alignas(8) uint64_t q_full;
  alignas(8) uint64_t full[Cfg<D>::kStages];
  alignas(8) uint64_t empty[Cfg<D>::kStages];
  alignas(8) uint64_t v_ok[Cfg<D>::kStages / 2];   // the V tile of a stage may be used
  alignas(8) uint64_t s_full[2];
  alignas(8) uint64_t p_full[2][2];                // P of the first and the last 64 keys
  alignas(8) uint64_t o_full[2];
  alignas(8) uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int bad;                          // an edge tile held infinite or NaN values
  PackedTile t;
};

template <int DT> __host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn_major) {
  constexpr uint32_t f = DT == VCATTN_DTYPE_BF16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_if(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts_if(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
// 2^x (the hardware's approximation, subnormal results 0).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
template <int DT> __device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (DT == VCATTN_DTYPE_BF16) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}
template <int DT> __device__ __forceinline__ bool not_finite(uint32_t bits16) {
  constexpr uint32_t e = DT == VCATTN_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
  return (bits16 & e) == e;
}
template <int DT> __device__ __forceinline__ float value16(uint32_t bits16) {
  if constexpr (DT == VCATTN_DTYPE_BF16) return __uint_as_float(bits16 << 16);
  else return __half2float(__ushort_as_half(static_cast<unsigned short>(bits16)));
}

// Keys [0, lim) of the sequence that the row of token `tok` sees.
__device__ __forceinline__ int row_limit(const PackedTile& t, int causal, int tok) {
  return causal ? max(0, min(t.lk, tok + t.lk - t.lq + 1)) : t.lk;
}
// Steps of a half whose first row is token r: up to the last key its last row sees.
__device__ __forceinline__ int half_steps(const PackedTile& t, int causal, int r) {
  if (r >= t.lq) return 0;
  const int keys = min(t.ke, row_limit(t, causal, min(r + kHalf, t.lq) - 1)) - t.kb;
  return keys > 0 ? (keys + kKeys - 1) / kKeys : 0;
}

template <int DT, int D>
__global__ void __launch_bounds__(kThreads, 1)
    attn_packed_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                          const __grid_constant__ CUtensorMap tm_v, const PackedArgs a) {
  using C = Cfg<D>;
  constexpr int kStages = C::kStages;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  PackedSmem<D>& sm = *reinterpret_cast<PackedSmem<D>*>(smem_raw + pad);
  DevStatus* status = &g_attn_packed_status;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = blockIdx.x % a.Hq;
  grid_release();
  if (tid == 0) {
    sm.t = load_tile(a, blockIdx.x / a.Hq, 1);
    sm.abort = 0;
    sm.bad = 0;
    mbar_init(&sm.q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int s = 0; s < kStages / 2; ++s) mbar_init(&sm.v_ok[s], 2);
    for (int h = 0; h < 2; ++h) {
      mbar_init(&sm.s_full[h], 1);
      mbar_init(&sm.p_full[h][0], 4);
      mbar_init(&sm.p_full[h][1], 4);
      mbar_init(&sm.o_full[h], 1);
    }
    mbar_init(&sm.drain, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, 512);
    tmem_relinquish();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = sm.tmem_base;
  volatile int* abort = &sm.abort;
  const PackedTile t = sm.t;
  const int n0 = half_steps(t, a.causal, t.r0), n1 = half_steps(t, a.causal, t.r0 + kHalf);
  const int n = max(n0, n1);

  if (warp < 4) {
    // launched at 168 x 384 = 64512 registers: 128 x 40 + 256 x 232
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;\n" ::: "memory");
    if (warp == 0) {
      // ---------------------------------------------------------- producer
      if (lane == 0 && n > 0) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        const int kvh = head / a.G;
        const int halves = n1 > 0 ? 2 : 1;
        mbar_expect_tx(&sm.q_full, halves * C::kTileBytes);
        for (int h = 0; h < halves; ++h)
          for (int b = 0; b < C::kBlocks; ++b)
            tma_load_3d(sm.q[h] + b * C::kBlockBytes, &tm_q, b * 64, head, t.q0 + t.r0 + h * kHalf, &sm.q_full);
        int issued = 0;
        bool ok = true;
        for (int i = 0; i < 2 * n; ++i) {
          const int s = i % kStages;
          if (i >= kStages && !(ok = mbar_wait(&sm.empty[s], ((i / kStages) + 1) & 1, abort, status, 1))) break;
          mbar_expect_tx(&sm.full[s], C::kTileBytes);
          const int row = t.k0 + t.kb + (i >> 1) * kKeys;
          for (int b = 0; b < C::kBlocks; ++b)
            tma_load_3d(sm.kv[s] + b * C::kBlockBytes, (i & 1) ? &tm_v : &tm_k, b * 64, kvh, row, &sm.full[s]);
          issued = i + 1;
        }
        // on an abandoned run, let the copies already issued land
        if (!ok || *abort) {
          for (int i = max(0, issued - kStages); i < issued; ++i) {
            const long long c0 = clock64();
            while (!mbar_try_wait(&sm.full[i % kStages], (i / kStages) & 1) && clock64() - c0 < kWaitCycles / 4) {
            }
          }
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ---------------------------------------------------------- MMA issuer
      const uint32_t leader = elect_one();
      constexpr uint32_t id_qk = idesc_f16<DT>(kHalf, kKeys, false);
      constexpr uint32_t id_pv = idesc_f16<DT>(kHalf, D, true);
      auto issue_s = [&](int h, int stage) {
        const uint32_t qa = smem_u32(sm.q[h]), ka = smem_u32(sm.kv[stage]);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * C::kBlockBytes + (kk & 3) * 32;
          mma_f16_if(tbase + kColS + h * 128, desc_kmajor(qa + off), desc_kmajor(ka + off), id_qk, kk > 0, leader);
        }
        tc_commit_if(&sm.s_full[h], leader);
      };
      auto issue_pv = [&](int h, int stage, int j) {
        const uint32_t va = smem_u32(sm.kv[stage]);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          if (!mbar_wait(&sm.p_full[h][part], j & 1, abort, status, 6)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = 4 * part; kk < 4 * part + 4; ++kk)   // 16 keys = two groups of eight 128-byte rows
            mma_f16_ts_if(tbase + kColO + h * 128, tbase + kColS + h * 128 + kk * 8,
                          smem_desc(va + kk * 2048, C::kBlockBytes, 1024), id_pv, j > 0 || kk > 0, leader);
        }
        return true;
      };
      bool ok = n > 0 && mbar_wait(&sm.q_full, 0, abort, status, 2) && mbar_wait(&sm.full[0], 0, abort, status, 3);
      if (ok) {
        tc_fence_after();
        if (n0 > 0) issue_s(0, 0);
        if (n1 > 0) issue_s(1, 0);
        tc_commit_if(&sm.empty[0], leader);
      }
      for (int j = 0; ok && j < n; ++j) {
        const int sv = (2 * j + 1) % kStages, sk = (2 * j + 2) % kStages;
        const bool more = j + 1 < n;
        if (!(ok = mbar_wait(&sm.v_ok[j % (kStages / 2)], (j / (kStages / 2)) & 1, abort, status, 4))) break;
        if (more && !(ok = mbar_wait(&sm.full[sk], ((2 * j + 2) / kStages) & 1, abort, status, 5))) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int nh = h ? n1 : n0;
          if (ok && j < nh) {
            if (!(ok = issue_pv(h, sv, j))) break;
            if (j + 1 < nh) issue_s(h, sk);
            else tc_commit_if(&sm.o_full[h], leader);
          }
        }
        if (!ok) break;
        tc_commit_if(&sm.empty[sv], leader);
        if (more) tc_commit_if(&sm.empty[sk], leader);
      }
      // every MMA issued must finish before tensor memory is released
      tc_commit_if(&sm.drain, leader);
      const long long c0 = clock64();
      while (!mbar_try_wait(&sm.drain, 0) && clock64() - c0 < kWaitCycles) {
      }
      __syncwarp();
    } else {
      // ---------------------------------------------------------- V edges
      const int w = tid - 64;   // 0..63
      const int seen = row_limit(t, a.causal, t.r0);   // keys below are seen by every row of the CTA
      for (int j = 0; j < n; ++j) {
        const int i = 2 * j + 1, s = i % kStages;
        if (!warp_wait(&sm.full[s], (i / kStages) & 1, abort, status, 7)) break;
        const int key0 = t.kb + j * kKeys;
        if (key0 + kKeys > min(seen, t.lk)) {
          bool wrote = false, found = false;
          for (int c = w; c < kKeys * C::kBlocks * 8; c += 64) {
            const int r = (c >> 3) % kKeys;      // row of the tile (the swizzle stays inside a row)
            const int key = key0 + r;
            if (key < seen && key < t.lk) continue;
            uint4* p = reinterpret_cast<uint4*>(sm.kv[s] + c * 16);
            if (key >= t.lk) {
              *p = make_uint4(0, 0, 0, 0);
              wrote = true;
            } else {
              uint4 x = *p;
              uint32_t* u = reinterpret_cast<uint32_t*>(&x);
              bool hit = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (not_finite<DT>(u[e])) { u[e] &= 0xffff0000u; hit = true; }
                if (not_finite<DT>(u[e] >> 16)) { u[e] &= 0x0000ffffu; hit = true; }
              }
              if (hit) {
                *p = x;
                wrote = found = true;
              }
            }
          }
          if (found) sm.bad = 1;
          if (wrote) fence_proxy_async_smem();
        }
        warp_arrive(&sm.v_ok[j % (kStages / 2)], lane);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;\n" ::: "memory");
    // ------------------------------------------------------------ softmax
    const int h = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const int tok = t.r0 + h * kHalf + row;
    const uint32_t lb = tbase + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t ts = lb + kColS + h * 128, to = lb + kColO + h * 128;
    const int nh = h ? n1 : n0;
    const bool live = tok < t.lq && t.q0 + tok < a.Tq;
    const int lim = min(t.ke, row_limit(t, a.causal, min(tok, t.lq - 1)));
    const int warp_lim = min(t.ke, row_limit(t, a.causal, min(t.r0 + h * kHalf + (warp & 3) * 32, t.lq - 1)));
    const float sl2 = a.scale_log2;
    float m = -INFINITY, l0 = 0.f, l1 = 0.f;
    bool ok = true;
    for (int j = 0; j < nh; ++j) {
      if (!(ok = warp_wait(&sm.s_full[h], j & 1, abort, status, 8))) break;
      tc_fence_after();
      float x[kKeys];
#pragma unroll
      for (int c = 0; c < kKeys / 32; ++c) tmem_ld32(ts + 32 * c, *reinterpret_cast<float(*)[32]>(x + 32 * c));
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < kKeys / 32; ++c) reg_fence(*reinterpret_cast<float(*)[32]>(x + 32 * c));
      const int valid = lim - t.kb - j * kKeys;   // keys of this tile that the row sees
      if (warp_lim - t.kb - j * kKeys < kKeys) {
#pragma unroll
        for (int c = 0; c < kKeys; ++c)
          if (c >= valid) x[c] = -INFINITY;
      }
      float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
      for (int c = 0; c < kKeys; c += 8) {
        m0 = fmax3(m0, x[c], x[c + 1]);
        m1 = fmax3(m1, x[c + 2], x[c + 3]);
        m2 = fmax3(m2, x[c + 4], x[c + 5]);
        m3 = fmax3(m3, x[c + 6], x[c + 7]);
      }
      const float mt = fmax3(m0, m1, fmaxf(m2, m3)) * sl2;
      const bool grow = mt > m + (kRaise<DT> + kGrow<DT>) || (m == -INFINITY && mt > m);
      if (__any_sync(0xffffffffu, grow)) {
        const float al = grow ? ex2(m - (mt - kRaise<DT>)) : 1.f;   // 0 while m is -inf
        if (grow) m = mt - kRaise<DT>;
        l0 *= al;
        l1 *= al;
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tmem_ld32(to + 32 * c, o);
            tmem_ld_wait();
            reg_fence(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= al;
            tmem_st32(to + 32 * c, o);
          }
        }
      }
      const float base = m == -INFINITY ? 0.f : -m;
#pragma unroll
      for (int c = 0; c < kKeys / 32; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float p0 = base, p1 = base;
          fma2(p0, p1, x[32 * c + 2 * e], x[32 * c + 2 * e + 1], sl2, sl2);
          p0 = ex2(p0);
          p1 = ex2(p1);
          add2(l0, l1, p0, p1);
          w[e] = pack16<DT>(p0, p1);
        }
        tmem_st16(ts + 16 * c, w);
        if (c % 2 == 1) {
          tmem_st_wait();
          tc_fence_before();
          warp_arrive(&sm.p_full[h][c / 2], lane);
        }
      }
    }
    if (ok && nh > 0) ok = warp_wait(&sm.o_full[h], 0, abort, status, 9);
    tc_fence_after();
    const float l = l0 + l1;
    const bool bad = __any_sync(0xffffffffu, *static_cast<volatile int*>(&sm.bad) != 0);
    const bool part = t.slot >= 0;
    const float inv = part ? 1.f : l != 0.f ? __fdiv_rn(1.f, l) : 0.f;   // (l is NaN where a score was)
    const int64_t prow = (static_cast<int64_t>(t.slot) * a.Hq + head) * (2 * kHalf) + h * kHalf + row;
    if (__all_sync(0xffffffffu, ok && *abort == 0)) {
      if (bad && nh > 0) {
        // The infinite and NaN values of the edge tiles, for the rows that see
        // them.  All of the row before any of it is written: out may be q.
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + head * a.qsh + static_cast<int64_t>(t.q0 + tok) * a.qsn;
        const uint16_t* k0 = static_cast<const uint16_t*>(a.k) + (head / a.G) * a.ksh;
        const uint16_t* v0 = static_cast<const uint16_t*>(a.v) + (head / a.G) * a.vsh;
        const int end = live ? min(lim, a.Tk - t.k0) : 0;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          __syncwarp();
          float o[32];
          tmem_ld32(to + 32 * c, o);
          tmem_ld_wait();
          reg_fence(o);
          for (int key = max(t.kb, row_limit(t, a.causal, t.r0)); key < end; ++key) {
            const uint16_t* v = v0 + static_cast<int64_t>(t.k0 + key) * a.vsn + 32 * c;
            bool hit = false;
            for (int e = 0; e < 32; ++e) hit |= not_finite<DT>(v[e]);
            if (!hit) continue;
            const uint16_t* k = k0 + static_cast<int64_t>(t.k0 + key) * a.ksn;
            float s = 0.f;
            for (int e = 0; e < D; ++e) s = fmaf(value16<DT>(q[e]), value16<DT>(k[e]), s);
            const float p = ex2(fmaf(s, sl2, m == -INFINITY ? 0.f : -m));
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (not_finite<DT>(v[e])) o[e] = fmaf(p, value16<DT>(v[e]), o[e]);
          }
          __syncwarp();
          tmem_st32(to + 32 * c, o);
        }
        tmem_st_wait();
      }
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        __syncwarp();   // the lanes part below, and the load of tensor memory is one of the whole warp
        float o[32];
        if (nh > 0) {
          tmem_ld32(to + 32 * c, o);
          tmem_ld_wait();
          reg_fence(o);
        }
        if (nh == 0 || lim <= t.kb) {   // no key of this range
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (live && part) {
          float4* po = reinterpret_cast<float4*>(a.part_o + prow * D + 32 * c);
#pragma unroll
          for (int e = 0; e < 8; ++e) po[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        } else if (live) {
          uint4* po = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + head * a.osh +
                                               static_cast<int64_t>(t.q0 + tok) * a.osn + 32 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            po[e] = make_uint4(pack16<DT>(o[8 * e] * inv, o[8 * e + 1] * inv), pack16<DT>(o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                               pack16<DT>(o[8 * e + 4] * inv, o[8 * e + 5] * inv), pack16<DT>(o[8 * e + 6] * inv, o[8 * e + 7] * inv));
        }
      }
      if (live && part) *reinterpret_cast<float2*>(a.part_ml + prow * 2) = make_float2(m, l);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

// ---- host side ---------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// (rows, heads, D) 16-bit elements, box of 128 rows x 64 channels of one head
// in the 128-byte swizzle; rows outside read 0.
bool make_map(CUtensorMap* m, const void* base, int D, int heads, int rows, int64_t sh, int64_t sn) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads),
                        static_cast<cuuint64_t>(std::max(rows, 1))};
  // (the stride of a dimension of size 1 is never used: any valid value)
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(heads > 1 ? sh : D) * 2, static_cast<cuuint64_t>(rows > 1 ? sn : D) * 2};
  cuuint32_t box[3] = {64, 1, kHalf};
  cuuint32_t es[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DT, int D>
cudaError_t launch(const PackedArgs& a, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  if (!make_map(&mq, a.q, D, a.Hq, a.Tq, a.qsh, a.qsn) || !make_map(&mk, a.k, D, a.Hk, a.Tk, a.ksh, a.ksn) ||
      !make_map(&mv, a.v, D, a.Hk, a.Tk, a.vsh, a.vsn))
    return cudaErrorInvalidValue;
  auto k = attn_packed_tc_kernel<DT, D>;
  const int smem = static_cast<int>(sizeof(PackedSmem<D>)) + 1024;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  k<<<static_cast<unsigned>(a.n_tiles) * static_cast<unsigned>(a.Hq), kThreads, smem, st>>>(mq, mk, mv, a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attn_packed_tc(const PackedArgs& a, int dtype, cudaStream_t st) {
  if (dtype == VCATTN_DTYPE_BF16)
    return a.D == 128 ? launch<VCATTN_DTYPE_BF16, 128>(a, st) : launch<VCATTN_DTYPE_BF16, 64>(a, st);
  return a.D == 128 ? launch<VCATTN_DTYPE_F16, 128>(a, st) : launch<VCATTN_DTYPE_F16, 64>(a, st);
}

cudaError_t attn_packed_status(int* code, int* where, int* block, bool reset) {
  tc::DevStatus s{};
  cudaError_t e = cudaMemcpyFromSymbol(&s, g_attn_packed_status, sizeof(s));
  if (e != cudaSuccess) return e;
  *code = s.code;
  *where = s.where;
  *block = s.block;
  if (reset) {
    tc::DevStatus z{};
    e = cudaMemcpyToSymbol(g_attn_packed_status, &z, sizeof(z));
  }
  return e;
}

}  // namespace vcattn
