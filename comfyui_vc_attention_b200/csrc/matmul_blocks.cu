// E4M3 matrix product with block scales, fp32 result rounded once:
//   C[m, n] = sum_kb sa[m, kb] sb[n / 128, kb] sum_{k in kb} A[m, k] B[n, k]  (+ bias[n])
// with kb running over blocks of 128 columns (the last one may be short).
//
// tcgen05 kind::f8f6f4: each k-block of 128 is one accumulation of four MMAs in
// tensor memory, in one of two or four buffers; the promotion warps read the
// finished block sum and add it to fp32 registers with its scale while the next
// block runs.  Thread = output row (TMEM lane) and 64 columns, so the scale of a
// block is one scalar per thread.
//   warp 0       TMA producer        warp 1   MMA issuer, tensor-memory owner
//   warps 2-3    sa * sb of four k-blocks at a time, in two groups in shared
//                memory, the next group's loads in flight
//   warps 4-     promotion and output
// 16384 x 7168 x 5376: 577-593 us (2.1-2.2 PFLOP/s) in short runs and 674 at the
// power cap; 523 without the promotion, 410 without the loads (48 KB per k-block and
// SM from L2, 13.5 TB/s over all).  Eight promotion warps of 128 columns whose
// scales came from global memory took 1050 us.
#include <cuda.h>
#include <mutex>
#include <string>

#include "kernels.cuh"
#include "launch.cuh"
#include "tc_common.cuh"
#include "tc_math.cuh"

namespace vcattn {

__device__ tc::DevStatus g_matmul_status;

namespace {

using namespace tc;

constexpr int kBM = 128;
constexpr int kBK = 128;   // columns of a k-block

struct MatmulArgs {
  const float *sa, *sb;
  int64_t sam, sak, sbn, sbk;
  const float* bias;
  void* out;
  int64_t ldo;
  int M, N, kb;
  int mt, nt, tiles, group;
  int vec_out;   // rows of `out` start on 16-byte boundaries
  int ranks;     // CTAs of a cluster that share a tile's k-blocks (1: persistent CTAs over whole tiles)
  // Persistent CTAs: `full` tiles run whole (a multiple of the grid); each of
  // the others is split in `parts` ranges of k-blocks (1: whole), whose sums go
  // to `part`.
  int full, parts;
  float* part;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(const float* p, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(a) : "memory");
  return v;
}

template <int ODT> __device__ __forceinline__ void store1(void* out, int64_t i, float v) {
  if constexpr (ODT == VCATTN_DTYPE_BF16) static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  else if constexpr (ODT == VCATTN_DTYPE_F16) static_cast<__half*>(out)[i] = __float2half_rn(v);
  else static_cast<float*>(out)[i] = v;
}

constexpr int kGroup = 4;   // k-blocks whose scales change hands together (two groups in shared memory)

template <int BN> struct MmCfg {
  static constexpr int kStages = BN == 256 ? 3 : 5;
  static constexpr int kPromo = BN / 64 * 4;               // promotion warps
  static constexpr int kThreads = 128 + 32 * kPromo;
  static constexpr int kBufs = 512 / BN;                   // block sums in tensor memory
  // Output staging of a warp: 32 bytes of each of its 32 rows at a time, 16
  // bytes apart so that the rows start in different banks.
  static constexpr int kOutPitch = 128 + 16;
  static constexpr int kPartPitch = BN + 4;   // floats of a row of a rank's sums
  static_assert(kBM * kPartPitch * 4 <= kStages * kBM * kBK + kStages * BN * kBK, "a rank's sums fit over the stages");
};

template <int BN> struct MmSmem {
  alignas(1024) uint8_t a[MmCfg<BN>::kStages][kBM * kBK];
  alignas(1024) uint8_t b[MmCfg<BN>::kStages][BN * kBK];
  alignas(16) uint8_t out[MmCfg<BN>::kPromo][32 * MmCfg<BN>::kOutPitch];
  alignas(16) float scale[2][BN / 128][kBM][kGroup];
  alignas(8) uint64_t full[MmCfg<BN>::kStages];
  alignas(8) uint64_t empty[MmCfg<BN>::kStages];
  alignas(8) uint64_t t_full[MmCfg<BN>::kBufs];
  alignas(8) uint64_t t_empty[MmCfg<BN>::kBufs];
  alignas(8) uint64_t s_full[2];
  alignas(8) uint64_t s_empty[2];
  alignas(8) uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

// Tile t of the launch order: groups of `group` row tiles, rows fastest, so the
// tiles that run together share their A and B panels in L2.
__device__ __forceinline__ void tile_coords(const MatmulArgs& a, int t, int& m, int& n) {
  const int per = a.group * a.nt;
  const int g = t / per, r = t - g * per;
  const int rows = min(a.group, a.mt - g * a.group);
  n = r / rows;
  m = g * a.group + (r - n * rows);
}

// How a tile is shared: not at all, its k-blocks by the CTAs of a cluster, or
// (the tiles of the last round) in parts that a second kernel joins.
enum Share { kWhole, kCluster, kParts };

// The pieces of work of a CTA, one after the other: k-blocks [k0, k1) of a
// tile, and which part of it that is (-1: all of it, or a cluster's share).
template <Share SHARE> struct Pieces;
template <> struct Pieces<kWhole> {
  int t = blockIdx.x;
  __device__ __forceinline__ explicit Pieces(const MatmulArgs&) {}
  __device__ __forceinline__ bool any(const MatmulArgs& a) const { return t < a.tiles; }
  __device__ __forceinline__ void next(const MatmulArgs&) { t += gridDim.x; }
  __device__ __forceinline__ int tile() const { return t; }
  __device__ __forceinline__ int k0() const { return 0; }
  __device__ __forceinline__ int k1(const MatmulArgs& a) const { return a.kb; }
  __device__ __forceinline__ int part() const { return -1; }
};
template <> struct Pieces<kCluster> {
  int t, b, e;
  __device__ __forceinline__ explicit Pieces(const MatmulArgs& a) {
    const int rank = static_cast<int>(cluster_rank());
    t = blockIdx.x / a.ranks;
    b = static_cast<int>(static_cast<int64_t>(a.kb) * rank / a.ranks);
    e = static_cast<int>(static_cast<int64_t>(a.kb) * (rank + 1) / a.ranks);
  }
  __device__ __forceinline__ bool any(const MatmulArgs& a) const { return t < a.tiles; }
  __device__ __forceinline__ void next(const MatmulArgs& a) { t = a.tiles; }
  __device__ __forceinline__ int tile() const { return t; }
  __device__ __forceinline__ int k0() const { return b; }
  __device__ __forceinline__ int k1(const MatmulArgs&) const { return e; }
  __device__ __forceinline__ int part() const { return -1; }
};
template <> struct Pieces<kParts> {
  int u, t, b, e, p;
  __device__ __forceinline__ explicit Pieces(const MatmulArgs& a) : u(blockIdx.x) { place(a); }
  __device__ __forceinline__ void place(const MatmulArgs& a) {
    t = u;
    b = 0;
    e = a.kb;
    p = -1;
    if (u >= a.full) {
      t = a.full + (u - a.full) / a.parts;
      p = (u - a.full) % a.parts;
      b = static_cast<int>(static_cast<int64_t>(a.kb) * p / a.parts);
      e = static_cast<int>(static_cast<int64_t>(a.kb) * (p + 1) / a.parts);
    }
  }
  __device__ __forceinline__ bool any(const MatmulArgs& a) const { return t < a.tiles; }
  __device__ __forceinline__ void next(const MatmulArgs& a) {
    u += gridDim.x;
    place(a);
  }
  __device__ __forceinline__ int tile() const { return t; }
  __device__ __forceinline__ int k0() const { return b; }
  __device__ __forceinline__ int k1(const MatmulArgs&) const { return e; }
  __device__ __forceinline__ int part() const { return p; }
};

template <int BN, int ODT, Share SHARE>
__global__ void __launch_bounds__(MmCfg<BN>::kThreads, 1)
    matmul_blocks_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                         const MatmulArgs a) {
  using Cfg = MmCfg<BN>;
  constexpr int kStages = Cfg::kStages, kBufs = Cfg::kBufs;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  MmSmem<BN>& sm = *reinterpret_cast<MmSmem<BN>*>(smem_raw + pad);
  DevStatus* status = &g_matmul_status;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    sm.abort = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < Cfg::kBufs; ++b) {
      mbar_init(&sm.t_full[b], 1);
      mbar_init(&sm.t_empty[b], Cfg::kPromo);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.s_full[b], 2);
      mbar_init(&sm.s_empty[b], Cfg::kPromo);
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
  if constexpr (SHARE == kParts) grid_release();
  if (warp < 4) {
  // BN = 256 is launched at 96 x 640 = 61440 registers: 128 x 56 + 512 x 104 = 60416
  if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n" ::: "memory");
  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_tmap(&tm_a);
      prefetch_tmap(&tm_b);
      int it = 0;
      bool ok = true;
      for (Pieces<SHARE> pc(a); ok && pc.any(a); pc.next(a)) {
        int m, n;
        tile_coords(a, pc.tile(), m, n);
        for (int k = pc.k0(); k < pc.k1(a); ++k, ++it) {
          const int s = it % kStages;
          if (it >= kStages && !(ok = mbar_wait(&sm.empty[s], ((it / kStages) + 1) & 1, abort, status, 1))) break;
          mbar_expect_tx(&sm.full[s], (kBM + BN) * kBK);
          tma_load_2d(sm.a[s], &tm_a, k * kBK, m * kBM, &sm.full[s]);
          tma_load_2d(sm.b[s], &tm_b, k * kBK, n * BN, &sm.full[s]);
        }
      }
      // on an abandoned run, let the copies already issued land
      if (!ok || *abort) {
        for (int j = max(0, it - kStages); j < it; ++j) {
          const long long c0 = clock64();
          while (!mbar_try_wait(&sm.full[j % kStages], (j / kStages) & 1) && clock64() - c0 < kWaitCycles / 4) {
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t leader = elect_one();
    const uint32_t idesc = idesc_e4m3(kBM, BN, false);
    int it = 0;
    bool ok = true;
    for (Pieces<SHARE> pc(a); ok && pc.any(a); pc.next(a)) {
      for (int k = pc.k0(); k < pc.k1(a); ++k, ++it) {
        const int s = it % kStages, b = it % kBufs;
        if (it >= kBufs && !(ok = mbar_wait(&sm.t_empty[b], ((it / kBufs) + 1) & 1, abort, status, 2))) break;
        if (!(ok = mbar_wait(&sm.full[s], (it / kStages) & 1, abort, status, 3))) break;
        tc_fence_after();
        const uint32_t aa = smem_u32(sm.a[s]), ba = smem_u32(sm.b[s]);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_f8_if(tbase + b * BN, desc_kmajor(aa + kk * 32), desc_kmajor(ba + kk * 32), idesc, kk > 0, leader);
        tc_commit_if(&sm.t_full[b], leader);
        tc_commit_if(&sm.empty[s], leader);
      }
    }
    // every MMA issued must finish before tensor memory is released
    tc_commit_if(&sm.drain, leader);
    const long long c0 = clock64();
    while (!mbar_try_wait(&sm.drain, 0) && clock64() - c0 < kWaitCycles) {
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ scales
    const int r = tid - 64;   // rows r and r + 64
    int grp = 0;              // groups handed over
    bool ok = true;
    for (Pieces<SHARE> pc(a); ok && pc.any(a); pc.next(a)) {
      int mt, nt;
      tile_coords(a, pc.tile(), mt, nt);
      // (rows and columns past the matrix take the scale of the last one: nothing of them is written)
      const float* sa0 = a.sa + static_cast<int64_t>(min(mt * kBM + r, a.M - 1)) * a.sam;
      const float* sa1 = a.sa + static_cast<int64_t>(min(mt * kBM + r + 64, a.M - 1)) * a.sam;
      const float* sb = a.sb + static_cast<int64_t>(nt) * (BN / 128) * a.sbn;
      const int64_t sb1 = (nt * BN + 128 < a.N) ? a.sbn : 0;
      float x0[kGroup], x1[kGroup], y0[kGroup], y1[kGroup];
      auto load = [&](int k) {
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
          const int kk = min(k + u, pc.k1(a) - 1);
          x0[u] = __ldg(sa0 + kk * a.sak);
          x1[u] = __ldg(sa1 + kk * a.sak);
          y0[u] = __ldg(sb + kk * a.sbk);
          if constexpr (BN == 256) y1[u] = __ldg(sb + sb1 + kk * a.sbk);
        }
      };
      load(pc.k0());
      for (int k = pc.k0(); k < pc.k1(a); k += kGroup, ++grp) {
        const int s = grp & 1;
        if (grp >= 2 && !(ok = warp_wait(&sm.s_empty[s], ((grp >> 1) + 1) & 1, abort, status, 5))) break;
        *reinterpret_cast<float4*>(sm.scale[s][0][r]) = make_float4(x0[0] * y0[0], x0[1] * y0[1], x0[2] * y0[2], x0[3] * y0[3]);
        *reinterpret_cast<float4*>(sm.scale[s][0][r + 64]) = make_float4(x1[0] * y0[0], x1[1] * y0[1], x1[2] * y0[2], x1[3] * y0[3]);
        if constexpr (BN == 256) {
          *reinterpret_cast<float4*>(sm.scale[s][1][r]) = make_float4(x0[0] * y1[0], x0[1] * y1[1], x0[2] * y1[2], x0[3] * y1[3]);
          *reinterpret_cast<float4*>(sm.scale[s][1][r + 64]) = make_float4(x1[0] * y1[0], x1[1] * y1[1], x1[2] * y1[2], x1[3] * y1[3]);
        }
        warp_arrive(&sm.s_full[s], lane);
        if (k + kGroup < pc.k1(a)) load(k + kGroup);   // in flight while the promotion works on this group
      }
    }
  }
  } else {
    if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;\n" ::: "memory");
    // ------------------------------------------------------------ promotion and output
    const int wq = warp & 3, quarter = (warp - 4) >> 2;   // 32 rows x 64 columns
    const uint32_t lb = tbase + (static_cast<uint32_t>(wq * 32) << 16) + quarter * 64;
    constexpr int ES = ODT == VCATTN_DTYPE_F32 ? 4 : 2;
    uint8_t* stage = sm.out[warp - 4];
    const float* scale = sm.scale[0][quarter >> 1][wq * 32 + lane];
    uint32_t b = 0, b_par = 0, g = 0, g_par = 0;   // tensor-memory buffer and scale group, and their phases
    bool ok = true;
    for (Pieces<SHARE> pc(a); ok && pc.any(a); pc.next(a)) {
      int mt, nt;
      tile_coords(a, pc.tile(), mt, nt);
      const int m0 = mt * kBM + wq * 32, n0 = nt * BN + quarter * 64;
      float acc[64];
#pragma unroll
      for (int c = 0; c < 64; ++c) acc[c] = 0.f;
      for (int k = pc.k0(); k < pc.k1(a); k += kGroup) {
        // (The lanes of a warp may learn at different times that a wait was given
        // up, so none leaves the loop for it: the waits return at once from then
        // on, and the vote below ends the work.  A vote or a break here costs 8 %.)
        mbar_wait(&sm.s_full[g], g_par, abort, status, 4);
        const float4 s4 = *reinterpret_cast<const float4*>(scale + g * (BN / 128 * kBM * kGroup));
        warp_arrive(&sm.s_empty[g], lane);
        g ^= 1;
        g_par ^= g ^ 1;   // (flips when g returns to 0)
        const float s[kGroup] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
          if (k + u >= pc.k1(a)) break;
          mbar_wait(&sm.t_full[b], b_par, abort, status, 6);
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x[32];
            tmem_ld32(lb + b * BN + h * 32, x);
            tmem_ld_wait();
            reg_fence(x);
            if (h == 1) {
              tc_fence_before();
              warp_arrive(&sm.t_empty[b], lane);
            }
#pragma unroll
            for (int c = 0; c < 32; c += 2) fma2(acc[h * 32 + c], acc[h * 32 + c + 1], x[c], x[c + 1], s[u], s[u]);
          }
          b = (b + 1) % kBufs;
          b_par ^= b == 0;
        }
      }
      ok = __all_sync(0xffffffffu, *abort == 0);
      if (!ok) continue;
      if constexpr (SHARE == kCluster) {
        // this rank's sums over the operand stages (every MMA has read them)
        float* part = reinterpret_cast<float*>(sm.a) + (wq * 32 + lane) * Cfg::kPartPitch + quarter * 64;
#pragma unroll
        for (int c = 0; c < 64; c += 4) *reinterpret_cast<float4*>(part + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
        continue;
      }
      if (SHARE == kParts && pc.part() >= 0) {
        // part of a tile: [tile, part][warp][column / 4][lane], four columns each
        float4* dst = reinterpret_cast<float4*>(a.part) +
                      ((static_cast<int64_t>(pc.tile() - a.full) * a.parts + pc.part()) * Cfg::kPromo + (warp - 4)) * 16 * 32 + lane;
#pragma unroll
        for (int c = 0; c < 16; ++c) dst[c * 32] = make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
        continue;
      }
      if (a.bias != nullptr) {
        // this warp's 64 values, two per lane (one coalesced load each), then
        // from lane to lane: 64 loads per thread cost 8 us (333 x 14336 x 5376,
        // the same inputs each time: 53 against 45; rotated inputs: 49.6)
        const float b0 = n0 + lane < a.N ? __ldg(a.bias + n0 + lane) : 0.f;
        const float b1 = n0 + 32 + lane < a.N ? __ldg(a.bias + n0 + 32 + lane) : 0.f;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          acc[c] += __shfl_sync(0xffffffffu, b0, c);
          acc[32 + c] += __shfl_sync(0xffffffffu, b1, c);
        }
      }
      // rows through shared memory, so that whole 32-byte sectors go out
      constexpr int PC = 128 / ES;   // columns per pass
#pragma unroll
      for (int p = 0; p < 64 / PC; ++p) {
        const int np = n0 + p * PC;
#pragma unroll
        for (int c = 0; c < PC; c += 16 / ES) {
          uint4 w;
#pragma unroll
          for (int e = 0; e < 16 / ES; e += 2) {
            stage2<ODT>(reinterpret_cast<uint8_t*>(&w) + e * ES, acc[p * PC + c + e], acc[p * PC + c + e + 1]);
          }
          *reinterpret_cast<uint4*>(stage + lane * Cfg::kOutPitch + c * ES) = w;
        }
        __syncwarp();
        const int c = (lane & 7) * (16 / ES), cols = a.N - np;   // 16-byte chunk of a row
#pragma unroll
        for (int r = lane >> 3; r < 32; r += 4) {
          if (m0 + r >= a.M || c >= cols) continue;
          const uint8_t* src = stage + r * Cfg::kOutPitch + c * ES;
          uint8_t* dst = static_cast<uint8_t*>(a.out) + (static_cast<int64_t>(m0 + r) * a.ldo + np + c) * ES;
          if (a.vec_out && c + 16 / ES <= cols) {
            *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
          } else {
            for (int e = 0; e < 16 / ES && c + e < cols; ++e) {
              if constexpr (ES == 2) reinterpret_cast<uint16_t*>(dst)[e] = reinterpret_cast<const uint16_t*>(src)[e];
              else reinterpret_cast<uint32_t*>(dst)[e] = reinterpret_cast<const uint32_t*>(src)[e];
            }
          }
        }
        __syncwarp();
      }
    }
  }
  __syncthreads();
  if (warp == 1) tmem_dealloc(tbase, 512);
  if constexpr (SHARE == kCluster) {
    // every rank adds the parts of its share of the rows, in rank order
    __syncwarp();
    cluster_sync();
    int mt, nt;
    tile_coords(a, blockIdx.x / a.ranks, mt, nt);
    const int rank = static_cast<int>(cluster_rank());
    const int rows = *abort ? 0 : min(kBM, a.M - mt * kBM);
    for (int r = rank * (Cfg::kThreads / 32) + warp; r < rows; r += a.ranks * (Cfg::kThreads / 32)) {
      for (int c = lane * 4; c < BN; c += 128) {
        const int n = nt * BN + c;
        if (n >= a.N) continue;
        const float* p = reinterpret_cast<const float*>(sm.a) + r * Cfg::kPartPitch + c;
        float4 v = ld_cluster4(p, 0);
        for (int q = 1; q < a.ranks; ++q) {
          const float4 w = ld_cluster4(p, q);
          v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
        }
        const float e[4] = {v.x, v.y, v.z, v.w};
        const int64_t o = static_cast<int64_t>(mt * kBM + r) * a.ldo + n;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < a.N) store1<ODT>(a.out, o + i, e[i] + (a.bias != nullptr ? __ldg(a.bias + n + i) : 0.f));
      }
    }
    __syncwarp();
    cluster_sync();   // no CTA leaves while another reads its part
  }
}

// Adds the parts of the split tiles (128 x 256) in k order: one CTA per 32 rows
// and 64 columns.
template <int ODT>
__global__ void __launch_bounds__(128) matmul_blocks_join_kernel(const MatmulArgs a) {
  grid_wait();   // the parts
  constexpr int kPromo = MmCfg<256>::kPromo, ES = ODT == VCATTN_DTYPE_F32 ? 4 : 2;
  __shared__ float rows[32][64 + 4];
  const int tile = blockIdx.x / kPromo, w = blockIdx.x % kPromo, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float4* src = reinterpret_cast<const float4*>(a.part) +
                      (static_cast<int64_t>(tile) * a.parts * kPromo + w) * 16 * 32 + warp * 4 * 32 + lane;
  float4 v[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = src[c * 32];
#pragma unroll 4
  for (int p = 1; p < a.parts; ++p) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float4 x = src[static_cast<int64_t>(p) * kPromo * 16 * 32 + c * 32];
      v[c].x += x.x; v[c].y += x.y; v[c].z += x.z; v[c].w += x.w;
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) *reinterpret_cast<float4*>(&rows[lane][(warp * 4 + c) * 4]) = v[c];
  __syncthreads();
  int mt, nt;
  tile_coords(a, a.full + tile, mt, nt);
  const int r = threadIdx.x >> 2, c0 = (threadIdx.x & 3) * 16;
  const int m = mt * kBM + (w & 3) * 32 + r, n = nt * 256 + (w >> 2) * 64 + c0;
  if (m >= a.M || n >= a.N) return;
  const int64_t o = static_cast<int64_t>(m) * a.ldo + n;
  float y[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) y[e] = rows[r][c0 + e] + (a.bias != nullptr && n + e < a.N ? __ldg(a.bias + n + e) : 0.f);
  if (a.vec_out && n + 16 <= a.N) {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.out) + o * ES);
#pragma unroll
    for (int q = 0; q < ES; ++q) {
      uint4 u;
#pragma unroll
      for (int e = 0; e < 16 / ES; e += 2)
        stage2<ODT>(reinterpret_cast<uint8_t*>(&u) + e * ES, y[q * (16 / ES) + e], y[q * (16 / ES) + e + 1]);
      dst[q] = u;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (n + e < a.N) store1<ODT>(a.out, o + e, y[e]);
  }
}

// ---- few rows ------------------------------------------------------------------
// For M up to 32 the weight's bytes bound the product.  Here the weight rows
// are the MMA's 128 rows and the activations its MN columns, and the k-blocks
// of a row tile are dealt to the CTAs of a cluster, so that every SM streams
// weights; the partial sums meet in shared memory of the cluster and are added
// in rank order.
//   warp 0  TMA producer     warp 1  MMA issuer     warps 4-7  promotion, output
constexpr int kFewStages = 4;

struct FewArgs {
  const float *sa, *sb;
  int64_t sam, sak, sbn, sbk;
  const float* bias;
  void* out;
  int64_t ldo;
  int M, N, kb;
};

template <int MN> struct FewSmem {
  alignas(1024) uint8_t w[kFewStages][128 * kBK];   // at the end: this CTA's sums, [activation row][weight row] fp32
  alignas(1024) uint8_t x[kFewStages][MN * kBK];
  alignas(16) float scale[2][MN];             // sa * sb of a k-block
  alignas(8) uint64_t full[kFewStages];
  alignas(8) uint64_t empty[kFewStages];
  alignas(8) uint64_t t_full[2];
  alignas(8) uint64_t t_empty[2];
  alignas(8) uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

template <int MN, int ODT>
__global__ void __launch_bounds__(256, MN == 16 ? 3 : 2)
    matmul_blocks_few_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                             const FewArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  FewSmem<MN>& sm = *reinterpret_cast<FewSmem<MN>*>(smem_raw + pad);
  DevStatus* status = &g_matmul_status;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ranks = cluster_size(), rank = cluster_rank();
  const int tile = blockIdx.x / ranks;
  // this CTA's k-blocks
  const int k0 = static_cast<int>(static_cast<int64_t>(a.kb) * rank / ranks);
  const int nk = static_cast<int>(static_cast<int64_t>(a.kb) * (rank + 1) / ranks) - k0;
  constexpr uint32_t kCols = 2 * MN < 32 ? 32 : 2 * MN;
  if (tid == 0) {
    sm.abort = 0;
    for (int s = 0; s < kFewStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.t_full[b], 1);
      mbar_init(&sm.t_empty[b], 4);
    }
    mbar_init(&sm.drain, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, kCols);
    tmem_relinquish();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = sm.tmem_base;
  volatile int* abort = &sm.abort;

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&tm_w);
      prefetch_tmap(&tm_x);
      int it = 0;
      bool ok = true;
      for (; it < nk; ++it) {
        const int s = it % kFewStages;
        if (it >= kFewStages && !(ok = mbar_wait(&sm.empty[s], ((it / kFewStages) + 1) & 1, abort, status, 11))) break;
        mbar_expect_tx(&sm.full[s], (128 + MN) * kBK);
        tma_load_2d(sm.w[s], &tm_w, (k0 + it) * kBK, tile * 128, &sm.full[s]);
        tma_load_2d(sm.x[s], &tm_x, (k0 + it) * kBK, 0, &sm.full[s]);
      }
      if (!ok || *abort) {
        for (int j = max(0, it - kFewStages); j < it; ++j) {
          const long long t0 = clock64();
          while (!mbar_try_wait(&sm.full[j % kFewStages], (j / kFewStages) & 1) && clock64() - t0 < kWaitCycles / 4) {
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t leader = elect_one();
    constexpr uint32_t idesc = idesc_e4m3(128, MN, false);
    for (int it = 0; it < nk; ++it) {
      const int s = it % kFewStages, b = it & 1;
      if (it >= 2 && !mbar_wait(&sm.t_empty[b], ((it >> 1) + 1) & 1, abort, status, 12)) break;
      if (!mbar_wait(&sm.full[s], (it / kFewStages) & 1, abort, status, 13)) break;
      tc_fence_after();
      const uint32_t wa = smem_u32(sm.w[s]), xa = smem_u32(sm.x[s]);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        mma_f8_if(tbase + b * MN, desc_kmajor(wa + kk * 32), desc_kmajor(xa + kk * 32), idesc, kk > 0, leader);
      tc_commit_if(&sm.t_full[b], leader);
      tc_commit_if(&sm.empty[s], leader);
    }
    tc_commit_if(&sm.drain, leader);
    const long long t0 = clock64();
    while (!mbar_try_wait(&sm.drain, 0) && clock64() - t0 < kWaitCycles) {
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int wq = warp & 3, row = wq * 32 + lane;   // weight row of the tile
    const uint32_t lb = tbase + (static_cast<uint32_t>(wq * 32) << 16);
    const int p = tid - 128;
    // thread p < MN brings the scale of activation row p, one block ahead
    const float* sa = a.sa + static_cast<int64_t>(min(p, a.M - 1)) * a.sam + k0 * a.sak;
    const float* sb = a.sb + static_cast<int64_t>(tile) * a.sbn + k0 * a.sbk;
    float acc[MN], xs = 0.f, ys = 0.f;
    bool ok = true;
#pragma unroll
    for (int c = 0; c < MN; ++c) acc[c] = 0.f;
    if (p < MN && nk > 0) {
      xs = __ldg(sa);
      ys = __ldg(sb);
    }
    for (int it = 0; it < nk; ++it) {
      const int b = it & 1;
      if (p < MN) {
        sm.scale[b][p] = xs * ys;
        if (it + 1 < nk) {
          xs = __ldg(sa + (it + 1) * a.sak);
          ys = __ldg(sb + (it + 1) * a.sbk);
        }
      }
      asm volatile("bar.sync 1, 128;\n" ::: "memory");   // the scales of this block are written, those of it - 1 read
      // (a warp that gave up keeps step with the others' barrier)
      ok = ok && warp_wait(&sm.t_full[b], (it >> 1) & 1, abort, status, 14);
      tc_fence_after();
      float x[MN];
#pragma unroll
      for (int c = 0; c < MN; c += 16) tmem_ld16(lb + b * MN + c, *reinterpret_cast<float(*)[16]>(x + c));
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < MN; c += 16) reg_fence16(*reinterpret_cast<float(*)[16]>(x + c));
      tc_fence_before();
      warp_arrive(&sm.t_empty[b], lane);
#pragma unroll
      for (int c = 0; c < MN; c += 4) {
        const float4 s = *reinterpret_cast<const float4*>(&sm.scale[b][c]);
        fma2(acc[c], acc[c + 1], x[c], x[c + 1], s.x, s.y);
        fma2(acc[c + 2], acc[c + 3], x[c + 2], x[c + 3], s.z, s.w);
      }
    }
#pragma unroll
    // (every MMA has read its weights: t_full of the last block is through)
    for (int c = 0; c < MN; ++c) reinterpret_cast<float*>(sm.w)[c * 128 + row] = acc[c];
  }
  __syncthreads();
  if (warp == 1) tmem_dealloc(tbase, kCols);
  cluster_sync();
  // each rank adds the parts of its share of the (row, column) pairs, columns fastest
  const int all = min(MN, a.M) * 128;
  const bool dead = *abort != 0;
  for (int i = rank * 256 + tid; i < all && !dead; i += ranks * 256) {
    const int m = i >> 7, c = i & 127, n = tile * 128 + c;
    if (n >= a.N) continue;
    float v = 0.f, part[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) part[r] = r < ranks ? ld_cluster(reinterpret_cast<const float*>(sm.w) + i, r) : 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) v += part[r];
    if (a.bias != nullptr) v += __ldg(a.bias + n);
    const int64_t o = static_cast<int64_t>(m) * a.ldo + n;
    store1<ODT>(a.out, o, v);
  }
  __syncwarp();
  cluster_sync();   // no CTA leaves while another reads its part
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

// (rows, K) bytes, row pitch ld, box of box_rows x 128 columns in the 128-byte swizzle; outside reads 0.
bool make_map(CUtensorMap* m, const void* base, int64_t rows, int64_t K, int64_t ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {kBK, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t es[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Which kernel runs a product, and how its tiles are shared out.
struct Plan {
  enum { kFew16, kFew32, kWide, kNarrow, kShared } kind;
  int ranks = 1, full = 0, parts = 1;
  size_t workspace = 0;   // partial sums
};

Plan plan_product(int64_t M, int64_t N, int64_t kb) {
  Plan p{};
  // Few rows: the kernel that streams the weight.  K = 5376, N = 7168: 16 rows
  // 13.0 us, 32 rows 14.4, 128-row tiles 16.4 (the form for 64 rows took 21).  Wide
  // weights bring both sides together: N = 14336, 24 rows 20.6 against 27.8, 32 rows
  // 22.4 against 20.5; N = 28672, 36.6 against 37.8 and 37.8 against 33.1.
  if (M <= 32) {
    p.kind = M <= 16 ? Plan::kFew16 : Plan::kFew32;
    return p;
  }
  // Time on the busiest SM in k-blocks of a 128 x 256 tile.  A 128 x 128 tile
  // takes 0.55 of that (it reads twice the A bytes per MMA).  The last, partial
  // round of 256-column tiles is split along K over all SMs where that takes
  // more than 40 k-blocks off it: about 22 go to partial sums and their join,
  // and few tiles alone run faster than a full round (1000 x 5376 x 14336: 168
  // tiles, 148 whole and 20 in seven parts, 103 -> 84 us; 4096 x 7168 x 5376,
  // 39 k-blocks, 156 -> 166 us if it were split).
  const int64_t sms = sm_count(), mt = (M + 127) / 128;
  const int64_t t256 = mt * ((N + 255) / 256), t128 = mt * ((N + 127) / 128);
  const int64_t rest = t256 % sms, parts = rest ? min(sms / rest, kb / 2) : 1;
  int64_t wide = (t256 + sms - 1) / sms * kb;
  const int64_t saved = kb - (parts > 0 ? (kb + parts - 1) / parts : kb);
  if (t256 > sms && saved > 40) {
    wide -= saved - 22;
    p.full = static_cast<int>(t256 - rest);
    p.parts = static_cast<int>(parts);
    p.workspace = static_cast<size_t>(rest) * parts * 128 * 256 * sizeof(float);
  }
  if (20 * wide <= 11 * ((t128 + sms - 1) / sms) * kb) {
    p.kind = Plan::kWide;
    return p;
  }
  p = Plan{};
  // Tiles for less than half of the SMs: clusters share their k-blocks.
  p.ranks = static_cast<int>(min(min(sms / t128, int64_t{8}), kb / 4));
  p.kind = p.ranks >= 2 ? Plan::kShared : Plan::kNarrow;
  return p;
}

struct Operands {
  const uint8_t *a, *b;
  int64_t lda, ldb, K;
};

template <typename K, typename A>
cudaError_t launch_cluster(K kernel, unsigned ctas, int threads, int smem, int ranks, cudaStream_t st,
                           const CUtensorMap& m0, const CUtensorMap& m1, const A& a) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ranks;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, m0, m1, a);
}

template <int BN, int ODT, Share SHARE>
cudaError_t launch(const Operands& op, MatmulArgs a, const Plan& plan, cudaStream_t st) {
  CUtensorMap ma, mb;
  if (!make_map(&ma, op.a, a.M, op.K, op.lda, kBM) || !make_map(&mb, op.b, a.N, op.K, op.ldb, BN))
    return cudaErrorInvalidValue;
  a.mt = (a.M + kBM - 1) / kBM;
  a.nt = (a.N + BN - 1) / BN;
  a.tiles = a.mt * a.nt;
  a.group = 16;
  a.ranks = plan.ranks;
  a.full = plan.full;
  a.parts = plan.parts;
  auto k = matmul_blocks_kernel<BN, ODT, SHARE>;
  const int smem = static_cast<int>(sizeof(MmSmem<BN>)) + 1024;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  if constexpr (SHARE == kCluster)
    return launch_cluster(k, static_cast<unsigned>(a.tiles) * plan.ranks, MmCfg<BN>::kThreads, smem, plan.ranks, st, ma, mb, a);
  k<<<static_cast<unsigned>(min(a.tiles, sm_count())), MmCfg<BN>::kThreads, smem, st>>>(ma, mb, a);
  e = cudaGetLastError();
  if constexpr (SHARE == kParts) {
    if (e == cudaSuccess)
      e = launch_after(matmul_blocks_join_kernel<ODT>, dim3((a.tiles - a.full) * MmCfg<256>::kPromo), 128, 0, st, true, a);
  }
  return e;
}

template <int MN, int ODT>
cudaError_t launch_few(const Operands& op, const MatmulArgs& m, cudaStream_t st) {
  CUtensorMap mw, mx;
  if (!make_map(&mw, op.b, m.N, op.K, op.ldb, 128) || !make_map(&mx, op.a, m.M, op.K, op.lda, MN))
    return cudaErrorInvalidValue;
  FewArgs a{m.sa, m.sb, m.sam, m.sak, m.sbn, m.sbk, m.bias, m.out, m.ldo, m.M, m.N, m.kb};
  auto k = matmul_blocks_few_kernel<MN, ODT>;
  const int smem = static_cast<int>(sizeof(FewSmem<MN>)) + 1024;
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  // CTAs per row tile: as many as start at once (three or two fit on an SM, but
  // whole clusters do not fill every SM: N = 7168, K = 5376, 16 rows, 6 ranks
  // 13.0 us, 7 ranks 17.7; 32 rows, 4 ranks 14.4, 6 ranks 19.2), at least two
  // k-blocks each.
  const int tiles = (m.N + 127) / 128;
  const int want = (MN == 16 ? 23 : 16) * sm_count() / 10 / tiles;
  const int ranks = max(1, min(min(8, want), m.kb / 2));
  return launch_cluster(k, static_cast<unsigned>(tiles) * ranks, 256, smem, ranks, st, mw, mx, a);
}

template <int ODT>
cudaError_t dispatch(const Operands& op, const MatmulArgs& a, const Plan& plan, cudaStream_t st) {
  switch (plan.kind) {
    case Plan::kFew16: return launch_few<16, ODT>(op, a, st);
    case Plan::kFew32: return launch_few<32, ODT>(op, a, st);
    case Plan::kWide:
      return plan.parts > 1 ? launch<256, ODT, kParts>(op, a, plan, st) : launch<256, ODT, kWhole>(op, a, plan, st);
    case Plan::kNarrow: return launch<128, ODT, kWhole>(op, a, plan, st);
    default: return launch<128, ODT, kCluster>(op, a, plan, st);
  }
}

int arg_error(const char* msg) {
  return record_error(VCATTN_ERR_ARG, (std::string("vcattn_matmul_blocks: ") + msg).c_str());
}

}  // namespace

cudaError_t matmul_blocks_status(int* code, int* where, int* block, bool reset) {
  tc::DevStatus s{};
  cudaError_t e = cudaMemcpyFromSymbol(&s, g_matmul_status, sizeof(s));
  if (e != cudaSuccess) return e;
  *code = s.code;
  *where = s.where;
  *block = s.block;
  if (reset) {
    tc::DevStatus z{};
    e = cudaMemcpyToSymbol(g_matmul_status, &z, sizeof(z));
  }
  return e;
}

}  // namespace vcattn

extern "C" VCATTN_API size_t vcattn_matmul_blocks_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > (int64_t{1} << 30) || N > (int64_t{1} << 30) || K > (int64_t{1} << 30)) return 0;
  return vcattn::plan_product(M, N, (K + vcattn::kBK - 1) / vcattn::kBK).workspace;
}

extern "C" VCATTN_API int vcattn_matmul_blocks(const uint8_t* a8, int64_t lda, const float* a_scale, int64_t as_m,
                                               int64_t as_k, const uint8_t* b8, int64_t ldb, const float* b_scale,
                                               int64_t bs_n, int64_t bs_k, int64_t M, int64_t N, int64_t K,
                                               const float* bias, void* out, int out_dtype, int64_t ldo,
                                               void* workspace, size_t workspace_bytes, void* stream) {
  using namespace vcattn;
  clear_error();
  if (fault_injected("vcattn_matmul_blocks"))
    return record_error(VCATTN_ERR_INJECTED, "vcattn_matmul_blocks: injected fault");
  if (out_dtype != VCATTN_DTYPE_BF16 && out_dtype != VCATTN_DTYPE_F16 && out_dtype != VCATTN_DTYPE_F32)
    return arg_error("unsupported output dtype");
  if (M < 0 || N < 0 || K <= 0 || M > (int64_t{1} << 30) || N > (int64_t{1} << 30) || K > (int64_t{1} << 30))
    return arg_error("size out of range");
  if (M == 0 || N == 0) return VCATTN_OK;
  if (!a8 || !a_scale || !b8 || !b_scale || !out) return arg_error("null pointer");
  if ((reinterpret_cast<uintptr_t>(a8) & 15u) || (reinterpret_cast<uintptr_t>(b8) & 15u) || lda % 16 || ldb % 16 ||
      lda < K || ldb < K)
    return arg_error("code rows must be 16-byte aligned, with a pitch of at least K that is a multiple of 16");
  if (ldo < N) return arg_error("output row stride below N");
  if ((M + 127) / 128 * ((N + 127) / 128) >= (int64_t{1} << 31)) return arg_error("more than 2^31 tiles");
  const int es = out_dtype == VCATTN_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(out) % es) return arg_error("misaligned output");
  MatmulArgs a{};
  a.sa = a_scale; a.sam = as_m; a.sak = as_k; a.sb = b_scale; a.sbn = bs_n; a.sbk = bs_k;
  a.bias = bias; a.out = out; a.ldo = ldo; a.M = static_cast<int>(M); a.N = static_cast<int>(N);
  a.kb = static_cast<int>((K + kBK - 1) / kBK);
  a.vec_out = (reinterpret_cast<uintptr_t>(out) & 15u) == 0 && (ldo * es) % 16 == 0;
  const Plan plan = plan_product(M, N, a.kb);
  if (plan.workspace > 0 &&
      (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) || workspace_bytes < plan.workspace))
    return record_error(VCATTN_ERR_WORKSPACE, "vcattn_matmul_blocks: workspace too small");
  a.part = static_cast<float*>(workspace);
  const Operands op{a8, b8, lda, ldb, K};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = out_dtype == VCATTN_DTYPE_BF16  ? dispatch<VCATTN_DTYPE_BF16>(op, a, plan, st)
                        : out_dtype == VCATTN_DTYPE_F16 ? dispatch<VCATTN_DTYPE_F16>(op, a, plan, st)
                                                        : dispatch<VCATTN_DTYPE_F32>(op, a, plan, st);
  if (e != cudaSuccess)
    return record_error(VCATTN_ERR_CUDA, (std::string("vcattn_matmul_blocks: ") + cudaGetErrorString(e)).c_str());
  return VCATTN_OK;
}
