// Packed attention on register MMAs (mma.sync m16n8k16), for short query
// sequences: the rows of a KV head's group share one pass over its keys.
//
//   O = softmax(scale q k^T + mask) v,  one pass with a running maximum m and
//   sum l per row (both fp32):  O <- O 2^(m - m') + P V,  P = 2^(s - m' + kRaise)
//
// A tile is 64 or 16 rows (token, group head) of one sequence and KV head
// against a range of its keys.  cp.async brings K and V to shared memory; keys
// past the sequence's end are filled with zeros on the way in, so nothing of a
// neighbouring sequence (or of unwritten memory) is multiplied.  A tile over
// part of the keys writes its unnormalised rows, m and l; the join kernel adds
// the parts in key order.
#include "attn_packed.cuh"
#include "launch.cuh"

#include <string>

namespace vcattn {
namespace {

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// 16 bytes global -> shared; `bytes` of them read, the rest filled with zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <int DT>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT == VCATTN_DTYPE_BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == VCATTN_DTYPE_BF16) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// Two 16-bit elements: is either infinite or NaN, and the pair with those set to 0.
template <int DT> __device__ __forceinline__ uint32_t expo_mask() { return DT == VCATTN_DTYPE_BF16 ? 0x7f80u : 0x7c00u; }
template <int DT> __device__ __forceinline__ bool bad2(uint32_t w) {
  const uint32_t e = expo_mask<DT>();
  return (w & e) == e || ((w >> 16) & e) == e;
}
template <int DT> __device__ __forceinline__ uint32_t clean2(uint32_t w) {
  const uint32_t e = expo_mask<DT>();
  if ((w & e) == e) w &= 0xffff0000u;
  if (((w >> 16) & e) == e) w &= 0x0000ffffu;
  return w;
}
template <int DT> __device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (DT == VCATTN_DTYPE_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// P is made 2^kRaise times as large, and so are l and O, which cancels in O / l.
// In bf16 that changes nothing; f16 has steps of 2^-24 below 2^-14, which all
// the keys behind one of a much larger score would share (65536 keys, 18 nats
// below the first: 1.4 % of the output), so P uses its range up to 2^15.
template <int DT> constexpr float kRaise = DT == VCATTN_DTYPE_F16 ? 15.f : 0.f;

template <int D> constexpr int kPitch = D * 2 + 16;   // bytes of a row in shared memory: eight rows start in different banks

// Keys [key0, key0 + KEYS) of K or V into shared memory by THREADS threads.
template <int D, int KEYS, int THREADS>
__device__ __forceinline__ void load_keys(uint32_t dst, const PackedArgs& a, const void* base, int64_t sh, int64_t sn,
                                          const PackedTile& t, int head, int key0, int tid) {
  const uint16_t* p = static_cast<const uint16_t*>(base) + head * sh;
#pragma unroll
  for (int c = tid; c < KEYS * (D / 8); c += THREADS) {
    const int r = c / (D / 8), ch = c % (D / 8);
    const bool in = key0 + r < t.lk && t.k0 + key0 + r < a.Tk;
    const int64_t row = in ? t.k0 + key0 + r : 0;
    copy16(dst + r * kPitch<D> + ch * 16, p + row * sn + ch * 8, in ? 16 : 0);
  }
}

// The sixteen rows of one warp: queries, running reference, sum and output.
// Lane (gid, tig) holds rows gid and gid + 8.
template <int DT, int D> struct Rows16 {
  uint32_t qa[D / 16][4];
  float o[D / 8][4];
  float m[2], l[2];
  int tok[2], head[2], lim[2];
  bool live[2];
  int first_lim;   // keys that the first row, which sees the fewest, sees
  int lane, gid, tig;

  __device__ __forceinline__ void start(const PackedArgs& a, const PackedTile& t, int kvh, int row0, int lane_) {
    lane = lane_;
    gid = lane >> 2;
    tig = lane & 3;
    const int n_rows = t.lq * a.G;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = row0 + gid + 8 * i;
      tok[i] = r / a.G;
      head[i] = kvh * a.G + r - tok[i] * a.G;
      live[i] = r < n_rows && t.q0 + tok[i] < a.Tq;
      lim[i] = !live[i] ? 0 : a.causal ? min(t.lk, tok[i] + t.lk - t.lq + 1) : t.lk;   // keys [0, lim) are seen
      const uint16_t* p = static_cast<const uint16_t*>(a.q) +
                          (live[i] ? head[i] * a.qsh + static_cast<int64_t>(t.q0 + tok[i]) * a.qsn : 0);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qa[kk][i] = live[i] ? *reinterpret_cast<const uint32_t*>(p + kk * 16 + tig * 2) : 0u;
        qa[kk][2 + i] = live[i] ? *reinterpret_cast<const uint32_t*>(p + kk * 16 + 8 + tig * 2) : 0u;
      }
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
    first_lim = a.causal ? min(t.lk, row0 / a.G + t.lk - t.lq + 1) : t.lk;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  }

  // One tile of KEYS keys whose K and V rows are at `ks`, `vs` (vp: V, generic address).
  template <int KEYS>
  __device__ __forceinline__ void step(const PackedArgs& a, uint32_t ks, uint32_t vs, const uint8_t* vp, int key0) {
    constexpr int P = kPitch<D>;
    float s[KEYS / 8][4];
#pragma unroll
    for (int n = 0; n < KEYS / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int n = 0; n < KEYS / 8; n += 2) {
        // matrices: keys n*8.. (channels +0, +8), keys (n+1)*8.. (channels +0, +8)
        uint32_t b[4];
        ldsm4(b, ks + (n * 8 + (lane & 7) + ((lane >> 4) << 3)) * P + kk * 32 + ((lane >> 3) & 1) * 16);
        mma16<DT>(s[n], qa[kk], b[0], b[1]);
        mma16<DT>(s[n + 1], qa[kk], b[2], b[3]);
      }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < KEYS / 8; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = key0 + n * 8 + tig * 2 + (e & 1), i = e >> 1;
        s[n][e] = key < lim[i] ? s[n][e] * a.scale_log2 : -INFINITY;
        mx[i] = fmaxf(mx[i], s[n][e]);
      }
    }
    float base[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
    }
    // the rows of O are rescaled only where a maximum has grown
    if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float mn = fmaxf(m[i], mx[i]);
        const float al = exp2f(m[i] - (mn == -INFINITY ? 0.f : mn));
        l[i] *= al;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][2 * i] *= al;
          o[n][2 * i + 1] *= al;
        }
        m[i] = mn;
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) base[i] = m[i] == -INFINITY ? 0.f : m[i] - kRaise<DT>;   // (a row without a key so far: 0)
    uint32_t pa[KEYS / 16][4];
#pragma unroll
    for (int n = 0; n < KEYS / 8; ++n) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = exp2f(s[n][e] - base[e >> 1]);
        l[e >> 1] += p[e];
      }
      pa[n / 2][(n & 1) * 2] = pack2<DT>(p[0], p[1]);
      pa[n / 2][(n & 1) * 2 + 1] = pack2<DT>(p[2], p[3]);
    }
    // Where the causal mask ends inside this tile, a row's masked keys have
    // P = 0, but 0 times an infinite or NaN value is NaN.  If the tile holds
    // such values, they enter the product as 0 and are added to the rows that
    // do see them afterwards; the other rows' bits do not change.
    bool bad = false;
    if (first_lim < key0 + KEYS && a.causal) {
      for (int c = lane; c < KEYS * (D / 8); c += 32) {
        const uint4 w = *reinterpret_cast<const uint4*>(vp + (c / (D / 8)) * P + (c % (D / 8)) * 16);
        bad |= bad2<DT>(w.x) || bad2<DT>(w.y) || bad2<DT>(w.z) || bad2<DT>(w.w);
      }
      bad = __any_sync(0xffffffffu, bad);
    }
#pragma unroll
    for (int kk = 0; kk < KEYS / 16; ++kk) {
#pragma unroll
      for (int n = 0; n < D / 8; n += 2) {
        uint32_t b[4];
        ldsm4t(b, vs + (kk * 16 + (lane & 15)) * P + n * 16 + (lane >> 4) * 16);
        if (bad) {
#pragma unroll
          for (int e = 0; e < 4; ++e) b[e] = clean2<DT>(b[e]);
        }
        mma16<DT>(o[n], pa[kk], b[0], b[1]);
        mma16<DT>(o[n + 1], pa[kk], b[2], b[3]);
      }
    }
    if (bad) {
#pragma unroll
      for (int n8 = 0; n8 < KEYS / 8; ++n8) {
        for (int c = 0; c < 8; ++c) {   // key n8 * 8 + c: its P sits in lane c / 2 of the quad
          const int key = n8 * 8 + c;
          float p[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 f = unpack2<DT>(__shfl_sync(0xffffffffu, pa[n8 / 2][(n8 & 1) * 2 + i], (lane & 28) + (c >> 1)));
            p[i] = (c & 1) ? f.y : f.x;
          }
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(vp + key * P + n * 16 + tig * 4);
            if (bad2<DT>(w)) {
              const float2 f = unpack2<DT>(w);
              const bool x = !isfinite(f.x), y = !isfinite(f.y);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                if (key0 + key < lim[i]) {
                  if (x) o[n][2 * i] = fmaf(p[i], f.x, o[n][2 * i]);
                  if (y) o[n][2 * i + 1] = fmaf(p[i], f.y, o[n][2 * i + 1]);
                }
              }
            }
          }
        }
      }
    }
  }

  __device__ __forceinline__ void finish_sum() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
  }

  // Output rows, or the partial result `prow` (row gid of the warp's sixteen).
  __device__ __forceinline__ void store(const PackedArgs& a, const PackedTile& t, int64_t prow) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!live[i]) continue;
      if (t.slot >= 0) {
        const int64_t r = prow + gid + 8 * i;
        float* po = a.part_o + r * D + tig * 2;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(po + n * 8) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
        if (tig == 0) *reinterpret_cast<float2*>(a.part_ml + r * 2) = make_float2(m[i], l[i]);
      } else {
        const float inv = l[i] != 0.f ? __fdiv_rn(1.f, l[i]) : 0.f;   // no key, no output
        uint16_t* p = static_cast<uint16_t*>(a.out) + head[i] * a.osh + static_cast<int64_t>(t.q0 + tok[i]) * a.osn + tig * 2;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<uint32_t*>(p + n * 8) = pack2<DT>(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
      }
    }
  }
};

// ---- 64 rows: the warps own sixteen rows each and share the tiles ------------
// (8 sequences of 24 queries over 4096 keys, 32 / 8 heads x 128: 98 us.)
constexpr int kKeys = 64;
constexpr int kWarps = 4;
template <int D> constexpr int kTile = kKeys * kPitch<D>;
template <int D> constexpr int kSmem = 4 * kTile<D>;   // K and V, two stages

template <int DT, int D>
__global__ void __launch_bounds__(kWarps * 32) attn_packed_kernel(const PackedArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  grid_release();
  const PackedTile t = load_tile(a, blockIdx.x / a.Hk, a.G);   // longest first, over all heads
  const int kvh = blockIdx.x % a.Hk;
  const int tid = threadIdx.x, warp = tid >> 5;
  const uint32_t s0 = smem_addr(smem);
  Rows16<DT, D> rows;
  rows.start(a, t, kvh, t.r0 + warp * 16, tid & 31);

  const int steps = t.ke > t.kb ? (t.ke - t.kb + kKeys - 1) / kKeys : 0;
  auto load = [&](int j) {
    const uint32_t dst = s0 + (j & 1) * 2 * kTile<D>;
    load_keys<D, kKeys, kWarps * 32>(dst, a, a.k, a.ksh, a.ksn, t, kvh, t.kb + j * kKeys, tid);
    load_keys<D, kKeys, kWarps * 32>(dst + kTile<D>, a, a.v, a.vsh, a.vsn, t, kvh, t.kb + j * kKeys, tid);
  };
  if (steps > 0) load(0);
  copy_commit();
  for (int j = 0; j < steps; ++j) {
    if (j + 1 < steps) load(j + 1);
    copy_commit();
    copy_wait<1>();
    __syncthreads();
    const uint32_t ks = s0 + (j & 1) * 2 * kTile<D>, vs = ks + kTile<D>;
    rows.template step<kKeys>(a, ks, vs, smem + (vs - s0), t.kb + j * kKeys);
    __syncthreads();
  }
  rows.finish_sum();
  rows.store(a, t, (static_cast<int64_t>(t.slot) * a.Hk + kvh) * kPackedRows + warp * 16);
  grid_wait();
}

// ---- 16 rows: the warps take every fourth tile of sixteen keys ---------------
// A single new token gives a KV head's group only a few rows: the work is to
// stream K and V once.  Each warp fills and reads its own ring (no barrier
// until the end), and the four partial results are added in warp order through
// shared memory.  Two rings: three stages with two CTAs per SM keep 128 KB in
// flight (64 sequences of 2048 keys, 8 KV heads of 128: 91 us, 5.9 TB/s; two
// stages with three CTAs: 118 us); two stages let three CTAs start at once,
// which is better when no CTA has to wait for that (12 sequences of 1 to 8192
// keys, 344 CTAs: 38 against 50 us).
constexpr int kFewKeys = 16;
template <int D> constexpr int kFewTile = kFewKeys * kPitch<D>;
template <int D, int STAGES> constexpr int kFewSmem = kWarps * STAGES * 2 * kFewTile<D>;

template <int DT, int D, int STAGES>
__global__ void __launch_bounds__(kWarps * 32, STAGES == 2 ? 3 : 2) attn_packed_few_kernel(const PackedArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  grid_release();
  const PackedTile t = load_tile(a, blockIdx.x / a.Hk, a.G);   // longest first, over all heads
  const int kvh = blockIdx.x % a.Hk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * STAGES * 2 * kFewTile<D>;
  const uint32_t r0 = smem_addr(ring);
  const int tiles = t.ke > t.kb ? (t.ke - t.kb + kFewKeys - 1) / kFewKeys : 0;
  const int steps = tiles > warp ? (tiles - warp + kWarps - 1) / kWarps : 0;
  auto load = [&](int j) {
    const uint32_t dst = r0 + (j % STAGES) * 2 * kFewTile<D>;
    const int key0 = t.kb + (j * kWarps + warp) * kFewKeys;
    load_keys<D, kFewKeys, 32>(dst, a, a.k, a.ksh, a.ksn, t, kvh, key0, lane);
    load_keys<D, kFewKeys, 32>(dst + kFewTile<D>, a, a.v, a.vsh, a.vsn, t, kvh, key0, lane);
  };
#pragma unroll
  for (int j = 0; j < STAGES - 1; ++j) {
    if (j < steps) load(j);
    copy_commit();
  }
  Rows16<DT, D> rows;
  rows.start(a, t, kvh, t.r0, lane);
  for (int j = 0; j < steps; ++j) {
    copy_wait<STAGES - 2>();
    __syncwarp();
    if (j + STAGES - 1 < steps) load(j + STAGES - 1);   // (over the tile that every lane has finished with)
    copy_commit();
    const int st = (j % STAGES) * 2 * kFewTile<D>;
    rows.template step<kFewKeys>(a, r0 + st, r0 + st + kFewTile<D>, ring + st + kFewTile<D>,
                                 t.kb + (j * kWarps + warp) * kFewKeys);
  }
  rows.finish_sum();
  copy_wait<0>();
  // add the warps' results: m first, then O and l relative to it
  __shared__ float wm[kWarps][16], wl[kWarps][16];
  if (rows.tig == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      wm[warp][rows.gid + 8 * i] = rows.m[i];
      wl[warp][rows.gid + 8 * i] = rows.l[i];
    }
  }
  __syncthreads();   // (the rings are free from here on)
  float* wo = reinterpret_cast<float*>(smem) + warp * 16 * D;   // [warp][row][channel]
  float mx[2], al[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = rows.gid + 8 * i;
    mx[i] = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
    al[i] = exp2f(rows.m[i] - (mx[i] == -INFINITY ? 0.f : mx[i]));
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      *reinterpret_cast<float2*>(wo + r * D + n * 8 + rows.tig * 2) = make_float2(rows.o[n][2 * i] * al[i], rows.o[n][2 * i + 1] * al[i]);
  }
  __syncthreads();
  // each warp adds a quarter of the channels of all sixteen rows
  constexpr int C = D / 32;   // channels per lane: lane = row * 2 + half
  const int row = lane >> 1, c0 = warp * (D / 4) + (lane & 1) * (D / 8);
  const int r = t.r0 + row, tok = r / a.G;
  if (r >= t.lq * a.G || t.q0 + tok >= a.Tq) {
    grid_wait();
    return;
  }
  float m = -INFINITY, l = 0.f, acc[D / 8];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, wm[w][row]);
#pragma unroll
  for (int c = 0; c < D / 8; ++c) acc[c] = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    l += wl[w][row] * exp2f(wm[w][row] - (m == -INFINITY ? 0.f : m));
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) + (w * 16 + row) * D + c0);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const float4 f = p[c];
      acc[4 * c] += f.x; acc[4 * c + 1] += f.y; acc[4 * c + 2] += f.z; acc[4 * c + 3] += f.w;
    }
  }
  if (t.slot >= 0) {
    const int64_t pr = (static_cast<int64_t>(t.slot) * a.Hk + kvh) * kPackedFewRows + row;
#pragma unroll
    for (int c = 0; c < C; ++c)
      *reinterpret_cast<float4*>(a.part_o + pr * D + c0 + 4 * c) = make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
    if (c0 == 0) *reinterpret_cast<float2*>(a.part_ml + pr * 2) = make_float2(m, l);
  } else {
    const float inv = l != 0.f ? __fdiv_rn(1.f, l) : 0.f;
    uint16_t* p = static_cast<uint16_t*>(a.out) + (kvh * a.G + r - tok * a.G) * a.osh + static_cast<int64_t>(t.q0 + tok) * a.osn + c0;
#pragma unroll
    for (int c = 0; c < D / 8; c += 2) *reinterpret_cast<uint32_t*>(p + c) = pack2<DT>(acc[c] * inv, acc[c + 1] * inv);
  }
  grid_wait();
}

// out = sum_p 2^(m_p - m) O_p / sum_p 2^(m_p - m) l_p, one warp per row.  The
// parts of a tile of R rows belong to `heads` heads; row = token * G + g is
// query head head * G + g.
template <int DT, int D, int R>
__global__ void __launch_bounds__(256) attn_packed_join_kernel(const PackedArgs a, int heads, int G) {
  grid_wait();   // the parts
  const PackedJoin jn = load_join(a, blockIdx.x / (R / 8), G);
  const int row = (blockIdx.x % (R / 8)) * 8 + (threadIdx.x >> 5), head = blockIdx.y, lane = threadIdx.x & 31;
  const int r = jn.r0 + row, tok = r / G;
  if (tok >= jn.lq || jn.q0 + tok >= a.Tq) return;
  const int64_t step = static_cast<int64_t>(heads) * R;
  const int64_t first = (static_cast<int64_t>(jn.slot0) * heads + head) * R + row;
  constexpr int C = D / 32, P = 8;   // channels of a lane, parts in flight
  float acc[C], den = 0.f, mx = -INFINITY;
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.f;
  for (int p = lane; p < jn.pieces; p += 32) mx = fmaxf(mx, a.part_ml[(first + p * step) * 2]);
  mx = warp_max(mx);
  const float base = mx == -INFINITY ? 0.f : mx;
  for (int p0 = 0; p0 < jn.pieces; p0 += 32) {
    // lane p holds the weight and the sum of part p0 + p
    float w = 0.f, l = 0.f;
    if (p0 + lane < jn.pieces) {
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (first + (p0 + lane) * step) * 2);
      w = exp2f(ml.x - base);
      l = ml.y;
    }
    const int n = min(32, jn.pieces - p0);
    for (int q = 0; q < n; q += P) {
      float x[P][C];
#pragma unroll
      for (int u = 0; u < P; ++u) {
        const float* src = a.part_o + (first + (p0 + min(q + u, n - 1)) * step) * D + lane * C;
        if constexpr (C == 4) {
          const float4 f = *reinterpret_cast<const float4*>(src);
          x[u][0] = f.x; x[u][1] = f.y; x[u][2] = f.z; x[u][3] = f.w;
        } else {
          const float2 f = *reinterpret_cast<const float2*>(src);
          x[u][0] = f.x; x[u][1] = f.y;
        }
      }
#pragma unroll
      for (int u = 0; u < P; ++u) {   // (in the order of the parts)
        const float wu = __shfl_sync(0xffffffffu, w, (q + u) & 31), lu = __shfl_sync(0xffffffffu, l, (q + u) & 31);
        if (q + u < n) {
          den = fmaf(wu, lu, den);
#pragma unroll
          for (int c = 0; c < C; ++c) acc[c] = fmaf(wu, x[u][c], acc[c]);
        }
      }
    }
  }
  const float inv = den != 0.f ? __fdiv_rn(1.f, den) : 0.f;
  uint16_t* o = static_cast<uint16_t*>(a.out) + (head * G + r - tok * G) * a.osh + static_cast<int64_t>(jn.q0 + tok) * a.osn;
#pragma unroll
  for (int c = 0; c < C; c += 2) *reinterpret_cast<uint32_t*>(o + lane * C + c) = pack2<DT>(acc[c] * inv, acc[c + 1] * inv);
}

template <int DT, int D, int R>
cudaError_t join(const PackedArgs& a, int heads, int G, cudaStream_t st) {
  if (a.n_joins == 0) return cudaSuccess;
  return launch_after(attn_packed_join_kernel<DT, D, R>, dim3(a.n_joins * (R / 8), heads), 256, 0, st, true, a, heads, G);
}

template <int DT, int D, int STAGES>
cudaError_t launch_few(const PackedArgs& a, unsigned ctas, bool after, cudaStream_t st) {
  auto k = attn_packed_few_kernel<DT, D, STAGES>;
  constexpr int smem = kFewSmem<D, STAGES>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  return e == cudaSuccess ? launch_after(k, dim3(ctas), kWarps * 32, smem, st, after, a) : e;
}

// The three lists of a batch (kPackedFewRows, kPackedRows, kPackedWideRows
// rows per tile).  The lists do not depend on each other, so the CTAs of the
// next one start on the SMs that the one before no longer fills.
template <int DT, int D>
cudaError_t launch(const PackedArgs (&list)[3], cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  const PackedArgs &few = list[0], &mid = list[1], &wide = list[2];
  bool after = false;
  if (wide.n_tiles > 0) {
    e = launch_attn_packed_tc(wide, DT, st);
    after = true;
  }
  if (e == cudaSuccess && mid.n_tiles > 0) {
    auto k = attn_packed_kernel<DT, D>;
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem<D>);
    if (e == cudaSuccess) e = launch_after(k, dim3(static_cast<unsigned>(mid.n_tiles) * mid.Hk), kWarps * 32, kSmem<D>, st, after, mid);
    after = true;
  }
  if (e == cudaSuccess && few.n_tiles > 0) {
    const unsigned ctas = static_cast<unsigned>(few.n_tiles) * few.Hk;
    e = ctas <= 3u * sm_count() ? launch_few<DT, D, 2>(few, ctas, after, st) : launch_few<DT, D, 3>(few, ctas, after, st);
  }
  if (e == cudaSuccess) e = join<DT, D, kPackedWideRows>(wide, wide.Hq, 1, st);
  if (e == cudaSuccess) e = join<DT, D, kPackedRows>(mid, mid.Hk, mid.G, st);
  if (e == cudaSuccess) e = join<DT, D, kPackedFewRows>(few, few.Hk, few.G, st);
  return e;
}

int arg_error(const char* msg) {
  return record_error(VCATTN_ERR_ARG, (std::string("vcattn_attn_packed: ") + msg).c_str());
}

bool rows_fit(const vcattn_bhnd* v) {
  return v != nullptr && v->data != nullptr && (reinterpret_cast<uintptr_t>(v->data) & 15u) == 0 && v->sh % 8 == 0 &&
         v->sn % 8 == 0;
}

}  // namespace
}  // namespace vcattn

extern "C" {

VCATTN_API size_t vcattn_attn_packed_workspace_bytes(const vcattn_packed_work* work, int Hq, int Hk, int D) {
  if (work == nullptr || Hq <= 0 || Hk <= 0 || D <= 0) return 0;
  size_t rows = 0;
  for (int i = 0; i < 3; ++i) {
    if (work->slots[i] < 0) return 0;
    rows += static_cast<size_t>(work->slots[i]) * vcattn::kListRows[i] * (i == 2 ? Hq : Hk);
  }
  return rows * (D + 2) * sizeof(float);
}

VCATTN_API int vcattn_attn_packed(const vcattn_bhnd* q, const vcattn_bhnd* k, const vcattn_bhnd* v, int dtype, int Hq,
                                  int Hk, int Tq, int Tk, int D, const vcattn_packed_work* work, int causal,
                                  float scale, const vcattn_bhnd* out, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  using namespace vcattn;
  static_assert(sizeof(PackedTile) == sizeof(vcattn_packed_tile) && sizeof(PackedJoin) == sizeof(vcattn_packed_join),
                "the C ABI's records are the kernels'");
  clear_error();
  if (fault_injected("vcattn_attn_packed"))
    return record_error(VCATTN_ERR_INJECTED, "vcattn_attn_packed: injected fault");
  if (dtype != VCATTN_DTYPE_BF16 && dtype != VCATTN_DTYPE_F16) return arg_error("dtype must be bf16 or f16");
  if (D != 64 && D != 128) return arg_error("D must be 64 or 128");
  if (Hq <= 0 || Hk <= 0 || Hq % Hk || Hq > 65535) return arg_error("Hq must be a positive multiple of Hk, at most 65535");
  if (!work) return arg_error("null pointer");
  bool sized = Tq >= 0 && Tk >= 0, given = true, few = true;
  int64_t tiles = 0;
  for (int i = 0; i < 3; ++i) {
    sized &= work->n_tiles[i] >= 0 && work->n_joins[i] >= 0 && work->slots[i] >= 0;
    given &= (work->n_tiles[i] <= 0 || work->tiles[i]) && (work->n_joins[i] <= 0 || work->joins[i]);
    few &= static_cast<int64_t>(work->n_tiles[i]) * Hq < (int64_t{1} << 31) &&
           static_cast<int64_t>(work->n_joins[i]) * (kListRows[i] / 8) < (int64_t{1} << 31);
    tiles += work->n_tiles[i];
  }
  if (!sized) return arg_error("negative size");
  if (!(scale > 0.f) || scale > 1e30f) return arg_error("scale must be positive and finite");
  if (Tq == 0 || tiles == 0) return VCATTN_OK;
  if (!given) return arg_error("null pointer");
  if (!few) return arg_error("more than 2^31 tiles");
  if (!rows_fit(q) || !rows_fit(out) || (Tk > 0 && (!rows_fit(k) || !rows_fit(v))))
    return arg_error("q, k, v and out must be 16-byte aligned with strides of 16-byte multiples");
  const size_t need = vcattn_attn_packed_workspace_bytes(work, Hq, Hk, D);
  if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) || workspace_bytes < need))
    return record_error(VCATTN_ERR_WORKSPACE, "vcattn_attn_packed: workspace too small");
  PackedArgs a{};
  a.q = q->data; a.out = const_cast<void*>(out->data);
  a.qsh = q->sh; a.qsn = q->sn; a.osh = out->sh; a.osn = out->sn;
  if (Tk > 0) {
    a.k = k->data; a.v = v->data;
    a.ksh = k->sh; a.ksn = k->sn; a.vsh = v->sh; a.vsn = v->sn;
  } else {   // no key anywhere: nothing is read through these
    a.k = a.v = a.q;
    a.ksh = a.vsh = a.qsh;
    a.ksn = a.vsn = a.qsn;
  }
  a.Hq = Hq; a.Hk = Hk; a.G = Hq / Hk; a.D = D; a.Tq = Tq; a.Tk = Tk;
  a.causal = causal ? 1 : 0;
  a.scale_log2 = scale * kLog2e;
  PackedArgs list[3] = {a, a, a};
  float* ws = static_cast<float*>(workspace);
  for (int i = 0; i < 3; ++i) {
    PackedArgs& x = list[i];
    x.tiles = reinterpret_cast<const PackedTile*>(work->tiles[i]);
    x.joins = reinterpret_cast<const PackedJoin*>(work->joins[i]);
    x.n_tiles = work->n_tiles[i];
    x.n_joins = work->n_joins[i];
    x.slots = work->slots[i];
    const size_t rows = static_cast<size_t>(work->slots[i]) * kListRows[i] * (i == 2 ? Hq : Hk);
    x.part_o = ws;
    x.part_ml = ws + rows * D;
    ws += rows * (D + 2);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      dtype == VCATTN_DTYPE_BF16
          ? (D == 128 ? launch<VCATTN_DTYPE_BF16, 128>(list, st) : launch<VCATTN_DTYPE_BF16, 64>(list, st))
          : (D == 128 ? launch<VCATTN_DTYPE_F16, 128>(list, st) : launch<VCATTN_DTYPE_F16, 64>(list, st));
  if (e != cudaSuccess)
    return record_error(VCATTN_ERR_CUDA, (std::string("vcattn_attn_packed: ") + cudaGetErrorString(e)).c_str());
  return VCATTN_OK;
}

}  // extern "C"
