// 8-bit integer matrix product with one scale for each token (row of the
// activation) and one for each channel (row of the weight):
//   out[m, n] = T(fl(fl(float(sum_k a[m, k] w[n, k]) * xs[m]) * ws[n]) + bias[n]),
// with an exact int32 dot (K <= 131072: |dot| <= 127 * 127 K < 2^31).
// Layout NK reads w as (n, k) rows, the forward product; layout KN reads it
// as (k, n) rows: the same weight matrix contracted over its rows, the
// product of the input's gradient.  Integer sums are exact, so neither the
// tiling nor the split of K changes a bit.
//
// Two kernels on tcgen05 kind::i8, operands by TMA in 128-byte-swizzled
// tiles, accumulators in TMEM:
// * pair_kernel: CTA pairs (cta_group::2), 256 tokens x 256 channels a tile,
//   persistent, for products that fill the GPU with such tiles.  Bound by the
//   tensor cores.
// * swap_kernel: 128 channels on the MMA's M side and 16 to 128 tokens on its
//   N side, K split over a cluster, for few tokens or few tiles.  Bound by
//   reading the weights once.
#include <cudaTypedefs.h>

#include "rows.cuh"

namespace convrot {

namespace w4a4 {
int make_tmap_u8(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                 const uint32_t* box, CUtensorMapSwizzle swizzle, CUtensorMapDataType dtype);
}

namespace i8 {

constexpr int kMaxK = 131072;
constexpr int kBK = 128;  // K bytes of a stage: one 128-byte swizzle row
constexpr uint64_t kTimeoutNs = 4000000000ull;  // a single wait never legitimately takes this long

struct Params {
  const float* xscales;
  const float* wscales;  // may be null: ones
  const float* bias;     // may be null: zeros
  void* out;
  int m, n, k;
  int* err_word;
  // swap_kernel: the weight copies may be issued before the previous kernel
  // of the stream has completed (it only writes the activation)
  int early_weights;
};

// tcgen05 instruction descriptor: D s32, A and B s8, B N-major for bmn, A
// M-major for amn.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n, bool amn, bool bmn) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(amn) << 15) | (static_cast<uint32_t>(bmn) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// Wait for the phase of `bar` with parity `parity`, for at most kTimeoutNs;
// on time-out record `code` in *err and return false.  Cluster-scope acquire:
// barriers of a pair receive arrivals from both CTAs.
__device__ __noinline__ bool wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    if ((i & 255) == 0) {
      if (*reinterpret_cast<volatile int*>(err)) return false;
      if (globaltimer() - t0 > kTimeoutNs) {
        atomicCAS(err, 0, code);
        return false;
      }
    }
  }
}

// After an error: give copies that may still be in flight 2 ms to land.
__device__ __forceinline__ void settle() {
  const uint64_t t0 = globaltimer();
  while (globaltimer() - t0 < 2000000ull) {
  }
}

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

__device__ __forceinline__ void tma_load_2d_pair(void* smem_dst, const CUtensorMap* map, uint32_t bar_cluster_addr,
                                                 int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster_addr), "r"(x), "r"(y)
      : "memory");
}

// ===========================================================================
// Pair kernel.  Each CTA of a pair holds 128 tokens and 128 channels of the
// 256 x 256 tile:
//   warp 0   activation producer, warp 2 weight producer: lane s issues the
//            16 KB box of ring slot s (copies of one thread are served one
//            after another), completing on the leader's full[s]
//   warp 1   leader: MMA issuer (M = 256, N = 256); both: TMEM owner
//   warp 3   idle
//   warps 4-11  epilogue of this CTA's 128 rows: warp w reads TMEM lanes
//            32 (w % 4) .. + 31, columns 128 ((w - 4) / 4) .. + 127
// Two accumulators of 256 columns let the epilogue overlap the next tile.
// ===========================================================================
namespace pair {

constexpr int kTile = 256;
constexpr int kStages = 6;
constexpr int kOpBytes = 128 * kBK;  // one operand's half tile of a stage
constexpr int kWarpA = 0, kWarpMma = 1, kWarpB = 2, kWarpE0 = 4, kEWarps = 8;
constexpr int kThreads = (kWarpE0 + kEWarps) * 32;
constexpr uint32_t kTmemCols = 2 * kTile;
constexpr int kChunkBytes = 32 * 64;              // restaging: 32 rows x 64 bytes for each epilogue warp
constexpr int kVecBytes = kEWarps * 2 * 128 * 4;  // scales and bias of a warp's 128 columns

struct alignas(8) Bars {
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t mma_done;
  uint32_t tmem_base;
  int err;
};

constexpr size_t kSmem = 1024 + kStages * 2 * kOpBytes + kEWarps * kChunkBytes + kVecBytes + sizeof(Bars);
static_assert(kSmem <= 232448, "shared memory budget");

template <int LAYOUT, typename TOut>
__global__ void __launch_bounds__(kThreads, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + kStages * kOpBytes;
  uint8_t* stage_out = sB + kStages * kOpBytes;
  float* vecs = reinterpret_cast<float*>(stage_out + kEWarps * kChunkBytes);
  Bars* bars = reinterpret_cast<Bars*>(reinterpret_cast<uint8_t*>(vecs) + kVecBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();  // 0 = leader
  const int pair_id = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;
  const int m_tiles = (p.m + kTile - 1) / kTile, n_tiles = (p.n + kTile - 1) / kTile;
  const int num_tiles = m_tiles * n_tiles;
  const int k_stages = (p.k + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], 2 * kEWarps);
    }
    mbar_init(&bars->mma_done, 1);
    bars->err = 0;
    fence_mbar_init();
    prefetch_tensormap(&tmap_a);
    prefetch_tensormap(&tmap_b);
  }
  if (warp == kWarpMma) {
    tmem_alloc_pair(&bars->tmem_base, kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // barriers of both CTAs exist before any signal crosses
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  grid_dependency_wait();
  grid_dependents_launch();

  if (warp == kWarpA || warp == kWarpB) {
    if (lane < kStages) {
      const uint32_t lead_full = mapa_shared(&bars->full[lane], 0);
      int g = 0;
      bool ok = true;
      for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs) {
        const int row = (tile % m_tiles) * kTile + 128 * rank;
        const int col = (tile / m_tiles) * kTile + 128 * rank;
        for (int ks = 0; ks < k_stages; ++ks, ++g) {
          if (g % kStages != lane) continue;
          if (!wait(&bars->empty[lane], ((g / kStages) & 1) ^ 1, &bars->err, 61)) { ok = false; break; }
          if (warp == kWarpA) {
            if (rank == 0) mbar_arrive_expect_tx(&bars->full[lane], 4 * kOpBytes);
            tma_load_2d_pair(sA + lane * kOpBytes, &tmap_a, lead_full, ks * kBK, row);
          } else if (LAYOUT == CONVROT_LAYOUT_NK) {
            tma_load_2d_pair(sB + lane * kOpBytes, &tmap_b, lead_full, ks * kBK, col);
          } else {
            tma_load_2d_pair(sB + lane * kOpBytes, &tmap_b, lead_full, col, ks * kBK);
          }
        }
      }
      if (!ok) settle();
    }
  } else if (warp == kWarpMma) {
    if (rank == 0 && lane == 0) {
      constexpr uint32_t idesc = idesc_i8(kTile, kTile, false, LAYOUT == CONVROT_LAYOUT_KN);
      const uint32_t a_base = smem_u32(sA), b_base = smem_u32(sB);
      int g = 0, local = 0;
      bool ok = true;
      for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs, ++local) {
        const int buf = local & 1;
        if (!wait(&bars->acc_empty[buf], ((local >> 1) & 1) ^ 1, &bars->err, 62)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * kTile;
        for (int ks = 0; ks < k_stages; ++ks, ++g) {
          const int slot = g % kStages;
          if (!wait(&bars->full[slot], (g / kStages) & 1, &bars->err, 63)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = a_base + slot * kOpBytes, b_addr = b_base + slot * kOpBytes;
#pragma unroll
          for (int j = 0; j < kBK / 32; ++j) {  // K beyond the end is zero in both operands
            const uint64_t adesc = smem_desc(a_addr + j * 32, 16, 1024, 2);
            const uint64_t bdesc = LAYOUT == CONVROT_LAYOUT_NK ? smem_desc(b_addr + j * 32, 16, 1024, 2)
                                                               : smem_desc(b_addr + j * 4096, kOpBytes, 1024, 2);
            mma_i8_pair(d_tmem, adesc, bdesc, idesc, (ks | j) != 0 ? 1u : 0u);
          }
          mma_commit_pair_multicast(&bars->empty[slot], 0x3);
        }
        if (!ok) break;
        mma_commit_pair_multicast(&bars->acc_full[buf], 0x3);
      }
      // every MMA issued above finishes before the pair's TMEM is released
      mma_commit_pair_multicast(&bars->mma_done, 0x1);
      wait(&bars->mma_done, 0, &bars->err, 64);
    }
  } else if (warp >= kWarpE0) {
    const int ew = warp - kWarpE0, quarter = warp & 3, half = ew >> 2;
    float* sws = vecs + ew * 256;
    float* sbias = sws + 128;
    const uint32_t sb = smem_u32(stage_out) + ew * kChunkBytes;
    const uint32_t lead_empty0 = mapa_shared(&bars->acc_empty[0], 0);
    constexpr int kCols = 64 / sizeof(TOut);  // columns of a restaged chunk
    const bool vec_store = (static_cast<int64_t>(p.n) * sizeof(TOut)) % 16 == 0;
    int local = 0;
    for (int tile = pair_id; tile < num_tiles; tile += num_pairs, ++local) {
      const int buf = local & 1;
      const int row0 = (tile % m_tiles) * kTile + 128 * rank + quarter * 32;
      const int col0 = (tile / m_tiles) * kTile + 128 * half;
      const float xs = row0 + lane < p.m ? __ldg(p.xscales + row0 + lane) : 0.0f;
      __syncwarp();  // the previous tile's reads of the vectors are done
      for (int j = lane; j < 128; j += 32) {
        const bool in = col0 + j < p.n;
        sws[j] = in ? (p.wscales ? __ldg(p.wscales + col0 + j) : 1.0f) : 0.0f;
        sbias[j] = in && p.bias ? __ldg(p.bias + col0 + j) : 0.0f;
      }
      __syncwarp();
      if (!wait(&bars->acc_full[buf], (local >> 1) & 1, &bars->err, 65)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((static_cast<uint32_t>(quarter) * 32u) << 16) + buf * kTile + 128 * half;
      for (int c = 0; c < 4; ++c) {
        if (col0 + 32 * c >= p.n) break;  // uniform across the warp
        uint32_t r[32];
        __syncwarp();
        tmem_ld_32x32b_x32(t_row + c * 32, r);
        tmem_ld_wait();
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 w4 = *reinterpret_cast<const float4*>(sws + c * 32 + j);
          const float4 b4 = *reinterpret_cast<const float4*>(sbias + c * 32 + j);
          const float wv[4] = {w4.x, w4.y, w4.z, w4.w}, bv[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
          for (int u = 0; u < 4; ++u)
            v[j + u] = __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(static_cast<int32_t>(r[j + u])), xs), wv[u]), bv[u]);
        }
        // Restage so that a store instruction covers 8 rows of 64 contiguous
        // bytes instead of 32 rows of 16: 16-byte piece q of row r at
        // ((q + r / 2) % 4), conflict-free both ways.
#pragma unroll
        for (int part = 0; part < 32 / kCols; ++part) {
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t at = sb + lane * 64 + (((q + (lane >> 1)) & 3) << 4);
            const int o = part * kCols + q * (kCols / 4);
            float piece[kCols / 4];
#pragma unroll
            for (int e = 0; e < kCols / 4; ++e) piece[e] = v[o + e];
            Pack<TOut, kCols / 4> pk;
            pk.set(piece);
            sts128(at, pk.w[0], pk.w[1], pk.w[2], pk.w[3]);
          }
          __syncwarp();
          const int col = col0 + c * 32 + part * kCols;
          TOut* out = static_cast<TOut*>(p.out);
          if (vec_store) {
            const int q = lane & 3;
            if (col + (q + 1) * (kCols / 4) <= p.n) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int rr = i * 8 + (lane >> 2);
                if (row0 + rr < p.m)
                  *reinterpret_cast<uint4*>(out + static_cast<int64_t>(row0 + rr) * p.n + col + q * (kCols / 4)) =
                      lds128(sb + rr * 64 + (((q + (rr >> 1)) & 3) << 4));
              }
            }
          } else {
            // rows off the 16-byte grid: one element a lane, consecutive lanes on consecutive columns
            constexpr int kRowsAt = 32 / kCols;
            const int cc = lane % kCols;
            if (col + cc < p.n) {
              for (int rr = lane / kCols; rr < 32; rr += kRowsAt) {
                if (row0 + rr >= p.m) break;
                const int q = cc / (kCols / 4), e = cc % (kCols / 4);
                const uint8_t* src = stage_out + ew * kChunkBytes + rr * 64 + (((q + (rr >> 1)) & 3) << 4);
                out[static_cast<int64_t>(row0 + rr) * p.n + col + cc] = reinterpret_cast<const TOut*>(src)[e];
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(lead_empty0 + buf * 8);
    }
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync();  // no CTA leaves while its partner may still touch its shared memory or TMEM
  tc_fence_after();
  if (warp == kWarpMma) {
    __syncwarp();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
  if (threadIdx.x == 0 && bars->err) atomicCAS(p.err_word, 0, bars->err);
}

}  // namespace pair

// ===========================================================================
// Swap kernel.  One tile of 128 channels x BT tokens and one share of K for
// each CTA; a cluster of CTAs covers K.  Weights stream through a ring of
// 16 KB slots, all of them in flight before the first MMA.
//   warp 0  weight producer (lane s issues slot s), warp 1 MMA issuer and
//   TMEM owner, warp 2 activation producer; then all four warps run the
//   epilogue: lane l of warp w holds channel 32 w + l, so a store instruction
//   writes 32 consecutive channels of one token.
// With K split, each CTA leaves its int32 sums in shared memory and adds up
// its share of the tokens from all of the cluster's.
// ===========================================================================
namespace swap {

constexpr int kThreads = 128;
constexpr int kWBytes = 128 * kBK;
constexpr int kMaxCluster = 8;
constexpr int kMaxStages = 8;

struct alignas(8) Bars {
  uint64_t w_full[kMaxStages];
  uint64_t x_full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t mma_done;
  uint32_t tmem_base;
  int err;
};

template <int BT> constexpr int kStages = BT <= 32 ? 8 : (BT == 64 ? 8 : 6);
template <int BT> constexpr int kXBytes = BT * kBK;
template <int BT> constexpr size_t kSmem = 1024 + kStages<BT> * (kWBytes + kXBytes<BT>) + sizeof(Bars);
static_assert(kSmem<128> <= 232448 && kSmem<64> <= 232448, "shared memory budget");

__device__ __forceinline__ uint32_t dsmem_ld(uint32_t cluster_addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
  return v;
}

template <int LAYOUT, typename TOut, int BT>
__global__ void __launch_bounds__(kThreads)
    swap_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const Params p) {
  constexpr int S = kStages<BT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sX = sW + S * kWBytes;
  Bars* bars = reinterpret_cast<Bars*>(sX + S * kXBytes<BT>);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int ranks = gridDim.x, rank = blockIdx.x;  // the cluster spans the grid's x
  const int n0 = blockIdx.y * 128, m0 = blockIdx.z * BT;
  const int k_stages = (p.k + kBK - 1) / kBK;
  const int k_lo = static_cast<int>(static_cast<int64_t>(k_stages) * rank / ranks);
  const int k_hi = static_cast<int>(static_cast<int64_t>(k_stages) * (rank + 1) / ranks);
  constexpr uint32_t kTmemCols = BT < 32 ? 32 : BT;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&bars->w_full[s], 1);
      mbar_init(&bars->x_full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    mbar_init(&bars->mma_done, 1);
    bars->err = 0;
    fence_mbar_init();
    prefetch_tensormap(&tmap_x);
    prefetch_tensormap(&tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;
  if (!(warp == 0 && p.early_weights)) grid_dependency_wait();

  if (warp == 0 || warp == 2) {
    if (lane < S) {
      bool ok = true;
      for (int kb = k_lo + lane; kb < k_hi; kb += S) {
        const int g = kb - k_lo;
        if (!wait(&bars->empty[lane], ((g / S) & 1) ^ 1, &bars->err, 71)) { ok = false; break; }
        if (warp == 2) {
          mbar_arrive_expect_tx(&bars->x_full[lane], kXBytes<BT>);
          tma_load_2d(sX + lane * kXBytes<BT>, &tmap_x, &bars->x_full[lane], kb * kBK, m0);
        } else {
          mbar_arrive_expect_tx(&bars->w_full[lane], kWBytes);
          if (LAYOUT == CONVROT_LAYOUT_NK)
            tma_load_2d(sW + lane * kWBytes, &tmap_w, &bars->w_full[lane], kb * kBK, n0);
          else
            tma_load_2d(sW + lane * kWBytes, &tmap_w, &bars->w_full[lane], n0, kb * kBK);
        }
      }
      if (!ok) settle();
    }
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t idesc = idesc_i8(128, BT, LAYOUT == CONVROT_LAYOUT_KN, false);
    const uint32_t w_base = smem_u32(sW), x_base = smem_u32(sX);
    for (int kb = k_lo; kb < k_hi; ++kb) {
      const int g = kb - k_lo, slot = g % S;
      if (!wait(&bars->w_full[slot], (g / S) & 1, &bars->err, 72)) break;
      if (!wait(&bars->x_full[slot], (g / S) & 1, &bars->err, 73)) break;
      tc_fence_after();
#pragma unroll
      for (int j = 0; j < kBK / 32; ++j) {
        const uint32_t w_addr = w_base + slot * kWBytes;
        const uint64_t wdesc = LAYOUT == CONVROT_LAYOUT_NK ? smem_desc(w_addr + j * 32, 16, 1024, 2)
                                                           : smem_desc(w_addr + j * 4096, kWBytes, 1024, 2);
        const uint64_t xdesc = smem_desc(x_base + slot * kXBytes<BT> + j * 32, 16, 1024, 2);
        mma_i8(tmem_base, wdesc, xdesc, idesc, (g | j) != 0 ? 1u : 0u);
      }
      mma_commit(&bars->empty[slot]);
    }
    mma_commit(&bars->mma_done);
  }
  __syncwarp();
  grid_dependency_wait();  // warp 0 may not have waited yet; the epilogue reads the token scales
  grid_dependents_launch();
  const bool done = wait(&bars->mma_done, 0, &bars->err, 74);
  tc_fence_after();

  const int n = n0 + warp * 32 + lane;
  const bool n_ok = n < p.n;
  const float ws = n_ok && p.wscales ? __ldg(p.wscales + n) : 1.0f;
  const float b = n_ok && p.bias ? __ldg(p.bias + n) : 0.0f;
  TOut* out = static_cast<TOut*>(p.out);
  const uint32_t t_row = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
  auto emit = [&](int m, int32_t dot) {
    const float v = __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(dot), __ldg(p.xscales + m)), ws), b);
    if (n_ok) out[static_cast<int64_t>(m) * p.n + n] = cvt_out<TOut>(v);
  };
  if (ranks == 1) {
    for (int c = 0; c < BT && m0 + c < p.m && done; c += 16) {
      uint32_t r[16];
      __syncwarp();
      tmem_ld_32x32b_x16(t_row + c, r);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (m0 + c + i < p.m) emit(m0 + c + i, static_cast<int32_t>(r[i]));
    }
  } else {
    // int32 sums (token, channel) over the ring, whose copies have all been consumed
    uint32_t* part = reinterpret_cast<uint32_t*>(smem);
    for (int c = 0; c < BT && m0 + c < p.m && done; c += 16) {
      uint32_t r[16];
      __syncwarp();
      tmem_ld_32x32b_x16(t_row + c, r);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) part[(c + i) * 128 + warp * 32 + lane] = r[i];
    }
    __syncwarp();
    cluster_sync();
    uint32_t peer[kMaxCluster];
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) peer[r] = r < ranks ? mapa_shared(part + warp * 32 + lane, r) : 0u;
    const int rows = p.m - m0 < BT ? p.m - m0 : BT;
    for (int c = rank; c < rows && done; c += ranks) {
      uint32_t v[kMaxCluster];
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) v[r] = r < ranks ? dsmem_ld(peer[r] + c * 512) : 0u;
      uint32_t sum = 0;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) sum += v[r];
      emit(m0 + c, static_cast<int32_t>(sum));
    }
    __syncwarp();
    cluster_sync();  // no CTA leaves while another may still read its sums
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem_base, kTmemCols);
  }
  if (threadIdx.x == 0 && bars->err) atomicCAS(p.err_word, 0, bars->err);
}

}  // namespace swap

// ---------------------------------------------------------------------------
// host side

namespace {

int tmap(CUtensorMap* map, const int8_t* base, int64_t inner, int64_t rows, int64_t stride, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(inner), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(stride)};
  const uint32_t box[2] = {128, static_cast<uint32_t>(box_rows)};
  return w4a4::make_tmap_u8(map, base, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_UINT8);
}

struct Operands {
  const int8_t* act;
  const int8_t* weight;
  int64_t act_stride, weight_stride;
};

int weight_map(CUtensorMap* map, const Operands& o, int layout, const Params& p) {
  return layout == CONVROT_LAYOUT_NK ? tmap(map, o.weight, p.k, p.n, o.weight_stride, 128)
                                     : tmap(map, o.weight, p.n, p.k, o.weight_stride, 128);
}

template <int LAYOUT, typename TOut>
int launch_pair(const Operands& o, const Params& p, cudaStream_t stream) {
  CUtensorMap map_a, map_b;
  int rc = tmap(&map_a, o.act, p.k, p.m, o.act_stride, 128);
  if (rc == CONVROT_OK) rc = weight_map(&map_b, o, LAYOUT, p);
  if (rc != CONVROT_OK) return rc;
  auto kernel = pair::pair_kernel<LAYOUT, TOut>;
  CONVROT_CUDA_CHECK(
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(pair::kSmem)));
  const int64_t tiles = static_cast<int64_t>((p.m + 255) / 256) * ((p.n + 255) / 256);
  const int most = device_sm_count() / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(tiles < most ? tiles : most), 1, 1);
  cfg.blockDim = dim3(pair::kThreads, 1, 1);
  cfg.dynamicSmemBytes = pair::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see grid_dependency_wait
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, p));
  return check_launch("8-bit pair gemm");
}

template <int LAYOUT, typename TOut, int BT>
int launch_swap(const Operands& o, const Params& p, int ranks, cudaStream_t stream) {
  CUtensorMap map_x, map_w;
  int rc = tmap(&map_x, o.act, p.k, p.m, o.act_stride, BT);
  if (rc == CONVROT_OK) rc = weight_map(&map_w, o, LAYOUT, p);
  if (rc != CONVROT_OK) return rc;
  auto kernel = swap::swap_kernel<LAYOUT, TOut, BT>;
  CONVROT_CUDA_CHECK(
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(swap::kSmem<BT>)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ranks), static_cast<unsigned>((p.n + 127) / 128),
                     static_cast<unsigned>((p.m + BT - 1) / BT));
  cfg.blockDim = dim3(swap::kThreads, 1, 1);
  cfg.dynamicSmemBytes = swap::kSmem<BT>;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, map_x, map_w, p));
  return check_launch("8-bit swap gemm");
}

template <int LAYOUT, typename TOut>
int launch(const Operands& o, const Params& p, cudaStream_t s) {
  const int sms = device_sm_count();
  const int64_t pair_tiles = static_cast<int64_t>((p.m + 255) / 256) * ((p.n + 255) / 256);
  // Pair tiles need most of the GPU's pairs to be busy; otherwise smaller
  // tiles, with K split until the CTAs fill the SMs.
  if (p.m > 128 && 4 * pair_tiles >= sms) return launch_pair<LAYOUT, TOut>(o, p, s);
  const int bt = p.m <= 16 ? 16 : p.m <= 32 ? 32 : p.m <= 64 ? 64 : 128;
  const int64_t tiles = static_cast<int64_t>((p.n + 127) / 128) * ((p.m + bt - 1) / bt);
  const int k_stages = (p.k + kBK - 1) / kBK;
  int ranks = 1;
  while (ranks < swap::kMaxCluster && 2 * ranks * tiles <= sms && 2 * ranks <= k_stages) ranks *= 2;
  switch (bt) {
    case 16: return launch_swap<LAYOUT, TOut, 16>(o, p, ranks, s);
    case 32: return launch_swap<LAYOUT, TOut, 32>(o, p, ranks, s);
    case 64: return launch_swap<LAYOUT, TOut, 64>(o, p, ranks, s);
    default: return launch_swap<LAYOUT, TOut, 128>(o, p, ranks, s);
  }
}

int check_args(const int8_t* act, int64_t act_stride, const int8_t* weight, int64_t weight_stride, int layout,
               const float* xscales, const void* out, int out_dtype, int64_t m, int64_t n, int64_t k) {
  CONVROT_REQUIRE(layout == CONVROT_LAYOUT_NK || layout == CONVROT_LAYOUT_KN, CONVROT_ERR_INVALID, "unknown layout %d",
                  layout);
  CONVROT_REQUIRE(valid_dtype(out_dtype), CONVROT_ERR_INVALID, "unknown output dtype %d", out_dtype);
  CONVROT_REQUIRE(m >= 0 && n > 0 && k > 0, CONVROT_ERR_INVALID, "invalid shape m=%lld n=%lld k=%lld",
                  static_cast<long long>(m), static_cast<long long>(n), static_cast<long long>(k));
  CONVROT_REQUIRE(k <= kMaxK, CONVROT_ERR_UNSUPPORTED, "k %lld can overflow the int32 dot (at most %d)",
                  static_cast<long long>(k), kMaxK);
  CONVROT_REQUIRE(m < (1LL << 22) && n < (1LL << 22), CONVROT_ERR_UNSUPPORTED, "shape too large");
  CONVROT_REQUIRE(act_stride >= k && weight_stride >= (layout == CONVROT_LAYOUT_NK ? k : n) && act_stride % 16 == 0 &&
                      weight_stride % 16 == 0,
                  CONVROT_ERR_INVALID, "row strides must cover the rows and be multiples of 16 bytes (%lld, %lld)",
                  static_cast<long long>(act_stride), static_cast<long long>(weight_stride));
  if (m == 0) return CONVROT_OK;
  CONVROT_REQUIRE(act && weight && xscales && out, CONVROT_ERR_INVALID, "null pointer");
  CONVROT_REQUIRE(aligned_to(act, 16) && aligned_to(weight, 16) && aligned_to(out, 16), CONVROT_ERR_INVALID,
                  "activation, weight and output must be 16-byte aligned");
  return CONVROT_OK;
}

int run(const Operands& o, int layout, const float* xscales, const float* wscales, const float* bias, void* out,
        int out_dtype, int64_t m, int64_t n, int64_t k, bool early_weights, cudaStream_t s) {
  Params p{xscales, wscales, bias, out, static_cast<int>(m), static_cast<int>(n), static_cast<int>(k),
           device_error_word(), early_weights ? 1 : 0};
  CONVROT_REQUIRE(p.err_word != nullptr, CONVROT_ERR_CUDA, "device error word unavailable");
  if (layout == CONVROT_LAYOUT_NK) {
    switch (out_dtype) {
      case CONVROT_BF16: return launch<CONVROT_LAYOUT_NK, __nv_bfloat16>(o, p, s);
      case CONVROT_F16: return launch<CONVROT_LAYOUT_NK, __half>(o, p, s);
      default: return launch<CONVROT_LAYOUT_NK, float>(o, p, s);
    }
  }
  switch (out_dtype) {
    case CONVROT_BF16: return launch<CONVROT_LAYOUT_KN, __nv_bfloat16>(o, p, s);
    case CONVROT_F16: return launch<CONVROT_LAYOUT_KN, __half>(o, p, s);
    default: return launch<CONVROT_LAYOUT_KN, float>(o, p, s);
  }
}

}  // namespace
}  // namespace i8
}  // namespace convrot

extern "C" {

int convrot_i8_gemm(const int8_t* act, int64_t act_stride, const int8_t* weight, int64_t weight_stride, int layout,
                    const float* xscales, const float* wscales, const float* bias, void* out, int out_dtype, int64_t m,
                    int64_t n, int64_t k, void* stream) {
  using namespace convrot;
  const int rc = i8::check_args(act, act_stride, weight, weight_stride, layout, xscales, out, out_dtype, m, n, k);
  if (rc != CONVROT_OK || m == 0) return rc;
  return i8::run({act, weight, act_stride, weight_stride}, layout, xscales, wscales, bias, out, out_dtype, m, n, k,
                 /*early_weights=*/false, static_cast<cudaStream_t>(stream));
}

int convrot_i8_linear(const void* x, int x_dtype, int64_t x_stride, const float* col_scale, const int8_t* weight,
                      int64_t weight_stride, int layout, const float* wscales, const float* bias, void* out,
                      int out_dtype, int64_t m, int64_t n, int64_t k, int8_t* codes, int64_t codes_stride,
                      float* scales, void* stream) {
  using namespace convrot;
  int rc = i8::check_args(codes, codes_stride, weight, weight_stride, layout, scales, out, out_dtype, m, n, k);
  if (rc != CONVROT_OK) return rc;
  rc = convrot_quantize_i8(x, x_dtype, m, k, x_stride, col_scale, codes, codes_stride, scales, stream);
  if (rc != CONVROT_OK || m == 0) return rc;
  // The kernel before the product is the quantizer, which writes no weight
  // and lets the product start only once everything before it is complete.
  return i8::run({codes, weight, codes_stride, weight_stride}, layout, scales, wscales, bias, out, out_dtype, m, n, k,
                 /*early_weights=*/true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
