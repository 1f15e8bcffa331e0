// 8-bit integer matrix product with one scale for each token (row of the
// activation) and one for each channel (row of the weight):
//   out[m, n] = T(fl(fl(float(sum_k a[m, k] w[n, k]) * xs[m]) * ws[n]) + bias[n]),
// with an exact int32 dot (K <= 131072: |dot| <= 127 * 127 K < 2^31).
// Layout NK reads w as (n, k) rows, the forward product; layout KN reads it
// as (k, n) rows: the same weight matrix contracted over its rows, the
// product of the input's gradient.  Integer sums are exact, so neither the
// tiling nor the split of K changes a bit.
//
// Up to 8 tokens of the forward product: gemv_kernel, weights from memory into
// mma.sync fragments, bound by reading them once and by latency.  Else two
// kernels on tcgen05 kind::i8, operands by TMA in 128-byte-swizzled tiles,
// accumulators in TMEM:
// * pair_kernel: CTA pairs (cta_group::2), 256 tokens x 256 channels a tile,
//   persistent, for products that fill the GPU with such tiles.  Bound by the
//   copies and the MMAs holding up one another: a stage of 128 K takes the MMAs
//   alone 0.27 us, the copies alone 0.28, both 0.37 in one wave and 0.39 to 0.42
//   over many, while no unit is full (4096 x 3072 x 12288: tensor pipe active in
//   58% of the cycles, its reads of shared memory 29% of their peak rate, copies
//   into an SM 38 bytes a cycle, L2 37%).  8192^3 in 372 us (2950 TOPS); 4096 x
//   3072 x 12288 (tokens, K, channels) in 117 us (2630), 6% of it for the last
//   wave's idle pairs; 1536 x 3072 x 3072, one wave, in 16 us, of which 7 are
//   launch, first copies and the last tile's epilogue.  A tile's whole K is one
//   pair's work, so few tiles of a long K are far from either limit: 512 x 12288
//   x 3072, 24 tiles for 74 pairs, 33 us, floor 12.  Tiles of 192 channels take as
//   long a stage as 256 (0.36; 136 us instead of 117 for 12288 channels), so
//   they gain only where both give one wave: 13.3 us instead of 14.8 for 2000 x
//   1000 x 3000, too little for a second set of kernels.  Rings of 4 stages
//   125 us, copies in halves 117.
// * swap_kernel: 128 channels on the MMA's M side and 16 to 128 tokens on its
//   N side, K split over a cluster, for few tokens or few tiles.  Its tiles
//   read each operand twice as often as the pairs', and a stage takes a CTA 0.46
//   us, the latency of its ring, or more where two share an SM: 100 x 12288 x 3072
//   17 us (floor 6), 333 x 12288 x 3072 31 (8).
#include <algorithm>

#include "tile8.cuh"

namespace convrot {

namespace i8 {

using namespace tile8;

constexpr int kMaxK = 131072;

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
constexpr int kBand = 16;
constexpr int kStages = 6;
constexpr int kOpBytes = 128 * kBK;  // one operand's half tile of a stage
constexpr int kWarpA = 0, kWarpMma = 1, kWarpB = 2, kWarpE0 = 4, kEWarps = 8;
constexpr int kThreads = (kWarpE0 + kEWarps) * 32;
constexpr uint32_t kTmemCols = 2 * kTile;
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
  // Tiles in bands of kBand token tiles, within a band all of these for one
  // channel tile, then the next: the tiles in work at one time then share
  // about as many rows of either operand in L2.
  auto place = [&](int tile, int& m_blk, int& n_blk) {
    const int band = tile / (kBand * n_tiles), first = band * kBand;
    const int rows = min(kBand, m_tiles - first), at = tile - first * n_tiles;
    n_blk = at / rows;
    m_blk = first + at - n_blk * rows;
  };

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
        int m_blk, n_blk;
        place(tile, m_blk, n_blk);
        const int row = m_blk * kTile + 128 * rank, col = n_blk * kTile + 128 * rank;
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
    const uint32_t lead_empty0 = mapa_shared(&bars->acc_empty[0], 0);
    int local = 0;
    for (int tile = pair_id; tile < num_tiles; tile += num_pairs, ++local) {
      const int buf = local & 1;
      int m_blk, n_blk;
      place(tile, m_blk, n_blk);
      const int row0 = m_blk * kTile + 128 * rank + quarter * 32, col0 = n_blk * kTile + 128 * half;
      const float xs = row0 + lane < p.m ? ld_f32(p.xscales + row0 + lane) : 0.0f;
      __syncwarp();  // the previous tile's reads of the vectors are done
      for (int j = lane; j < 128; j += 32) {
        const bool in = col0 + j < p.n;
        sws[j] = in ? (p.wscales ? ld_f32(p.wscales + col0 + j) : 1.0f) : 0.0f;
        sbias[j] = in && p.bias ? ld_f32(p.bias + col0 + j) : 0.0f;
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
        store_rows(v, stage_out + ew * kChunkBytes, static_cast<TOut*>(p.out), row0, col0 + c * 32, p.m, p.n);
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

// two CTAs for each SM
template <int BT> constexpr int kStages = BT <= 32 ? 5 : (BT == 64 ? 4 : 3);
template <int BT> constexpr int kXBytes = BT * kBK;
template <int BT>
constexpr size_t kSmem = 1024 + kStages<BT> * (kWBytes + kXBytes<BT>) + BT * 4 + sizeof(Bars);
static_assert(kSmem<128> <= 113 * 1024 && kSmem<64> <= 113 * 1024 && kSmem<32> <= 113 * 1024, "shared memory budget");

// The sums of R ranks (token, 128 channels) for tokens c_lo to c_hi, every
// fourth of them a warp's, a lane with four channels; tokens past the last are
// read, in bounds, and not handed on.  16 reads of a thread are in flight: the
// latency between SMs is what this takes.
template <int R, int BT, typename Emit>
__device__ __forceinline__ void join(const uint32_t* part, int c_lo, int c_hi, Emit&& emit) {
  constexpr int kTokens = 16 / R;
  uint32_t peer[R];
#pragma unroll
  for (int r = 0; r < R; ++r) peer[r] = mapa_shared(part + (threadIdx.x & 31) * 4, r);
  for (int c = c_lo + (threadIdx.x >> 5); c < c_hi; c += 4 * kTokens) {
    uint4 v[kTokens][R];
#pragma unroll
    for (int t = 0; t < kTokens; ++t)
#pragma unroll
      for (int r = 0; r < R; ++r) v[t][r] = dsmem_ld128(peer[r] + min(c + 4 * t, BT - 1) * 512);
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      uint4 sum = v[t][0];
#pragma unroll
      for (int r = 1; r < R; ++r) sum.x += v[t][r].x, sum.y += v[t][r].y, sum.z += v[t][r].z, sum.w += v[t][r].w;
      if (c + 4 * t < c_hi) emit(sum, c + 4 * t);
    }
  }
}

template <int LAYOUT, typename TOut, int BT>
__global__ void __launch_bounds__(kThreads, 2)
    swap_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const Params p) {
  constexpr int S = kStages<BT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sX = sW + S * kWBytes;
  float* xs = reinterpret_cast<float*>(sX + S * kXBytes<BT>);  // the tokens' scales
  Bars* bars = reinterpret_cast<Bars*>(xs + BT);
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
  grid_dependents_launch();

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
  if (warp == 3) {  // has waited for the previous kernel
    for (int c = lane; c < BT; c += 32) xs[c] = m0 + c < p.m ? ld_f32(p.xscales + m0 + c) : 0.0f;
  }
  __syncthreads();
  const bool done = wait(&bars->mma_done, 0, &bars->err, 74);
  tc_fence_after();

  TOut* out = static_cast<TOut*>(p.out);
  const uint32_t t_row = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
  const int rows = p.m - m0 < BT ? p.m - m0 : BT;
  if (ranks == 1) {
    const int n = n0 + warp * 32 + lane;
    const bool n_ok = n < p.n;
    const float ws = n_ok && p.wscales ? ld_f32(p.wscales + n) : 1.0f;
    const float b = n_ok && p.bias ? ld_f32(p.bias + n) : 0.0f;
    for (int c = 0; c < rows && done; c += 16) {
      uint32_t r[16];
      __syncwarp();
      tmem_ld_32x32b_x16(t_row + c, r);
      tmem_ld_wait();
      // all values first, then all stores, since one warp a scheduler has only
      // itself to overlap
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        v[i] = __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(static_cast<int32_t>(r[i])), xs[c + i]), ws), b);
      TOut* dst = out + static_cast<int64_t>(m0 + c) * p.n + n;
      if (rows - c >= 16 && n_ok) {
#pragma unroll
        for (int i = 0; i < 16; ++i, dst += p.n) *dst = cvt_out<TOut>(v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i, dst += p.n)
          if (i < rows - c && n_ok) *dst = cvt_out<TOut>(v[i]);
      }
    }
  } else {
    const int n = n0 + 4 * lane;  // of four channels
    float ws[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ws[i] = n + i < p.n && p.wscales ? ld_f32(p.wscales + n + i) : 1.0f;
      b[i] = n + i < p.n && p.bias ? ld_f32(p.bias + n + i) : 0.0f;
    }
    const bool whole = p.n % 4 == 0;  // four channels in one store
    // int32 sums (token, channel) over the ring, whose copies have all been consumed
    uint32_t* part = reinterpret_cast<uint32_t*>(smem);
    for (int c = 0; c < rows && done; c += 16) {
      uint32_t r[16];
      __syncwarp();
      tmem_ld_32x32b_x16(t_row + c, r);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) part[(c + i) * 128 + warp * 32 + lane] = r[i];
    }
    __syncwarp();
    cluster_sync();
    const int c_lo = rows * rank / ranks, c_hi = done ? rows * (rank + 1) / ranks : 0;  // this CTA's share of the tokens
    auto emit = [&](const uint4& dots, int c) {
      const uint32_t dot[4] = {dots.x, dots.y, dots.z, dots.w};
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = __fadd_rn(__fmul_rn(__fmul_rn(__int2float_rn(static_cast<int32_t>(dot[i])), xs[c]), ws[i]), b[i]);
      TOut* dst = out + static_cast<int64_t>(m0 + c) * p.n + n;
      if (whole) {
        Pack<TOut, 4> pk;
        pk.set(v);
        if (n < p.n) pk.store(dst);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < p.n) dst[i] = cvt_out<TOut>(v[i]);
      }
    };
    if (ranks == 2) join<2, BT>(part, c_lo, c_hi, emit);
    else if (ranks == 4) join<4, BT>(part, c_lo, c_hi, emit);
    else join<8, BT>(part, c_lo, c_hi, emit);
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

// ===========================================================================
// GEMV kernel, up to 8 tokens.  A CTA has 16 channels; its 8 warps share out
// K in units of 64.  Thread (g, t) of a warp reads 16 bytes of channels g and
// g + 8 at k = 16 t of a unit: the four words of both are the A fragments of
// two MMAs (m16n8k32), with word 2 i as the fragment's first half of k and
// word 2 i + 1 as the second.  Which k a fragment index stands for only has to
// agree with the B fragment, which are the same four words of token g's codes.
// So weights go from memory to the MMA with no rearrangement, 64 contiguous
// bytes of a channel for each quad of lanes; two sets of four units are in
// flight in registers, also from one block of channels to the next (two CTAs
// for each SM walk the blocks).  The codes of all tokens are in shared memory, copied,
// or (FUSED, one or two tokens) formed there from x by every CTA itself, which
// costs less than a kernel of its own before this one.  Weights from HBM: 1 x
// 4096 x 4096 in 6.8 us (5.9 from L2), 8 x 4096 x 4096 in 7.6, 8 x 4096 x 12288
// in 14.1 (3.6 TB/s; a launch, a trip to memory and the join of the warps' sums
// are about 4 of each).
// ===========================================================================
namespace gemv {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kChannels = 16;
constexpr int kUnit = 64;
constexpr int kAhead = 4;  // units of a register set
constexpr int kMaxTokens = 8;
constexpr int kMaxFused = 2;
constexpr int kFusedVectors = 2;  // 16-byte vectors of a token a thread holds
constexpr int kMaxCodes = 96 * 1024;  // bytes of codes in shared memory

struct GemvParams {
  Params p;
  const void* x;  // FUSED: the activation, x_stride elements a row
  const int8_t* act;
  const int8_t* weight;
  int64_t x_stride, act_stride, weight_stride;
};

// Pitch of a token's codes: whole units, 64 bytes off a multiple of 128, so
// that two tokens' quads fall on different banks.
__host__ __device__ constexpr int pitch_of(int k) { return (k + kUnit - 1) / kUnit / 2 * 2 * kUnit + kUnit; }

__device__ __forceinline__ void mma_s8(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename TOut, bool FUSED>
__global__ void __launch_bounds__(kThreads, 2) gemv_kernel(const GemvParams q) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ int32_t part[2][kWarps][kMaxTokens][kChannels + 1];
  __shared__ float xs[kMaxTokens];
  __shared__ uint32_t red[kMaxFused][kWarps];
  const Params& p = q.p;
  int8_t* codes = reinterpret_cast<int8_t*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int pitch = pitch_of(p.k), units = (p.k + kUnit - 1) / kUnit;
  const int u_lo = units * warp / kWarps, u_hi = units * (warp + 1) / kWarps;
  const int blocks = (p.n + kChannels - 1) / kChannels;

  if (!p.early_weights) grid_dependency_wait();
  uint4 wa[2][kAhead], wb[2][kAhead];
  // The sets of this warp in its order: units from `at_u` on of channel block
  // `at_n`; past a block's last unit comes the next block.
  int at_n = blockIdx.x, at_u = u_lo;
  auto fetch = [&](uint4 (&w)[2][kAhead]) {
    const int n0 = at_n * kChannels;
    // channels past the last are read as the last, and not written
    const int8_t* row0 = q.weight + static_cast<int64_t>(min(n0 + g, p.n - 1)) * q.weight_stride;
    const int8_t* row1 = q.weight + static_cast<int64_t>(min(n0 + g + 8, p.n - 1)) * q.weight_stride;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int k0 = (at_u + i) * kUnit + 16 * t;
      const bool in = at_n < blocks && at_u + i < u_hi && k0 < p.k;
      w[0][i] = in ? load16(row0, k0, p.k - k0) : make_uint4(0, 0, 0, 0);
      w[1][i] = in ? load16(row1, k0, p.k - k0) : make_uint4(0, 0, 0, 0);
    }
    at_u += kAhead;
  };
  auto fetch_two = [&] {  // a block's sets come in pairs, the second perhaps empty
    fetch(wa);
    fetch(wb);
  };
  fetch_two();
  if (p.early_weights) grid_dependency_wait();
  grid_dependents_launch();

  if constexpr (FUSED) {
    // every CTA quantizes the tokens for itself
    constexpr int W = 16 / sizeof(TOut);
    Pack<TOut, W> x[kMaxFused][kFusedVectors];
#pragma unroll
    for (int m = 0; m < kMaxFused; ++m)
#pragma unroll
      for (int j = 0; j < kFusedVectors; ++j) {
        const int c = (threadIdx.x + j * kThreads) * W;
        x[m][j].clear();
        if (m < p.m && c < p.k) {
          const TOut* src = static_cast<const TOut*>(q.x) + m * q.x_stride + c;
          if (c + W <= p.k) x[m][j].load_ahead(src);
          else x[m][j].load_part(src, p.k - c);
        }
      }
#pragma unroll
    for (int m = 0; m < kMaxFused; ++m) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < kFusedVectors; ++j) top = max(top, x[m][j].top());
      top = warp_max(top);
      if (lane == 0) red[m][warp] = top;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < kMaxFused; ++m) {
      if (m >= p.m) break;
      const uint32_t top = warp_max(lane < kWarps ? red[m][lane] : 0u);
      const Quant8<float> quant(top);
      if (threadIdx.x == 0) xs[m] = scale8(top);
#pragma unroll
      for (int j = 0; j < kFusedVectors; ++j) {
        const int c = (threadIdx.x + j * kThreads) * W;
        if (c < units * kUnit) {
          float v[W];
          uint32_t code[W];
          x[m][j].get(v);
          quant.codes(v, code);
          store_codes<W>(codes + m * pitch + c, code, quant.mask());
        }
      }
    }
  } else {
    const int chunks = units * (kUnit / 16);
    for (int i = threadIdx.x; i < chunks; i += kThreads) {  // one place of all tokens at a time
      const int k0 = i * 16;
#pragma unroll 1
      for (int m0 = 0; m0 < p.m; m0 += 4) {
        uint4 v[4];
#pragma unroll
        for (int m = 0; m < 4; ++m)
          v[m] = m0 + m < p.m && k0 < p.k ? load16(q.act + (m0 + m) * q.act_stride, k0, p.k - k0)
                                          : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < 4; ++m)
          if (m0 + m < p.m) *reinterpret_cast<uint4*>(codes + (m0 + m) * pitch + k0) = v[m];
      }
    }
    if (threadIdx.x < p.m) xs[threadIdx.x] = ld_f32(p.xscales + threadIdx.x);
  }
  __syncthreads();

  auto use = [&](const uint4 (&w)[2][kAhead], int u, int32_t (&acc)[4]) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (u + i >= u_hi) break;  // uniform across the warp
      uint4 b = make_uint4(0, 0, 0, 0);
      if (g < p.m) b = *reinterpret_cast<const uint4*>(codes + g * pitch + (u + i) * kUnit + 16 * t);
      mma_s8(acc, w[0][i].x, w[1][i].x, w[0][i].y, w[1][i].y, b.x, b.y);
      mma_s8(acc, w[0][i].z, w[1][i].z, w[0][i].w, w[1][i].w, b.z, b.w);
    }
  };
  int turn = 0;
  for (int block = blockIdx.x; block < blocks; block += gridDim.x, turn ^= 1) {
    int32_t acc[4] = {};
    int u = u_lo;
    do {  // each pair of sets is followed by the next pair's loads
      const bool last = u + 2 * kAhead >= u_hi;
      if (last) {
        at_n = block + gridDim.x;
        at_u = u_lo;
      }
      use(wa, u, acc);
      fetch(wa);
      use(wb, u + kAhead, acc);
      fetch(wb);
      u += 2 * kAhead;
    } while (u < u_hi);
    // fragment C: rows g and g + 8 (channels), columns 2 t and 2 t + 1 (tokens)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[turn][warp][2 * t + (i & 1)][g + 8 * (i >> 1)] = acc[i];
    __syncthreads();
    const int m = threadIdx.x / kChannels, n = block * kChannels + threadIdx.x % kChannels;
    if (m < p.m && n < p.n) {
      int32_t dot = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) dot += part[turn][w][m][threadIdx.x % kChannels];
      float v = __fmul_rn(__int2float_rn(dot), xs[m]);
      if (p.wscales) v = __fmul_rn(v, ld_f32(p.wscales + n));
      if (p.bias) v = __fadd_rn(v, ld_f32(p.bias + n));
      static_cast<TOut*>(p.out)[static_cast<int64_t>(m) * p.n + n] = cvt_out<TOut>(v);
    }
  }
}

}  // namespace gemv

// ---------------------------------------------------------------------------
// host side

namespace {

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

template <typename TOut, bool FUSED>
int launch_gemv(const gemv::GemvParams& q, cudaStream_t stream) {
  auto kernel = gemv::gemv_kernel<TOut, FUSED>;
  const int smem = q.p.m * gemv::pitch_of(q.p.k);
  CONVROT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, gemv::kMaxCodes));
  cudaLaunchConfig_t cfg = {};
  const int blocks = (q.p.n + gemv::kChannels - 1) / gemv::kChannels, most = 2 * device_sm_count();
  cfg.gridDim = dim3(static_cast<unsigned>(blocks < most ? blocks : most), 1, 1);
  cfg.blockDim = dim3(gemv::kThreads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, q));
  return check_launch("8-bit gemv");
}

bool gemv_takes(int layout, int64_t m, int64_t k) {
  return layout == CONVROT_LAYOUT_NK && m <= gemv::kMaxTokens && m * gemv::pitch_of(static_cast<int>(k)) <= gemv::kMaxCodes;
}

// x quantized inside the product.
template <typename T>
int launch_fused(const void* x, int64_t x_stride, const Operands& o, Params p, cudaStream_t s) {
  p.early_weights = 0;  // the previous kernel of the stream may have written them
  return launch_gemv<T, true>({p, x, nullptr, o.weight, x_stride, 0, o.weight_stride}, s);
}

// Expected times of the two tile kernels in microseconds, fitted to sweeps of
// 16 to 1024 tokens, 512 to 12288 channels and K from 128 to 12288 (times of a
// call in a graph).  A stage of 128 K takes a pair 0.36 us in one wave; 0.45 over
// several lies between the 0.39 of K = 4096 and the 0.6 of K = 1024, whose waves'
// fill is no term of its own.  A swap CTA takes 0.46 us for a stage (the latency of its
// ring), more where two CTAs of an SM share 125 bytes a nanosecond; its
// epilogue takes 12 ns a token and the exchange of a split K the more, the more
// tokens and CTAs take part; a second wave of CTAs costs all of that again.
// Over the 72 sizes of 12 to 1000 tokens that it was fitted to the choices take
// 1% longer than the best of all splits and both kernels.  Measured on either side (tokens, K,
// channels; weights from HBM): 64 x 4096 x 4096 swap 10.2, pair 17.3; 512 x 4096
// x 4096 swap 16.5, pair 18.0; 200 x 4096 x 12288 swap 22.8, pair 19.6; 1000 x
// 3072 x 3072 swap 17.8, pair 15.8.
double pair_time(const Params& p, int sms) {
  const int64_t tiles = static_cast<int64_t>((p.m + 255) / 256) * ((p.n + 255) / 256), pairs = sms / 2;
  const int64_t waves = (tiles + pairs - 1) / pairs, stages = (p.k + kBK - 1) / kBK;
  return 6.0 + static_cast<double>(waves * stages) * (waves > 1 ? 0.45 : 0.36);
}

// The best split of K over 1, 2, 4 or 8 CTAs, and its time: 64 x 4096 x 12288
// takes 15.9 in two and 28 in eight, whose CTAs are three waves; 64 x 12288 x
// 3072 28 and 14.3.  (Splits in three pack badly into the GPU's clusters of SMs;
// clusters of four or eight do not fill it either: 72 of four are two waves.)
double swap_time(const Params& p, int bt, int sms, int* ranks) {
  const int64_t tiles = static_cast<int64_t>((p.n + 127) / 128) * ((p.m + bt - 1) / bt);
  const int64_t stages = (p.k + kBK - 1) / kBK;
  double best = 1e30;
  for (int r = 1; r <= swap::kMaxCluster && r <= stages; r *= 2) {
    const int64_t ctas = tiles * r, at_once = r < 4 ? 2 * sms : 2 * sms / 8 * 7;
    const int64_t waves = (ctas + at_once - 1) / at_once;
    const bool shared = ctas > sms;
    const double stage = shared ? std::max(0.46, 2.0 * (swap::kWBytes + bt * kBK) / 125e3) : 0.46;
    const double exchange = r > 1 ? 0.9 + 0.08 * r + bt * (0.006 + 0.001 * r) : 0.0;
    const double t = static_cast<double>(waves) * (2.8 + 0.012 * bt + static_cast<double>((stages + r - 1) / r) * stage +
                                                   exchange + (shared ? 0.4 + 0.007 * bt : 0.0));
    if (t < best) {
      best = t;
      *ranks = r;
    }
  }
  return best;
}

template <int LAYOUT, typename TOut>
int launch(const Operands& o, const Params& p, cudaStream_t s) {
  const int sms = device_sm_count();
  if (gemv_takes(LAYOUT, p.m, p.k)) {
    const gemv::GemvParams q{p, nullptr, o.act, o.weight, 0, o.act_stride, o.weight_stride};
    return launch_gemv<TOut, false>(q, s);
  }
  const int bt = p.m <= 16 ? 16 : p.m <= 32 ? 32 : p.m <= 64 ? 64 : 128;
  int ranks = 1;
  const double swap_us = swap_time(p, bt, sms, &ranks);
  if (pair_time(p, sms) < swap_us) return launch_pair<LAYOUT, TOut>(o, p, s);
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
  // One or two tokens: quantized inside the product, one kernel instead of two
  // (1 x 4096 x 4096: 7.1 us, 7.4 as two, and less work for the host).
  const int64_t x_size = valid_dtype(x_dtype) ? static_cast<int64_t>(dtype_size(x_dtype)) : 1;
  if (m > 0 && m <= i8::gemv::kMaxFused && !col_scale && x_dtype == out_dtype && i8::gemv_takes(layout, m, k) &&
      k * x_size <= i8::gemv::kFusedVectors * i8::gemv::kThreads * 16 && aligned_to(x, 16) && x_stride * x_size % 16 == 0) {
    CONVROT_REQUIRE(x != nullptr && x_stride >= k, CONVROT_ERR_INVALID, "null pointer, or a row stride below k");
    const i8::Operands o{codes, weight, codes_stride, weight_stride};
    const i8::Params p{scales, wscales, bias, out, static_cast<int>(m), static_cast<int>(n), static_cast<int>(k),
                       nullptr, 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (x_dtype) {
      case CONVROT_BF16: return i8::launch_fused<__nv_bfloat16>(x, x_stride, o, p, s);
      case CONVROT_F16: return i8::launch_fused<__half>(x, x_stride, o, p, s);
      default: return i8::launch_fused<float>(x, x_stride, o, p, s);
    }
  }
  rc = convrot_quantize_i8(x, x_dtype, m, k, x_stride, col_scale, codes, codes_stride, scales, stream);
  if (rc != CONVROT_OK || m == 0) return rc;
  // The kernel before the product is the quantizer, which writes no weight
  // and lets the product start only once everything before it is complete.
  return i8::run({codes, weight, codes_stride, weight_stride}, layout, scales, wscales, bias, out, out_dtype, m, n, k,
                 /*early_weights=*/true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
