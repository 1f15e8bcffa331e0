// 8-bit floating-point matrix product with a power-of-two scale for each block
// of 128:
//   out[m, n] = T(sum_b 2^(xs[m, b] + ws[n / 128, b]) sum_{k in b} a[m, k] w[n, k] + bias[n]),
// a and w e4m3 codes, b the blocks of 128 along K, sums in float32.  Layout NK
// reads w as (n, k) rows, the forward product; layout KN reads it as (k, n)
// rows: the same weight contracted over its rows, the product of the input's
// gradient.  The blocks of a weight are square, so its scales serve both.
//
// The products run on tcgen05 kind::mxf8f6f4, which multiplies each group of 32
// products by two power-of-two scales held in tensor memory: all four groups of
// a block name the same scale, and nothing is left to do for it outside of the
// tensor core.  Scales of 128 rows x 4 blocks are 512 bytes, row r at
// 16 (r % 32) + 4 (r / 32), one byte a block: so a warp forms them in shared
// memory from the rows' 4-byte words, and one tcgen05.cp brings them into 4
// columns of tensor memory, for 4 stages of K.
//
// Three kernels: gemv_kernel up to 8 tokens of the forward product, pair_kernel
// for products that fill the GPU with tiles of 256 x 256, swap_kernel between.
// Times of the product alone, weights from HBM, bf16 out (tokens x K x channels,
// us): 1 x 5120 x 5120 10.6 (26 MB; 4.0 at a copy's bandwidth), 8 x 5120 x 5120
// 13.4, 40 x 5120 x 5120 14.2, 451 x 2203 x 1301 13.0, 1536 x 5120 x 5120 46,
// 4096 x 3072 x 12288 142, 7800 x 5120 x 13824 480 (2300 TFLOP/s), 8192^3 458; for
// the gradient, whose few tokens the GEMV does not take, 1 x 5120 x 5120 12.0, 8
// 12.6, 40 14.3.
#include <algorithm>

#include "fp8.cuh"
#include "tile8.cuh"

namespace convrot {
namespace fp8 {

using namespace tile8;

constexpr int kGroup = 4;            // stages whose scales are copied at a time: the bytes of a word
constexpr int kScaleBytes = 512;     // of 128 rows and a group
constexpr uint32_t kOneWord = 0x7F7F7F7Fu;  // four scales of 1

struct Params {
  const uint8_t* xscales;  // (m, blocks of k): rows at multiples of 4 bytes, xs_stride bytes apart
  const uint8_t* wscales;  // of block n of the output and block b of K: n * ws_n + b * ws_k
  int64_t xs_stride, ws_n, ws_k;
  const float* bias;  // may be null: zeros
  void* out;
  int m, n, k;
  int* err_word;
  // the weight copies may be issued before the previous kernel of the stream
  // has completed (it only writes the activation)
  int early_weights;
  int add;  // float32 outputs: to what `out` holds
};

// Channels whose products one float32 output sums on the tensor core.  It adds
// 32 products at a time and cuts what is below the sum's last bit, so its error
// grows with their number: 5e-7 of the outputs' norm over 8192 channels, 1.1e-6
// over 15360, 3e-6 over 32768.  No 16-bit output shows that; float32 outputs of
// the tile kernels are summed in ranges, one launch after another, and the
// ranges in order (5e-7 over 32768).
constexpr int kMaxSum = 8192;

// tcgen05 instruction descriptor of kind::mxf8f6f4 with D float32: A and B e4m3
// (format 0), A M-major for amn, B N-major for bmn, scales ue8m0 (bit 23).  The
// byte of the scale words that an MMA reads goes into bits 29-30 (A) and 4-5 (B).
__host__ __device__ constexpr uint32_t idesc_mx(int m, int n, bool amn, bool bmn) {
  return (static_cast<uint32_t>(amn) << 15) | (static_cast<uint32_t>(bmn) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(m >> 7) << 27);
}
__device__ __forceinline__ uint32_t idesc_byte(uint32_t idesc, int byte) {
  return idesc | static_cast<uint32_t>(byte) << 29 | static_cast<uint32_t>(byte) << 4;
}

__device__ __forceinline__ void mma_mx(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t a_scale, uint32_t b_scale, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scale), "r"(b_scale), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void mma_mx_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t a_scale, uint32_t b_scale, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scale), "r"(b_scale), "r"(accumulate)
      : "memory");
}

// 512 bytes of scales (32 rows of 16, contiguous) to 4 columns of tensor
// memory, the same for each quarter of its lanes.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t saddr) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(smem_desc(saddr, 16, 128, 0))
               : "memory");
}

// The same in both CTAs of a pair, each from its own shared memory.
__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint32_t saddr) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(smem_desc(saddr, 16, 128, 0))
               : "memory");
}

// Bytes b0 to b0 + 3 of a row of scales: a row begins on a multiple of 4 bytes
// and is padded to one, and b0 lies in it.  What lies past its end is not read
// from memory and not used.
__device__ __forceinline__ uint32_t scale_word(const uint8_t* row, int b0, int blocks) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(row) + (b0 >> 2);
  const uint32_t lo = ld_32(w);
  if ((b0 & 3) == 0) return lo;
  const uint32_t hi = ((b0 >> 2) + 1) * 4 < blocks ? ld_32(w + 1) : 0u;
  return __funnelshift_r(lo, hi, 8 * (b0 & 3));
}

// The scales of output block `nb` of the weight for K blocks b0 to b0 + 3: a
// byte in each of four lanes, and from these the word in every lane of the warp.
__device__ __forceinline__ uint32_t weight_byte(const Params& p, int nb, int b0, int blocks) {
  const int b = b0 + (threadIdx.x & 3);
  return b < blocks && nb * 128 < p.n ? ld_8(p.wscales + nb * p.ws_n + b * p.ws_k) : 0x7Fu;
}
__device__ __forceinline__ uint32_t word_of(uint32_t byte) {
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) word |= __shfl_sync(0xFFFFFFFFu, byte, i) << (8 * i);
  return word;
}

// An arrival that publishes nothing of its own.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t bar_cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}

// ===========================================================================
// Pair kernel.  CTA pairs (cta_group::2), 256 tokens x 256 channels a tile,
// persistent.  Each CTA holds 128 tokens and 128 channels of a tile:
//   warp 0   activation producer, warp 2 weight producer: lane s issues the
//            16 KB box of ring slot s (copies of one thread are served one
//            after another), completing on the leader's full[s]
//   warp 1   leader: MMA issuer (M = 256, N = 256); both: TMEM owner
//   warp 3   scales of this CTA's 128 tokens and of the tile's 256 channels,
//            which both CTAs need
//   warps 4-11  epilogue of this CTA's 128 rows: warp w reads TMEM lanes
//            32 (w % 4) .. + 31, columns 128 ((w - 4) / 4) .. + 127
// Tensor memory has 512 columns: two accumulators of 256 that share 32, and
// two sets of scales of 12 (4 for the tokens, 8 for the channels).  The epilogue
// reads the shared columns first, and with them free the next tile may begin.
// In loops of two seconds, which the power limit holds at 1.52 to 1.57 GHz for this
// kernel and the integer one alike: 8192^3 547 us (at 1552 MHz; the integer kernel
// 437 at 1522), 7800 x 5120 x 13824 569 (1567; 465 at 1545).  So it takes 1.28 and
// 1.24 times the integer kernel's cycles, the copies of scales among them, and
// the clock takes the rest of what a call's loop has over a short run's.
// ===========================================================================
namespace pair {

constexpr int kTile = 256;
constexpr int kBand = 16;
constexpr int kStages = 6;
constexpr int kOpBytes = 128 * kBK;  // one operand's half tile of a stage
constexpr int kWarpA = 0, kWarpMma = 1, kWarpB = 2, kWarpS = 3, kWarpE0 = 4, kEWarps = 8;
constexpr int kThreads = (kWarpE0 + kEWarps) * 32;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kSecond = 224;    // column of the second accumulator
constexpr uint32_t kScaleCol = 480;  // 16 columns for each of two sets of scales
constexpr int kSetBytes = 3 * kScaleBytes;
constexpr int kVecBytes = kEWarps * 128 * 4;  // bias of a warp's 128 columns

struct alignas(8) Bars {
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t shared_empty;
  uint64_t mma_done;
  uint32_t tmem_base;
  int err;
};

constexpr size_t kSmem = 1024 + kStages * 2 * kOpBytes + 2 * kSetBytes + kEWarps * kChunkBytes + kVecBytes + sizeof(Bars);
static_assert(kSmem <= 232448, "shared memory budget");

template <int LAYOUT, typename TOut>
__global__ void __launch_bounds__(kThreads, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + kStages * kOpBytes;
  uint8_t* sS = sB + kStages * kOpBytes;  // each set: tokens, channels 0-127, channels 128-255
  uint8_t* stage_out = sS + 2 * kSetBytes;
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
      mbar_init(&bars->full[s], 3);  // the copies, and the scales of either CTA
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], 2 * kEWarps);
    }
    mbar_init(&bars->shared_empty, kEWarps);  // four warps of each CTA
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
          if (!wait(&bars->empty[lane], ((g / kStages) & 1) ^ 1, &bars->err, 81)) { ok = false; break; }
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
  } else if (warp == kWarpS) {
    // Each group's words are on their way while the group before is written: a
    // trip to memory takes as long as the MMAs of two to three stages.  A
    // stage is full only with this warp's arrival too, so that the MMA thread
    // has nothing more to wait for or to commit than without scales.
    const uint32_t lead_full0 = mapa_shared(&bars->full[0], 0);
    struct {
      uint32_t x[4], w0, w1;
    } now, next = {};
    int ahead = pair_id, b0 = 0;
    auto load_next = [&] {  // of group b0 of tile `ahead`, and on to the one after
      if (ahead >= num_tiles) return;
      int m_blk, n_blk;
      place(ahead, m_blk, n_blk);
      const int row = m_blk * kTile + 128 * rank + lane;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        next.x[j] = row + 32 * j < p.m ? scale_word(p.xscales + (row + 32 * j) * p.xs_stride, b0, k_stages) : kOneWord;
      next.w0 = weight_byte(p, 2 * n_blk, b0, k_stages);
      next.w1 = weight_byte(p, 2 * n_blk + 1, b0, k_stages);
      b0 += kGroup;
      if (b0 >= k_stages) {
        b0 = 0;
        ahead += num_pairs;
      }
    };
    auto wait_empty = [&](int stage) {  // whose MMAs are complete
      const bool ok = wait(&bars->empty[stage % kStages], (stage / kStages) & 1, &bars->err, 86);
      return !__any_sync(0xFFFFFFFFu, !ok);
    };
    load_next();
    int g = 0, group = 0, before = 0;  // stages of the group before
    bool ok = true;
    for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs) {
      for (int ks = 0; ks < k_stages; ++ks, ++g) {
        if (g >= kStages && !wait_empty(g - kStages)) { ok = false; break; }
        if (ks % kGroup == 0) {
          now = next;
          // the set's last group is the one two before
          if (group >= 2 && !wait_empty(g - before - 1)) { ok = false; break; }
          const uint32_t w0 = word_of(now.w0), w1 = word_of(now.w1);
          const uint32_t at = smem_u32(sS) + (group & 1) * kSetBytes + lane * 16;
          sts128(at, now.x[0], now.x[1], now.x[2], now.x[3]);
          sts128(at + kScaleBytes, w0, w0, w0, w0);
          sts128(at + 2 * kScaleBytes, w1, w1, w1, w1);
          fence_proxy_async_smem();
          __syncwarp();
          ++group;
          before = min(kGroup, k_stages - ks);
        }
        // A release of all memory at cluster scope would take a microsecond: only shared memory is published, and
        // before the next loads are issued, which it would wait for.
        if (lane == 0) {
          if (ks % kGroup == 0) mbar_arrive_cluster_publish_smem(lead_full0 + (g % kStages) * 8);
          else mbar_arrive_cluster_relaxed(lead_full0 + (g % kStages) * 8);
        }
        if (ks % kGroup == 0) load_next();
      }
    }
  } else if (warp == kWarpMma) {
    if (rank == 0 && lane == 0) {
      constexpr uint32_t idesc = idesc_mx(kTile, kTile, false, LAYOUT == CONVROT_LAYOUT_KN);
      const uint32_t a_base = smem_u32(sA), b_base = smem_u32(sB), s_base = smem_u32(sS);
      int g = 0, local = 0, group = 0;
      bool ok = true;
      for (int tile = pair_id; tile < num_tiles && ok; tile += num_pairs, ++local) {
        const int buf = local & 1;
        if (!wait(&bars->acc_empty[buf], ((local >> 1) & 1) ^ 1, &bars->err, 82)) break;
        if (local > 0 && !wait(&bars->shared_empty, (local - 1) & 1, &bars->err, 82)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (buf ? kSecond : 0);
        for (int ks = 0; ks < k_stages; ++ks, ++g) {
          const int slot = g % kStages;
          const uint32_t a_scale = tmem_base + kScaleCol + (group & 1) * 16, b_scale = a_scale + 4;
          if (!wait(&bars->full[slot], (g / kStages) & 1, &bars->err, 83)) { ok = false; break; }
          tc_fence_after();
          if (ks % kGroup == 0) {
            const uint32_t from = s_base + (group & 1) * kSetBytes;
            copy_scales_pair(a_scale, from);
            copy_scales_pair(b_scale, from + kScaleBytes);
            copy_scales_pair(b_scale + 4, from + 2 * kScaleBytes);
          }
          const uint32_t a_addr = a_base + slot * kOpBytes, b_addr = b_base + slot * kOpBytes;
          const uint32_t id = idesc_byte(idesc, ks % kGroup);
#pragma unroll
          for (int j = 0; j < kBK / 32; ++j) {  // K beyond the end is zero in both operands
            const uint64_t adesc = smem_desc(a_addr + j * 32, 16, 1024, 2);
            const uint64_t bdesc = LAYOUT == CONVROT_LAYOUT_NK ? smem_desc(b_addr + j * 32, 16, 1024, 2)
                                                               : smem_desc(b_addr + j * 4096, kOpBytes, 1024, 2);
            mma_mx_pair(d_tmem, adesc, bdesc, id, a_scale, b_scale, (ks | j) != 0 ? 1u : 0u);
          }
          mma_commit_pair_multicast(&bars->empty[slot], 0x3);
          if (ks % kGroup == kGroup - 1 || ks == k_stages - 1) ++group;
        }
        if (!ok) break;
        mma_commit_pair_multicast(&bars->acc_full[buf], 0x3);
      }
      // every MMA issued above finishes before the pair's TMEM is released
      mma_commit_pair_multicast(&bars->mma_done, 0x1);
      wait(&bars->mma_done, 0, &bars->err, 87);
    }
  } else if (warp >= kWarpE0) {
    const int ew = warp - kWarpE0, quarter = warp & 3, half = ew >> 2;
    float* sbias = vecs + ew * 128;
    const uint32_t lead_empty0 = mapa_shared(&bars->acc_empty[0], 0), lead_shared = mapa_shared(&bars->shared_empty, 0);
    int local = 0;
    for (int tile = pair_id; tile < num_tiles; tile += num_pairs, ++local) {
      const int buf = local & 1;
      int m_blk, n_blk;
      place(tile, m_blk, n_blk);
      const int row0 = m_blk * kTile + 128 * rank + quarter * 32, col0 = n_blk * kTile + 128 * half;
      __syncwarp();  // the previous tile's reads of the bias are done
      for (int j = lane; j < 128; j += 32) sbias[j] = col0 + j < p.n && p.bias ? ld_f32(p.bias + col0 + j) : 0.0f;
      __syncwarp();
      if (!wait(&bars->acc_full[buf], (local >> 1) & 1, &bars->err, 85)) break;
      tc_fence_after();
      const uint32_t t_row =
          tmem_base + ((static_cast<uint32_t>(quarter) * 32u) << 16) + (buf ? kSecond : 0) + 128 * half;
      // the columns that both accumulators have: the last 32 of the first, the first 32 of the second
      const bool shared = half != buf;
      for (int i = 0; i < 4; ++i) {
        const int c = shared && !buf ? (i + 3) & 3 : i;
        const bool in = col0 + 32 * c < p.n;  // uniform across the warp
        uint32_t r[32];
        if (in) {
          __syncwarp();
          tmem_ld_32x32b_x32(t_row + c * 32, r);
          tmem_ld_wait();
        }
        if (shared && i == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_publish_smem(lead_shared);
        }
        if (!in) continue;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 b4 = *reinterpret_cast<const float4*>(sbias + c * 32 + j);
          const float bv[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) v[j + u] = __fadd_rn(__uint_as_float(r[j + u]), bv[u]);
        }
        if constexpr (sizeof(TOut) == 4) {
          if (p.add && row0 + lane < p.m) {
            const float* held = static_cast<const float*>(p.out) + static_cast<int64_t>(row0 + lane) * p.n + col0 + c * 32;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (col0 + c * 32 + j < p.n) v[j] = __fadd_rn(held[j], v[j]);
          }
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
// Swap kernel.  One tile of 128 channels (the MMA's M side) x BT tokens and one
// share of K for each CTA; a cluster of CTAs covers K.
//   warp 0  weight producer (lane s issues slot s), warp 1 MMA issuer and
//   TMEM owner, warp 2 activation producer, warp 3 scales; then all four warps
//   run the epilogue: lane l of warp w holds channel 32 w + l, so a store
//   instruction writes 32 consecutive channels of one token.
// With K split, each CTA leaves its sums in shared memory and adds up its share
// of the tokens from all of the cluster's, in the order of the ranks.
// Two sets of scales, in shared and in tensor memory: the scales of a group are
// written once the MMAs of the group two before it are complete, which a commit
// says (sf_empty).  100 x 5120 x 5120 in 17 us (4.1 at a copy's bandwidth): a
// stage takes a CTA about 0.5 us, the latency of its ring, and the first scales'
// way through shared memory about 1 us before the first MMA.
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
  uint64_t sf_full[2];
  uint64_t sf_empty[2];
  uint64_t mma_done;
  uint32_t tmem_base;
  int err;
};

// two CTAs for each SM
template <int BT> constexpr int kStages = BT <= 32 ? 5 : (BT == 64 ? 4 : 3);
template <int BT> constexpr int kXBytes = BT * kBK;
template <int BT> constexpr int kTmemCols = BT == 16 ? 32 : (BT == 32 ? 64 : (BT == 64 ? 128 : 256));
template <int BT>
constexpr size_t kSmem = 1024 + kStages<BT> * (kWBytes + kXBytes<BT>) + 4 * kScaleBytes + sizeof(Bars);
static_assert(kSmem<128> <= 113 * 1024 && kSmem<64> <= 113 * 1024 && kSmem<32> <= 113 * 1024, "shared memory budget");

// The sums of R ranks (token, 128 channels) for tokens c_lo to c_hi, every
// fourth of them a warp's, a lane with four channels; tokens past the last are
// read, in bounds, and not handed on.  16 reads of a thread are in flight: the
// latency between SMs is what this takes.
template <int R, int BT, typename Emit>
__device__ __forceinline__ void join(const float* part, int c_lo, int c_hi, Emit&& emit) {
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
      float sum[4] = {};
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t w[4] = {v[t][r].x, v[t][r].y, v[t][r].z, v[t][r].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = __fadd_rn(sum[i], __uint_as_float(w[i]));
      }
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
  uint8_t* sS = sX + S * kXBytes<BT>;  // scales of the weight, then of the tokens, for each of two groups
  Bars* bars = reinterpret_cast<Bars*>(sS + 4 * kScaleBytes);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int ranks = gridDim.x, rank = blockIdx.x;  // the cluster spans the grid's x
  const int n0 = blockIdx.y * 128, m0 = blockIdx.z * BT;
  const int k_stages = (p.k + kBK - 1) / kBK;
  const int k_lo = static_cast<int>(static_cast<int64_t>(k_stages) * rank / ranks);
  const int k_hi = static_cast<int>(static_cast<int64_t>(k_stages) * (rank + 1) / ranks);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&bars->w_full[s], 1);
      mbar_init(&bars->x_full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bars->sf_full[s], 1);
      mbar_init(&bars->sf_empty[s], 1);
    }
    mbar_init(&bars->mma_done, 1);
    bars->err = 0;
    fence_mbar_init();
    prefetch_tensormap(&tmap_x);
    prefetch_tensormap(&tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, kTmemCols<BT>);
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
        if (!wait(&bars->empty[lane], ((g / S) & 1) ^ 1, &bars->err, 91)) { ok = false; break; }
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
  } else if (warp == 3) {
    constexpr int kRows = (BT + 31) / 32;  // of a lane
    struct {
      uint32_t x[4], w;
    } now, next = {{kOneWord, kOneWord, kOneWord, kOneWord}, 0};
    auto load_next = [&](int b0) {
      if (b0 >= k_hi) return;
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        if (m0 + lane + 32 * j < p.m) next.x[j] = scale_word(p.xscales + (m0 + lane + 32 * j) * p.xs_stride, b0, k_stages);
      next.w = weight_byte(p, n0 / 128, b0, k_stages);
    };
    load_next(k_lo);
    for (int b0 = k_lo, i = 0; b0 < k_hi; b0 += kGroup, ++i) {
      now = next;
      const bool ok = wait(&bars->sf_empty[i & 1], ((i >> 1) & 1) ^ 1, &bars->err, 95);
      if (__any_sync(0xFFFFFFFFu, !ok)) break;
      const uint32_t at = smem_u32(sS) + (i & 1) * 2 * kScaleBytes + lane * 16;
      const uint32_t w = word_of(now.w);
      sts128(at, w, w, w, w);
      sts128(at + kScaleBytes, now.x[0], now.x[1], now.x[2], now.x[3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->sf_full[i & 1]);
      load_next(b0 + kGroup);  // behind the fence, which would wait for it
    }
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t idesc = idesc_mx(128, BT, LAYOUT == CONVROT_LAYOUT_KN, false);
    const uint32_t w_base = smem_u32(sW), x_base = smem_u32(sX), s_base = smem_u32(sS);
    const uint32_t t_scales = tmem_base + BT;  // 8 columns for each of two groups
    for (int kb = k_lo; kb < k_hi; ++kb) {
      const int g = kb - k_lo, slot = g % S, set = (g / kGroup) & 1;
      const uint32_t w_scale = t_scales + set * 8, x_scale = w_scale + 4;
      if (g % kGroup == 0) {
        if (!wait(&bars->sf_full[set], (g / (2 * kGroup)) & 1, &bars->err, 96)) break;
        tc_fence_after();
        copy_scales(w_scale, s_base + set * 2 * kScaleBytes);
        copy_scales(x_scale, s_base + (set * 2 + 1) * kScaleBytes);
      }
      if (!wait(&bars->w_full[slot], (g / S) & 1, &bars->err, 92)) break;
      if (!wait(&bars->x_full[slot], (g / S) & 1, &bars->err, 93)) break;
      tc_fence_after();
      const uint32_t id = idesc_byte(idesc, g % kGroup);
#pragma unroll
      for (int j = 0; j < kBK / 32; ++j) {
        const uint32_t w_addr = w_base + slot * kWBytes;
        const uint64_t wdesc = LAYOUT == CONVROT_LAYOUT_NK ? smem_desc(w_addr + j * 32, 16, 1024, 2)
                                                           : smem_desc(w_addr + j * 4096, kWBytes, 1024, 2);
        const uint64_t xdesc = smem_desc(x_base + slot * kXBytes<BT> + j * 32, 16, 1024, 2);
        mma_mx(tmem_base, wdesc, xdesc, id, w_scale, x_scale, (g | j) != 0 ? 1u : 0u);
      }
      mma_commit(&bars->empty[slot]);
      if (g % kGroup == kGroup - 1) mma_commit(&bars->sf_empty[set]);
    }
    mma_commit(&bars->mma_done);
  }
  __syncwarp();
  __syncthreads();
  const bool done = wait(&bars->mma_done, 0, &bars->err, 94);
  tc_fence_after();

  TOut* out = static_cast<TOut*>(p.out);
  const uint32_t t_row = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
  const int rows = p.m - m0 < BT ? p.m - m0 : BT;
  if (ranks == 1) {
    const int n = n0 + warp * 32 + lane;
    const bool n_ok = n < p.n;
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
      for (int i = 0; i < 16; ++i) v[i] = __fadd_rn(__uint_as_float(r[i]), b);
      TOut* dst = out + static_cast<int64_t>(m0 + c) * p.n + n;
      if constexpr (sizeof(TOut) == 4) {
        if (p.add) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i < rows - c && n_ok) v[i] = __fadd_rn(dst[static_cast<int64_t>(i) * p.n], v[i]);
        }
      }
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
    float b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = n + i < p.n && p.bias ? ld_f32(p.bias + n + i) : 0.0f;
    const bool whole = p.n % 4 == 0;  // four channels in one store
    // sums (token, channel) over the ring, whose copies have all been consumed
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
    auto emit = [&](const float (&sum)[4], int c) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __fadd_rn(sum[i], b[i]);
      TOut* dst = out + static_cast<int64_t>(m0 + c) * p.n + n;
      if constexpr (sizeof(TOut) == 4) {
        if (p.add) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n + i < p.n) v[i] = __fadd_rn(dst[i], v[i]);
        }
      }
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
    const float* sums = reinterpret_cast<const float*>(part);
    if (ranks == 2) join<2, BT>(sums, c_lo, c_hi, emit);
    else if (ranks == 4) join<4, BT>(sums, c_lo, c_hi, emit);
    else join<8, BT>(sums, c_lo, c_hi, emit);
    __syncwarp();
    cluster_sync();  // no CTA leaves while another may still read its sums
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem_base, kTmemCols<BT>);
  }
  if (threadIdx.x == 0 && bars->err) atomicCAS(p.err_word, 0, bars->err);
}

}  // namespace swap

// ===========================================================================
// GEMV kernel, up to 8 tokens of the forward product.  A CTA has 16 channels;
// its 8 warps share out the blocks of 128 of K.  Thread (g, t) of a warp reads
// 16 bytes of channels g and g + 8 at k = 16 t of each half of a block; as f16
// pairs (a conversion each, exact) pairs 2 j and 2 j + 1 of both are the A
// fragment of MMA j (m16n8k16).  Which k a fragment index stands for only has to
// agree with the B fragment, which are the same pairs of token g's codes.  So
// weights go from memory to the MMA with no rearrangement; two sets of two
// blocks are in flight in registers, also from one set of channels to the next.
// A block's products are summed from 0 and added to the total with its two
// scales.  The tokens are in shared memory as f16, converted from their codes
// or (FUSED, one or two tokens) quantized there by every CTA itself, which costs
// less than a kernel of its own before this one.  A launch of a few microseconds
// waits for its instructions as much as for its data: the loop has each piece
// of code once (1 x 5120 x 5120 10.6 us; 15.0 with e4m3 MMAs, which this GPU
// takes apart into conversions and f16 MMAs, and the loop's ends unrolled).  Two
// CTAs an SM take 5120 channels in two rounds, 4736 in one (8.4 us); 1 x 4096 x
// 4096 6.4, 8 x 5120 x 13824 20.5.
// ===========================================================================
namespace gemv {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kChannels = 16;
constexpr int kAhead = 2;  // blocks of a register set
constexpr int kMaxTokens = 8;
constexpr int kMaxFused = 2;
constexpr int kMaxBytes = 96 * 1024;  // of shared memory for the tokens and their scales

struct GemvParams {
  Params p;
  const void* x;  // FUSED: the activation, x_stride elements a row
  const uint8_t* act;
  const uint8_t* weight;
  int64_t x_stride, act_stride, weight_stride;
};

__host__ __device__ constexpr int blocks_of(int k) { return (k + kBK - 1) / kBK; }
// Bytes of a token: 16 off a multiple of 128, so that the 32 bytes of eight
// tokens' quads fall on different banks.  Then come the scales, a float32 a
// token and block.
__host__ __device__ constexpr int pitch_of(int k) { return 2 * blocks_of(k) * kBK + 16; }
__host__ __device__ constexpr int smem_of(int m, int k) { return m * (pitch_of(k) + 4 * blocks_of(k)); }

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four codes as two pairs of f16.
__device__ __forceinline__ uint2 halves_of(uint32_t w) {
  uint2 r;
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(r.x), "=r"(r.y)
      : "r"(w));
  return r;
}

// 16 bytes of a row of codes with those past `count` cleared (rows are on a
// pitch of whole 16 bytes, and all of them can be read).
__device__ __forceinline__ uint4 only(uint4 v, int count) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int keep = min(max(count - 4 * i, 0), 4);
    w[i] &= static_cast<uint32_t>((1ull << (8 * keep)) - 1);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void store_halves(uint8_t* to, uint4 codes) {
  const uint2 a = halves_of(codes.x), b = halves_of(codes.y), c = halves_of(codes.z), d = halves_of(codes.w);
  reinterpret_cast<uint4*>(to)[0] = make_uint4(a.x, a.y, b.x, b.y);
  reinterpret_cast<uint4*>(to)[1] = make_uint4(c.x, c.y, d.x, d.y);
}

// The value of a scale's byte: 2^(byte - 127), NaN for 255.
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7FC00000u : byte == 0u ? 0x00400000u : byte << 23);
}

// Of two scales; NaN where one is.
__device__ __forceinline__ float lesser(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float greater(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename TOut, bool FUSED>
__global__ void __launch_bounds__(kThreads, 2) gemv_kernel(const GemvParams q) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ float part[2][kWarps][kMaxTokens][kChannels + 1];
  const Params& p = q.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int pitch = pitch_of(p.k), k_blocks = blocks_of(p.k);
  uint8_t* tokens = smem_raw;
  float* xs = reinterpret_cast<float*>(smem_raw + p.m * pitch);  // of token m and block b at m * k_blocks + b
  const int b_lo = k_blocks * warp / kWarps, b_hi = k_blocks * (warp + 1) / kWarps;
  const int sets = (p.n + kChannels - 1) / kChannels;  // of channels

  if (!p.early_weights) grid_dependency_wait();
  struct Set {
    uint4 w[2][2][kAhead];  // half of the block, channel g or g + 8
    uint32_t scale[kAhead];
  } ring[2];
  // The blocks of this warp in its order, two register sets of kAhead a round:
  // from `at_b` on of channel set `at_n`; past its last block comes the next
  // channel set.
  int at_n = blockIdx.x, at_b = b_lo;
  float acc[4];
  bool first = true;  // nothing has been fetched yet
  int turn = 0, set = blockIdx.x;
#pragma unroll 1
  while (set < sets) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = 0.0f;
    int b = b_lo;
#pragma unroll 1
    do {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        Set& s = ring[r];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int block = b + r * kAhead + i;
          if (first || block >= b_hi) break;  // uniform across the warp
          float sum[4] = {};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k0 = block * kBK + 64 * h + 16 * t;
            uint4 w0 = s.w[h][0][i], w1 = s.w[h][1][i];
            if (k0 + 16 > p.k) w0 = only(w0, p.k - k0), w1 = only(w1, p.k - k0);
            uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
            if (g < p.m) {
              const uint4* x = reinterpret_cast<const uint4*>(tokens + g * pitch + 2 * k0);
              x0 = x[0], x1 = x[1];
            }
            const uint32_t wa[4] = {w0.x, w0.y, w0.z, w0.w}, wb[4] = {w1.x, w1.y, w1.z, w1.w};
            const uint32_t xw[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint2 c = halves_of(wa[j]), d = halves_of(wb[j]);
              mma_f16_16816(sum, c.x, d.x, c.y, d.y, xw[2 * j], xw[2 * j + 1]);
            }
          }
          // fragment C: rows g and g + 8 (channels), columns 2 t and 2 t + 1 (tokens)
          const float ws = scale_of(s.scale[i]);
          const float x0 = 2 * t < p.m ? xs[2 * t * k_blocks + block] : 0.0f;
          const float x1 = 2 * t + 1 < p.m ? xs[(2 * t + 1) * k_blocks + block] : 0.0f;
          // The smaller scale first: a sum of codes, a multiple of 2^-18 below 2^25,
          // times it is exact however small it is, and too large only where the
          // result is.
          const float lo[2] = {lesser(ws, x0), lesser(ws, x1)}, hi[2] = {greater(ws, x0), greater(ws, x1)};
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = __fmaf_rn(__fmul_rn(sum[j], lo[j & 1]), hi[j & 1], acc[j]);
        }
        const int n0 = at_n * kChannels;
        // channels past the last are read as the last, and not written
        const uint8_t* row0 = q.weight + min(n0 + g, p.n - 1) * q.weight_stride + 16 * t;
        const uint8_t* row1 = q.weight + min(n0 + g + 8, p.n - 1) * q.weight_stride + 16 * t;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int block = at_b + r * kAhead + i;
          const bool live = at_n < sets && block < b_hi;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k0 = block * kBK + 64 * h;
            const bool in = live && k0 + 16 * t < p.k;
            s.w[h][0][i] = in ? ld_128(row0 + k0) : make_uint4(0, 0, 0, 0);
            s.w[h][1][i] = in ? ld_128(row1 + k0) : make_uint4(0, 0, 0, 0);
          }
          s.scale[i] = live ? ld_8(p.wscales + n0 / 128 * p.ws_n + block * p.ws_k) : 0u;
        }
      }
      b += 2 * kAhead;
      at_b += 2 * kAhead;
      if (at_b >= b_hi) {
        at_b = b_lo;
        at_n += gridDim.x;
      }
    } while (!first && b < b_hi);
    if (first) {
      first = false;
      if (p.early_weights) grid_dependency_wait();
      grid_dependents_launch();
      if constexpr (FUSED) {
        // every CTA quantizes the tokens for itself
        const int chunks = k_blocks * kSpanThreads, all = p.m * chunks;
#pragma unroll 1
        for (int i0 = 0; i0 < all; i0 += kThreads) {
          const int i = i0 + threadIdx.x, m = i / chunks, c = (i - m * chunks) * kChunk;
          Pack<TOut, kChunk> w;
          load_pieces(static_cast<const TOut*>(q.x) + m * q.x_stride, c, i < all ? p.k : 0, w);
          const uint32_t byte = scale_byte(span_max(w.top()));
          if (i < all) {
            P2 v[kChunk / 2];
            w.get_lanes(v);
            store_halves(tokens + m * pitch + 2 * c, codes_of(v, byte));
            if (c % kSpan == 0) xs[m * k_blocks + c / kSpan] = scale_of(byte);
          }
        }
      } else {
        const int chunks = k_blocks * (kBK / 16), all = p.m * chunks;
        for (int i = threadIdx.x; i < all; i += kThreads) {
          const int m = i / chunks, k0 = (i - m * chunks) * 16;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (k0 < p.k) v = ld_128(q.act + m * q.act_stride + k0);
          store_halves(tokens + m * pitch + 2 * k0, k0 + 16 > p.k ? only(v, p.k - k0) : v);
        }
        for (int i = threadIdx.x; i < p.m * k_blocks; i += kThreads) {
          const int m = i / k_blocks;
          xs[i] = scale_of(ld_8(p.xscales + m * p.xs_stride + (i - m * k_blocks)));
        }
      }
      __syncthreads();
      continue;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) part[turn][warp][2 * t + (i & 1)][g + 8 * (i >> 1)] = acc[i];
    __syncthreads();
    const int m = threadIdx.x / kChannels, n = set * kChannels + threadIdx.x % kChannels;
    if (m < p.m && n < p.n) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v = __fadd_rn(v, part[turn][w][m][threadIdx.x % kChannels]);
      if (p.bias) v = __fadd_rn(v, ld_f32(p.bias + n));
      TOut* dst = static_cast<TOut*>(p.out) + static_cast<int64_t>(m) * p.n + n;
      if constexpr (sizeof(TOut) == 4) {
        if (p.add) v = __fadd_rn(*dst, v);
      }
      *dst = cvt_out<TOut>(v);
    }
    set += gridDim.x;
    turn ^= 1;
  }
}

}  // namespace gemv

// ---------------------------------------------------------------------------
// host side

namespace {

struct Operands {
  const uint8_t* act;
  const uint8_t* weight;
  int64_t act_stride, weight_stride;
};

int tile_map(CUtensorMap* map, const uint8_t* base, int64_t inner, int64_t rows, int64_t stride, int box_rows) {
  return tmap(map, reinterpret_cast<const int8_t*>(base), inner, rows, stride, box_rows);
}

int weight_map(CUtensorMap* map, const Operands& o, int layout, const Params& p) {
  return layout == CONVROT_LAYOUT_NK ? tile_map(map, o.weight, p.k, p.n, o.weight_stride, 128)
                                     : tile_map(map, o.weight, p.n, p.k, o.weight_stride, 128);
}

template <int LAYOUT, typename TOut>
int launch_pair(const Operands& o, const Params& p, cudaStream_t stream) {
  CUtensorMap map_a, map_b;
  int rc = tile_map(&map_a, o.act, p.k, p.m, o.act_stride, 128);
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
  return check_launch("8-bit float pair gemm");
}

template <int LAYOUT, typename TOut, int BT>
int launch_swap(const Operands& o, const Params& p, int ranks, cudaStream_t stream) {
  CUtensorMap map_x, map_w;
  int rc = tile_map(&map_x, o.act, p.k, p.m, o.act_stride, BT);
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
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see grid_dependency_wait
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, map_x, map_w, p));
  return check_launch("8-bit float swap gemm");
}

template <typename TOut, bool FUSED>
int launch_gemv(const gemv::GemvParams& q, cudaStream_t stream) {
  auto kernel = gemv::gemv_kernel<TOut, FUSED>;
  CONVROT_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, gemv::kMaxBytes));
  cudaLaunchConfig_t cfg = {};
  const int sets = (q.p.n + gemv::kChannels - 1) / gemv::kChannels, most = 2 * device_sm_count();
  cfg.gridDim = dim3(static_cast<unsigned>(sets < most ? sets : most), 1, 1);
  cfg.blockDim = dim3(gemv::kThreads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(gemv::smem_of(q.p.m, q.p.k));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CONVROT_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, q));
  return check_launch("8-bit float gemv");
}

bool gemv_takes(int layout, int64_t m, int64_t k) {
  return layout == CONVROT_LAYOUT_NK && m <= gemv::kMaxTokens &&
         m * (2 * k + 2 * kBK + 16 + 4 * (k / kBK + 1)) <= gemv::kMaxBytes;  // no less than smem_of
}

// x quantized inside the product, which waits for the previous kernel of the
// stream before it reads anything.
template <typename T>
int launch_fused(const void* x, int64_t x_stride, const Operands& o, const Params& p, cudaStream_t s) {
  return launch_gemv<T, true>({p, x, nullptr, o.weight, x_stride, 0, o.weight_stride}, s);
}

// Expected times of the two tile kernels in microseconds, as the 8-bit integer
// product's model has them: stages of 128 K, waves of tiles, the exchange of a
// split K.  Over 161 sizes of 12 to 2000 tokens, 640 to 13824 channels and K from
// 256 to 13824 its choices take 0.9% longer than the best of the pair kernel and
// all splits, 9% at most.  Measured on either side (tokens, K, channels; weights
// from HBM): 100 x 2203 x 13824 swap 17.1, pair 15.7; 200 x 1280 x 2560 swap 10.6,
// pair 10.4; 451 x 5120 x 640 swap 14.8, pair 23.1; 451 x 13824 x 13824 swap 144,
// pair 105.
double pair_time(const Params& p, int sms) {
  const int64_t tiles = static_cast<int64_t>((p.m + 255) / 256) * ((p.n + 255) / 256), pairs = sms / 2;
  const int64_t waves = (tiles + pairs - 1) / pairs, stages = (p.k + kBK - 1) / kBK;
  return 6.0 + static_cast<double>(waves * stages) * (waves > 1 ? 0.45 : 0.36);
}

// The best split of K over 1, 2, 4 or 8 CTAs, and its time.
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
int launch_range(const Operands& o, const Params& p, cudaStream_t s) {
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

template <int LAYOUT, typename TOut>
int launch(const Operands& o, const Params& p, cudaStream_t s) {
  // the GEMV sums each block from 0, whatever K
  if (sizeof(TOut) < 4 || p.k <= kMaxSum || gemv_takes(LAYOUT, p.m, p.k)) return launch_range<LAYOUT, TOut>(o, p, s);
  for (int at = 0; at < p.k; at += kMaxSum) {
    Operands part = o;
    part.act += at;
    part.weight += LAYOUT == CONVROT_LAYOUT_NK ? at : at * o.weight_stride;
    Params q = p;
    q.xscales += at / kSpan;
    q.wscales += at / kSpan * p.ws_k;
    q.k = std::min(kMaxSum, p.k - at);
    if (at) q.bias = nullptr, q.early_weights = 0, q.add = 1;
    const int rc = launch_range<LAYOUT, TOut>(part, q, s);
    if (rc != CONVROT_OK) return rc;
  }
  return CONVROT_OK;
}

struct Call {
  Operands o;
  int layout;
  const uint8_t *xscales, *wscales;
  int64_t xs_stride, ws_stride;
  const float* bias;
  void* out;
  int out_dtype;
  int64_t m, n, k;
};

int check_call(const Call& c) {
  CONVROT_REQUIRE(c.layout == CONVROT_LAYOUT_NK || c.layout == CONVROT_LAYOUT_KN, CONVROT_ERR_INVALID,
                  "unknown layout %d", c.layout);
  CONVROT_REQUIRE(valid_dtype(c.out_dtype), CONVROT_ERR_INVALID, "unknown output dtype %d", c.out_dtype);
  CONVROT_REQUIRE(c.m >= 0 && c.n > 0 && c.k > 0, CONVROT_ERR_INVALID, "invalid shape m=%lld n=%lld k=%lld",
                  static_cast<long long>(c.m), static_cast<long long>(c.n), static_cast<long long>(c.k));
  CONVROT_REQUIRE(c.m < (1LL << 22) && c.n < (1LL << 22) && c.k < (1LL << 22), CONVROT_ERR_UNSUPPORTED, "shape too large");
  const int64_t k_blocks = (c.k + kBK - 1) / kBK, n_blocks = (c.n + kBK - 1) / kBK;
  const bool nk = c.layout == CONVROT_LAYOUT_NK;
  CONVROT_REQUIRE(c.o.act_stride >= c.k && c.o.weight_stride >= (nk ? c.k : c.n) && c.o.act_stride % 16 == 0 &&
                      c.o.weight_stride % 16 == 0,
                  CONVROT_ERR_INVALID, "row strides must cover the rows and be multiples of 16 bytes (%lld, %lld)",
                  static_cast<long long>(c.o.act_stride), static_cast<long long>(c.o.weight_stride));
  CONVROT_REQUIRE(c.xs_stride >= (k_blocks + 3) / 4 * 4 && c.xs_stride % 4 == 0 &&
                      c.ws_stride >= (nk ? k_blocks : n_blocks),
                  CONVROT_ERR_INVALID,
                  "strides of scales must cover their rows, those of the activation in multiples of 4 bytes (%lld, %lld)",
                  static_cast<long long>(c.xs_stride), static_cast<long long>(c.ws_stride));
  if (c.m == 0) return CONVROT_OK;
  CONVROT_REQUIRE(c.o.act && c.o.weight && c.xscales && c.wscales && c.out, CONVROT_ERR_INVALID, "null pointer");
  CONVROT_REQUIRE(aligned_to(c.o.act, 16) && aligned_to(c.o.weight, 16) && aligned_to(c.out, 16) &&
                      aligned_to(c.xscales, 4) && aligned_to(c.bias, 4),
                  CONVROT_ERR_INVALID,
                  "activation, weight and output must be 16-byte aligned, the activation's scales and the bias 4-byte aligned");
  return CONVROT_OK;
}

template <typename TOut>
int by_layout(const Call& c, const Params& p, cudaStream_t s) {
  return c.layout == CONVROT_LAYOUT_NK ? launch<CONVROT_LAYOUT_NK, TOut>(c.o, p, s)
                                       : launch<CONVROT_LAYOUT_KN, TOut>(c.o, p, s);
}

Params params_of(const Call& c, int* err_word, bool early_weights) {
  const bool nk = c.layout == CONVROT_LAYOUT_NK;
  return {c.xscales, c.wscales, c.xs_stride, nk ? c.ws_stride : 1, nk ? 1 : c.ws_stride, c.bias, c.out,
          static_cast<int>(c.m), static_cast<int>(c.n), static_cast<int>(c.k), err_word, early_weights ? 1 : 0, 0};
}

int run(const Call& c, bool early_weights, cudaStream_t s) {
  const Params p = params_of(c, device_error_word(), early_weights);
  CONVROT_REQUIRE(p.err_word != nullptr, CONVROT_ERR_CUDA, "device error word unavailable");
  switch (c.out_dtype) {
    case CONVROT_BF16: return by_layout<__nv_bfloat16>(c, p, s);
    case CONVROT_F16: return by_layout<__half>(c, p, s);
    default: return by_layout<float>(c, p, s);
  }
}

}  // namespace
}  // namespace fp8
}  // namespace convrot

extern "C" {

int convrot_fp8_gemm(const uint8_t* act, int64_t act_stride, const uint8_t* xscales, int64_t xscales_stride,
                     const uint8_t* weight, int64_t weight_stride, int layout, const uint8_t* wscales,
                     int64_t wscales_stride, const float* bias, void* out, int out_dtype, int64_t m, int64_t n,
                     int64_t k, void* stream) {
  using namespace convrot;
  const fp8::Call c{{act, weight, act_stride, weight_stride}, layout, xscales, wscales, xscales_stride, wscales_stride,
                    bias, out, out_dtype, m, n, k};
  const int rc = fp8::check_call(c);
  if (rc != CONVROT_OK || m == 0) return rc;
  return fp8::run(c, /*early_weights=*/false, static_cast<cudaStream_t>(stream));
}

int convrot_fp8_linear(const void* x, int x_dtype, int64_t x_stride, const uint8_t* weight, int64_t weight_stride,
                       int layout, const uint8_t* wscales, int64_t wscales_stride, const float* bias, void* out,
                       int out_dtype, int64_t m, int64_t n, int64_t k, uint8_t* codes, int64_t codes_stride,
                       uint8_t* scales, int64_t scales_stride, void* stream) {
  using namespace convrot;
  const fp8::Call c{{codes, weight, codes_stride, weight_stride}, layout, scales, wscales, scales_stride, wscales_stride,
                    bias, out, out_dtype, m, n, k};
  int rc = fp8::check_call(c);
  if (rc != CONVROT_OK) return rc;
  // One or two tokens: quantized inside the product, one kernel instead of two
  // (1 x 5120 x 5120: 10.9 us, 12.0 as two).
  const int64_t x_size = valid_dtype(x_dtype) ? static_cast<int64_t>(dtype_size(x_dtype)) : 1;
  if (m > 0 && m <= fp8::gemv::kMaxFused && x_dtype == out_dtype && fp8::gemv_takes(layout, m, k) && aligned_to(x, 16) &&
      x_stride * x_size % 16 == 0 && k * x_size % 16 == 0) {
    CONVROT_REQUIRE(x != nullptr && x_stride >= k, CONVROT_ERR_INVALID, "null pointer, or a row stride below k");
    const fp8::Params p = fp8::params_of(c, nullptr, false);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (x_dtype) {
      case CONVROT_BF16: return fp8::launch_fused<__nv_bfloat16>(x, x_stride, c.o, p, s);
      case CONVROT_F16: return fp8::launch_fused<__half>(x, x_stride, c.o, p, s);
      default: return fp8::launch_fused<float>(x, x_stride, c.o, p, s);
    }
  }
  rc = convrot_quantize_fp8(x, x_dtype, m, k, x_stride, codes, codes_stride, scales, scales_stride, stream);
  if (rc != CONVROT_OK || m == 0) return rc;
  // The kernel before the product is the quantizer, which writes no weight
  // and lets the product start only once everything before it is complete.
  return fp8::run(c, /*early_weights=*/true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
