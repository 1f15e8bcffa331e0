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
#include <algorithm>

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
};

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

// 512 bytes of scales (32 rows of 16, contiguous) to 4 columns of tensor
// memory, the same for each quarter of its lanes.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t saddr) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(smem_desc(saddr, 16, 128, 0))
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

// The scales of output block `nb` of the weight for K blocks b0 to b0 + 3 as a
// word, in every lane of the warp.
__device__ __forceinline__ uint32_t weight_word(const Params& p, int nb, int b0, int blocks) {
  const int lane = threadIdx.x & 31, b = b0 + (lane & 3);
  const uint32_t v = b < blocks ? ld_8(p.wscales + nb * p.ws_n + b * p.ws_k) : 0x7Fu;
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) word |= __shfl_sync(0xFFFFFFFFu, v, i) << (8 * i);
  return word;
}

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
// says (sf_empty).
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
    for (int b0 = k_lo, i = 0; b0 < k_hi; b0 += kGroup, ++i) {
      const uint32_t w = weight_word(p, n0 / 128, b0, k_stages);
      uint32_t x[4] = {kOneWord, kOneWord, kOneWord, kOneWord};
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        if (m0 + lane + 32 * j < p.m) x[j] = scale_word(p.xscales + (m0 + lane + 32 * j) * p.xs_stride, b0, k_stages);
      const bool ok = wait(&bars->sf_empty[i & 1], ((i >> 1) & 1) ^ 1, &bars->err, 95);
      if (__any_sync(0xFFFFFFFFu, !ok)) break;
      const uint32_t at = smem_u32(sS) + (i & 1) * 2 * kScaleBytes + lane * 16;
      sts128(at, w, w, w, w);
      sts128(at + kScaleBytes, x[0], x[1], x[2], x[3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->sf_full[i & 1]);
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

template <int LAYOUT, typename TOut>
int launch(const Operands& o, const Params& p, cudaStream_t s) {
  const int bt = p.m <= 16 ? 16 : p.m <= 32 ? 32 : p.m <= 64 ? 64 : 128;
  int ranks = 1;
  switch (bt) {
    case 16: return launch_swap<LAYOUT, TOut, 16>(o, p, ranks, s);
    case 32: return launch_swap<LAYOUT, TOut, 32>(o, p, ranks, s);
    case 64: return launch_swap<LAYOUT, TOut, 64>(o, p, ranks, s);
    default: return launch_swap<LAYOUT, TOut, 128>(o, p, ranks, s);
  }
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
  CONVROT_REQUIRE(aligned_to(c.o.act, 16) && aligned_to(c.o.weight, 16) && aligned_to(c.out, 16) && aligned_to(c.xscales, 4),
                  CONVROT_ERR_INVALID,
                  "activation, weight and output must be 16-byte aligned, the activation's scales 4-byte aligned");
  return CONVROT_OK;
}

template <typename TOut>
int by_layout(const Call& c, const Params& p, cudaStream_t s) {
  return c.layout == CONVROT_LAYOUT_NK ? launch<CONVROT_LAYOUT_NK, TOut>(c.o, p, s)
                                       : launch<CONVROT_LAYOUT_KN, TOut>(c.o, p, s);
}

int run(const Call& c, bool early_weights, cudaStream_t s) {
  const bool nk = c.layout == CONVROT_LAYOUT_NK;
  const Params p{c.xscales, c.wscales, c.xs_stride, nk ? c.ws_stride : 1, nk ? 1 : c.ws_stride, c.bias, c.out,
                 static_cast<int>(c.m), static_cast<int>(c.n), static_cast<int>(c.k), device_error_word(),
                 early_weights ? 1 : 0};
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
  rc = convrot_quantize_fp8(x, x_dtype, m, k, x_stride, codes, codes_stride, scales, scales_stride, stream);
  if (rc != CONVROT_OK || m == 0) return rc;
  // The kernel before the product is the quantizer, which writes no weight
  // and lets the product start only once everything before it is complete.
  return fp8::run(c, /*early_weights=*/true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
