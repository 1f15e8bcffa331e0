// What the two 8-bit matrix products (int8_gemm.cu, fp8_gemm.cu) share: bounded
// waits, tiles by TMA, stores of an accumulator's rows.
#pragma once

#include <cudaTypedefs.h>

#include "rows.cuh"

namespace convrot {

namespace w4a4 {
int make_tmap_u8(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                 const uint32_t* box, CUtensorMapSwizzle swizzle, CUtensorMapDataType dtype);
}

namespace tile8 {

constexpr int kBK = 128;  // K bytes of a stage: one 128-byte swizzle row
constexpr uint64_t kTimeoutNs = 4000000000ull;  // a single wait never legitimately takes this long

// Wait for the phase of `bar` with parity `parity`, for at most kTimeoutNs;
// on time-out record `code` in *err and return false.  Cluster-scope acquire:
// barriers of a pair receive arrivals from both CTAs.
static __device__ __noinline__ bool wait(uint64_t* bar, uint32_t parity, int* err, int code) {
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

__device__ __forceinline__ uint4 dsmem_ld128(uint32_t cluster_addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

// 16 bytes of a row at k0 (a multiple of 16), of which the row has `count`;
// beyond the row's end the bytes of its padding are not read.
__device__ __forceinline__ uint4 load16(const int8_t* row, int k0, int count) {
  if (count >= 16) return ld_128(row + k0);
  uint32_t w[4] = {};
  for (int i = 0; i < count; ++i) w[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k0 + i])) << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 32 values of each lane's row, columns col to col + 31 of rows row0 to row0 +
// 31 of a row-major (m, n) output, whatever of them lies in it.  Restaged in
// `space` (kChunkBytes of shared memory of the warp's own) so that a store
// instruction covers 8 rows of 64 contiguous bytes instead of 32 rows of 16:
// 16-byte piece q of row r at ((q + r / 2) % 4), conflict-free both ways.
constexpr int kChunkBytes = 32 * 64;
template <typename TOut>
__device__ __forceinline__ void store_rows(const float (&v)[32], uint8_t* space, TOut* out, int row0, int col, int m,
                                           int n) {
  constexpr int kCols = 64 / sizeof(TOut);  // columns of a restaged chunk
  const int lane = threadIdx.x & 31;
  const uint32_t sb = smem_u32(space);
  const bool vec_store = (static_cast<int64_t>(n) * sizeof(TOut)) % 16 == 0;
#pragma unroll
  for (int part = 0; part < 32 / kCols; ++part, col += kCols) {
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
    if (vec_store) {
      const int q = lane & 3;
      if (col + (q + 1) * (kCols / 4) <= n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rr = i * 8 + (lane >> 2);
          if (row0 + rr < m)
            *reinterpret_cast<uint4*>(out + static_cast<int64_t>(row0 + rr) * n + col + q * (kCols / 4)) =
                lds128(sb + rr * 64 + (((q + (rr >> 1)) & 3) << 4));
        }
      }
    } else {
      // rows off the 16-byte grid: one element a lane, consecutive
      // lanes on consecutive columns, eight rows' reads at a time
      constexpr int kRowsAt = 32 / kCols;
      const int cc = lane % kCols, q = cc / (kCols / 4), e = cc % (kCols / 4);
      TOut* dst = out + static_cast<int64_t>(row0 + lane / kCols) * n + col + cc;
      const int64_t step = static_cast<int64_t>(kRowsAt) * n;
      const bool col_ok = col + cc < n;
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += 8 * kRowsAt) {
        TOut v8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = r0 + i * kRowsAt + lane / kCols;
          v8[i] = reinterpret_cast<const TOut*>(space + rr * 64 + (((q + (rr >> 1)) & 3) << 4))[e];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i, dst += step)
          if (col_ok && row0 + r0 + i * kRowsAt + lane / kCols < m) *dst = v8[i];
      }
    }
  }
}

// A (rows, inner) byte matrix in tiles of 128 bytes x box_rows.
inline int tmap(CUtensorMap* map, const int8_t* base, int64_t inner, int64_t rows, int64_t stride, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(inner), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(stride)};
  const uint32_t box[2] = {128, static_cast<uint32_t>(box_rows)};
  return w4a4::make_tmap_u8(map, base, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_UINT8);
}

}  // namespace tile8
}  // namespace convrot
