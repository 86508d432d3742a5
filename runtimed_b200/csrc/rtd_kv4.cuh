// rtd_kv4.cuh -- the 4-bit pages' layout and what the kernels that read them share.
//
// A page is 16 tokens of one kv head, 20 * D bytes (D = head_dim, NG = D / 32 groups):
//   [0, 8D)     K codes, D / 2 bytes a token     [8D, 10D)   K headers, 4 bytes a group
//   [10D, 18D)  V codes                          [18D, 20D)  V headers
// A header is (f16 step d, f16 minimum m); a code c stands for d * c + m, with
// d = f16((max - min) / 15), m = f16(min) over the 32 dims of the group.  A group with a
// value that is not finite, or whose header overflows f16, is held as d = m = NaN: reading
// it gives NaN, as a 16-bit cache would.
//
// The codes lie in the order the attention's fragments want them:
//   K: word i * NG + g of a token holds dims 32 g + 8 i .. + 7 (i < 4): lane i of a quad
//      reads its words of every group with one load, and a warp's eight tokens are one
//      contiguous, conflict-free span.
//   V: word n holds, in its low and high half, dims 4 n .. 4 n + 3 of two neighbouring
//      groups (n < 8), so that the halves of two tokens' words join into f16 pairs of one
//      dim.  With four groups both pairs' words alternate (one 64-bit load), and tokens
//      with bit 1 set have the words 8 apart exchanged, which spreads a quad's four tokens
//      over all 32 banks.  A last odd group fills half words.
// A token owns whole bytes everywhere, so tokens of one page may be appended by different
// CTAs of one launch.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "rtd_common.cuh"
#include "rtd_kernels.h"

namespace rtd {

constexpr int kTok = 16;  // tokens of a page

// The kernel's shared-memory limit, set once per device (a bit each in `configured`).
template <typename K>
cudaError_t configure_once(K kernel, int smem, std::atomic<uint64_t>& configured) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (e != cudaSuccess || (configured.load(std::memory_order_relaxed) & bit)) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) configured.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

__device__ __forceinline__ float load_as_f32(const void* p, int dt, int64_t i) {
  if (dt == 0) return static_cast<const float*>(p)[i];
  if (dt == 1) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_from_f32(void* p, int dt, int64_t i, float v) {
  if (dt == 0)
    static_cast<float*>(p)[i] = v;
  else if (dt == 1)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ __half2 as_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // |e| <= 126

// A call of rtd_attention_kv4, as its kernels take it.
struct Kv4AttnArgs {
  const void* q;
  int q_dtype;
  int q_wide;  // f32 rows on 16-byte boundaries
  int64_t ldq;
  int T, n_head, n_kv;
  float scale;
  const int* q_start;
  const int* ctx_len;
  int S;
  const int* table;
  int max_blocks, max_q, max_ctx;
  const uint8_t* pages;
  int num_blocks;
  void* o;
  int o_dtype;
  int o_wide;       // rows on 16-byte boundaries
  int64_t ldo;
  int wide_rows;    // sequences with at least so many rows (queries x G) are the wide kernel's,
  int64_t wide_total;  // if all of these have so many (queries x n_head) together
  int* redo;        // [S] raised by the wide kernel: sequences of its that are the line kernel's all the same
  int min_share;    // pages a CTA takes at least
  float* part;      // [CTA][2][8 (D + 2)]: the units begun before it, and left open by it
  unsigned* count;  // [CTA]: arrivals at the unit it leaves open, whole kArrive between calls
  int* status;
};

// A sequence's rows if it is a prompt chunk, else 0; what is wrong with it counts for nothing.
__device__ __forceinline__ int chunk_rows(const Kv4AttnArgs& a, int s) {
  const int qs = __ldg(a.q_start + s), nq = __ldg(a.q_start + s + 1) - qs;
  if (qs < 0 || nq < 0 || (int64_t)qs + nq > a.T || nq > a.max_q) return 0;
  const int rows = nq * (a.n_head / a.n_kv);
  return rows < a.wide_rows ? 0 : rows;
}

// Prompt chunks (rtd_kv4_wide.cu): the sequences of at least a.wide_rows rows, 16-bit outputs,
// head_dim 64 or 128.
cudaError_t launch_kv4_wide(const Kv4AttnArgs& a, int head_dim, cudaStream_t st);

}  // namespace rtd
