// rtd_kv4_wide.cu -- attention over 4-bit pages for prompt chunks, sm_100a: many query rows
// against the same keys, on the tcgen05 tensor cores.
//
// A CTA takes (sequence, kv head, 256 rows; row = token * G + head of the group) as two
// tiles of 128 rows, and walks the keys in tiles of 128:
//   loader      bulk copies of raw pages, two a stage, in page-table order;
//   4 warps     turn the codes into f16 tiles d * c + m in shared memory, once for both row
//               tiles: K [key][dim] and V transposed [dim][key], both K-major in 128-byte
//               swizzled atoms, two buffers each;
//   MMA thread  S = Q K^T (Q, K in shared memory) and O += P V (P in tensor memory);
//   2 x 4 warps softmax, a thread a row, one row tile each: S from tensor memory, P back over
//               the same columns in f16.  While one tile's softmax runs, the tensor cores
//               work on the other's.
// Tensor memory: S0 S1 O0 O1, 128 columns each.
//
// The running maximum moves only when a score passes it by 2^12, so O is rescaled rarely;
// 2^(x - max + 8) stays inside f16, whose 11 bits P, K, V and the queries (scaled by a power
// of two per row) are rounded to.  Values beyond f16's 65504 become infinite.
//
// Bound: per 128 x 128 scores 1024 clocks of tensor cores (at head_dim 128) and as many of
// the exponential unit; two row tiles share the decoding, 2000 warp instructions a key tile.
#include <algorithm>
#include <cstdint>

#include "rtd_kv4.cuh"
#include "rtd_tcgen05.cuh"

namespace rtd {
namespace {

constexpr int kKeys = 128;             // keys of a tile
constexpr int kStageKeys = 2 * kTok;   // keys of a raw stage
constexpr int kRaw = 6;                // raw stages
constexpr int kSoftWarps = 8, kDecodeWarps = 4;
constexpr int kMmaWarp = kSoftWarps + kDecodeWarps, kLoadWarp = kMmaWarp + 1;
constexpr int kWideThreads = 512;  // and two idle warps, for a whole number of warpgroups
// Registers: launched with 128 a thread, 65536 in all; 256 x 176 + 128 x 96 + 128 x 64 are the same.
constexpr int kSoftRegs = 176, kDecodeRegs = 96, kOtherRegs = 64;
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr float kHeadroom = 8.0f, kGrowth = 12.0f;

template <int NG>
struct WidePlan {
  static constexpr int D = 32 * NG, PB = 20 * D;
  static constexpr int kTile = kKeys * D * 2;  // a K or V tile, or 128 queries
  static constexpr int offQ = 0;
  static constexpr int offK = offQ + 2 * kTile;
  static constexpr int offV = offK + 2 * kTile;
  static constexpr int offRaw = offV + 2 * kTile;
  static constexpr int offBar = offRaw + kRaw * 2 * PB;
  static constexpr int kSmem = offBar + 512 + 1024;  // and the alignment of the tiles
};

// 32 accumulator columns of this warp's lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  // the registers pass through the wait, so that no use is scheduled before it
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27])
               :
               : "memory");
  asm volatile("" : "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

// Nibbles 0 and 4 (ODD = false) or 1 and 5 of w as the f16 pair c, exactly.
template <bool ODD>
__device__ __forceinline__ __half2 code_pair(uint32_t w) {
  const __half2 h = as_h2(lop_and_or(w, ODD ? 0x00F000F0u : 0x000F000Fu, 0x64006400u));
  return ODD ? __hfma2(h, __float2half2_rn(0.0625f), __float2half2_rn(-64.0f)) : __hadd2(h, __float2half2_rn(-1024.0f));
}

template <int NG>
__global__ void __launch_bounds__(kWideThreads, 1) kv4_wide_kernel(const Kv4AttnArgs a, int tiles) {
  using P = WidePlan<NG>;
  constexpr int D = P::D, PB = P::PB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sm32 = smem_u32(sm);
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(sm + P::offBar);
  uint64_t* raw_empty = raw_full + kRaw;
  uint64_t* kv_full = raw_empty + kRaw;   // [2]
  uint64_t* kv_empty = kv_full + 2;       // [2]
  uint64_t* s_full = kv_empty + 2;        // [row tile]: S is there, and O of the key tile before
  uint64_t* p_full = s_full + 2;          // [row tile]
  uint64_t* q_full = p_full + 2;
  uint64_t* drained = q_full + 1;
  uint32_t* misc = reinterpret_cast<uint32_t*>(drained + 1);  // tensor-memory base, flags
  volatile uint32_t* abort_flag = misc + 1;

  // ---- the unit: later row tiles see more keys and come first
  const int G = a.n_head / a.n_kv;
  unsigned bid = blockIdx.x;
  const int kvh = (int)(bid % a.n_kv);
  bid /= a.n_kv;
  const int s = (int)(bid % a.S), tile = tiles - 1 - (int)(bid / a.S);
  const int qs = __ldg(a.q_start + s), nq = __ldg(a.q_start + s + 1) - qs;
  int ctx = __ldg(a.ctx_len + s);
  if (qs < 0 || nq < 0 || (int64_t)qs + nq > a.T || nq > a.max_q) return;  // the other kernel tells
  const int rows = nq * G, row0 = tile * 256;
  if (rows < a.wide_rows || row0 >= rows) return;
  if (ctx > a.max_ctx || ctx < 0) ctx = 0;
  auto seen = [&](int row) { return max(0, ctx - nq + row / G + 1); };
  const int least = seen(row0), most = seen(min(row0 + 256, rows) - 1);
  const int nt = (most + kKeys - 1) / kKeys;              // key tiles
  const int pages = (most + kTok - 1) / kTok;
  const int nraw = (pages + 1) / 2;                       // raw stages
  const int qtiles = rows - row0 > 128 ? 2 : 1;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(misc), 512);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < kRaw; ++i) {
      mbar_init(raw_full + i, 1);
      mbar_init(raw_empty + i, 32 * kDecodeWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(kv_full + i, 32 * kDecodeWarps);
      mbar_init(kv_empty + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 128);
    }
    mbar_init(q_full, 128 * qtiles);
    mbar_init(drained, 1);
    misc[1] = 0;  // abort
    misc[2] = 0;  // a block id outside the pool
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = misc[0];

  // Bounded: one that gives up ends the CTA's other waits too.
  auto wait = [&](uint64_t* b, uint32_t parity) -> bool {
    if (mbar_try_wait(b, parity)) return true;
    const uint64_t t0 = global_ns();
    for (;;) {
      if (mbar_try_wait_sleep(b, parity, 20000u)) return true;
      if (*abort_flag) return false;
      if (global_ns() - t0 > kWaitBudgetNs) {
        raise_status(a.status, kDevWaitTimeout);
        *abort_flag = 1;
        return false;
      }
    }
  };

  if (warp >= kMmaWarp) regs_down<kOtherRegs>();
  if (warp == kLoadWarp) {
    // ------------------------------------------------------------ loader
    const int* table = a.table + (int64_t)s * a.max_blocks;
    int i = 0, ids = 0;
    bool ok = true;
    for (; i < nraw && ok; ++i) {
      const int st = i % kRaw;
      if ((i & 15) == 0) {  // block ids of 16 stages, a lane each
        ids = 0;
        bool bad = false;
        if (2 * i + lane < pages) {
          ids = __ldg(table + 2 * i + lane);
          bad = (unsigned)ids >= (unsigned)a.num_blocks;
          if (bad) ids = 0;
        }
        if (__any_sync(0xffffffffu, bad) && lane == 0) {
          raise_status(a.status, kDevCache);
          misc[2] = 1;
        }
      }
      const int b0 = __shfl_sync(0xffffffffu, ids, (2 * i) & 31), b1 = __shfl_sync(0xffffffffu, ids, (2 * i + 1) & 31);
      if (lane == 0 && i >= kRaw) ok = wait(raw_empty + st, (uint32_t)(((i / kRaw) - 1) & 1));
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
      if (!ok) break;
      if (lane == 0) {
        const bool two = 2 * i + 1 < pages;
        mbar_arrive_expect_tx(raw_full + st, two ? 2 * PB : PB);
        uint8_t* dst = sm + P::offRaw + st * 2 * PB;
        bulk_g2s(dst, a.pages + ((int64_t)b0 * a.n_kv + kvh) * PB, PB, raw_full + st);
        if (two) bulk_g2s(dst + PB, a.pages + ((int64_t)b1 * a.n_kv + kvh) * PB, PB, raw_full + st);
      }
    }
    // no copy may still be landing when the CTA exits (an aborted run alone leaves any)
    if (lane == 0 && *abort_flag)
      for (int k = max(0, i - kRaw); k < i; ++k) mbar_wait_ns(raw_full + k % kRaw, (uint32_t)((k / kRaw) & 1), kWaitBudgetNs, a.status);
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ MMA
    if (lane == 0 && nt > 0) {
      const uint32_t idesc_s = idesc_f16(kKeys), idesc_o = idesc_f16(D);
      auto scores = [&](int t, int buf) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (uint32_t)((k / 4) * (128 * 128) + (k % 4) * 32);
          umma_f16(tmem + 128u * t, kmajor_desc(sm32 + P::offQ + t * P::kTile + off),
                   kmajor_desc(sm32 + P::offK + buf * P::kTile + off), idesc_s, k > 0);
        }
      };
      auto output = [&](int t, int buf, bool more) {
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k) {
          const uint32_t off = (uint32_t)((k / 4) * (D * 128) + (k % 4) * 32);
          umma_f16_ts(tmem + 256u + 128u * t, tmem + 128u * t + 8u * k, kmajor_desc(sm32 + P::offV + buf * P::kTile + off), idesc_o,
                      more || k > 0);
        }
      };
      bool ok = wait(q_full, 0) && wait(kv_full, 0);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < qtiles; ++t) {
          scores(t, 0);
          umma_commit(s_full + t);
        }
        for (int j = 0; j < nt && ok; ++j) {
          for (int t = 0; t < qtiles && ok; ++t) {
            ok = wait(p_full + t, (uint32_t)(j & 1));
            if (!ok) break;
            tc_fence_after();
            output(t, j & 1, j > 0);
            if (t == qtiles - 1) umma_commit(kv_empty + (j & 1));  // both tiles are done with these keys
            if (j + 1 < nt) {
              if (t == 0) ok = wait(kv_full + ((j + 1) & 1), (uint32_t)(((j + 1) >> 1) & 1));
              if (!ok) break;
              tc_fence_after();
              scores(t, (j + 1) & 1);  // over P, whose product was issued before
            }
            umma_commit(s_full + t);
          }
        }
      }
      // an aborted run leaves MMAs in flight
      umma_commit(drained);
      mbar_wait_ns(drained, 0, kWaitBudgetNs, a.status);
    }
    __syncwarp();
  } else if (warp >= kMmaWarp) {
    // idle
  } else if (warp >= kSoftWarps) {
    // ------------------------------------------------------------ decode
    regs_down<kDecodeRegs>();
    const int dt = tid - 32 * kSoftWarps, dw = dt >> 5;
    bool ok = true;
    // K: (token, quarter of 8 dims in every group); tokens t and t + 4 share eight lanes, whose
    // stores then fill all banks
    const int kt = 8 * dw + ((lane >> 3) & 3) + 4 * ((lane >> 2) & 1), ki = lane & 3;
    // V: (eight keys, four dims of a group): octets and the parity of n in the low bits, likewise
    const int oct = lane & 3, vn = ((lane >> 2) & 1) | (lane >> 3) << 1, vg = dw;
    for (int j = 0; j < nt && ok; ++j) {
      const int buf = j & 1;
      if (j >= 2) ok = wait(kv_empty + buf, (uint32_t)(((j >> 1) - 1) & 1));
      for (int q = 0; q < kKeys / kStageKeys && ok; ++q) {
        const int i = j * (kKeys / kStageKeys) + q, st = i % kRaw;
        const uint32_t raw = sm32 + P::offRaw + st * 2 * PB;
        const int key = i * kStageKeys;
        if (i < nraw) {
          ok = wait(raw_full + st, (uint32_t)((i / kRaw) & 1));
          if (!ok) break;
        }
        {  // K, [key][dim]; a quarter's dims in the order 0 4 1 5 2 6 3 7, as the queries'
          const int t = kt & 15;
          const uint32_t page = raw + (kt >> 4) * PB;
          const bool there = key + kt < most;
          const int row = q * kStageKeys + kt;
          // A NaN of V that some rows of the tile do not see would reach them as 0 * NaN.  From
          // the first row's position on it goes into the key instead, whose score only the
          // rows that see it take.
          bool poison = false;
          if (key + kStageKeys > least && there && key + kt >= least) {
#pragma unroll
            for (int g = 0; g < NG; ++g) poison |= (lds32(page + 18 * D + (t * NG + g) * 4) & 0x7c00u) == 0x7c00u;
          }
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            __half2 v[4] = {};
            if (there) {
              const uint32_t w = lds32(page + t * (D / 2) + (ki * NG + g) * 4), h = lds32(page + 8 * D + (t * NG + g) * 4);
              const __half2 d = __low2half2(as_h2(h)), m = __high2half2(as_h2(h));
              v[0] = __hfma2(code_pair<false>(w), d, m);
              v[1] = __hfma2(code_pair<true>(w), d, m);
              v[2] = __hfma2(code_pair<false>(w >> 8), d, m);
              v[3] = __hfma2(code_pair<true>(w >> 8), d, m);
              if (poison) v[0] = as_h2(0x7fff7fffu);
            }
            const int k = 32 * g + 8 * ki;
            sts128(sm32 + P::offK + buf * P::kTile + (k >> 6) * (128 * 128) + sw_off(row, k & 63), as_u32(v[0]), as_u32(v[1]),
                   as_u32(v[2]), as_u32(v[3]));
          }
        }
        if (vg < NG) {  // V, [dim][key]
          const uint32_t page = raw + (oct >> 1) * PB + 10 * D;
          const int t0 = 8 * (oct & 1);
          uint32_t w[8], h[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int t = t0 + e;
            uint32_t at;
            if constexpr (NG == 4)
              at = (uint32_t)((((vn * 2 + (vg >> 1)) ^ (8 * ((t >> 1) & 1))) << 2) + (vg & 1) * 2);
            else
              at = (uint32_t)(vn * 4 + (vg & 1) * 2);
            const bool there = key + 8 * oct + e < most;
            w[e] = there ? lds16(page + t * (D / 2) + at) : 0;
            h[e] = there ? lds32(page + 8 * D + (t * NG + vg) * 4) : 0;
          }
          uint32_t out[4][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = w[2 * e] | (w[2 * e + 1] << 16);
            const __half2 d = as_h2(prmt(h[2 * e], h[2 * e + 1], 0x5410u)), m = as_h2(prmt(h[2 * e], h[2 * e + 1], 0x7632u));
            out[0][e] = as_u32(__hfma2(code_pair<false>(x), d, m));
            out[1][e] = as_u32(__hfma2(code_pair<true>(x), d, m));
            out[2][e] = as_u32(__hfma2(code_pair<false>(x >> 8), d, m));
            out[3][e] = as_u32(__hfma2(code_pair<true>(x >> 8), d, m));
          }
          if (key + kStageKeys > least) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (key + 8 * oct + e >= least && (h[e] & 0x7c00u) == 0x7c00u) {
#pragma unroll
                for (int p = 0; p < 4; ++p) out[p][e >> 1] &= (e & 1) ? 0x0000ffffu : 0xffff0000u;
              }
          }
          const int k = q * kStageKeys + 8 * oct;
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const int d = 32 * vg + 4 * vn + p;
            sts128(sm32 + P::offV + buf * P::kTile + (k >> 6) * (D * 128) + sw_off(d, k & 63), out[p][0], out[p][1], out[p][2],
                   out[p][3]);
          }
        }
        if (i < nraw) mbar_arrive(raw_empty + st);
      }
      fence_async_shared();
      mbar_arrive(kv_full + buf);
    }
  } else {
    // ------------------------------------------------------------ softmax, a thread a row
    regs_up<kSoftRegs>();
    const int t = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lanes + 128u * t, to = tmem + lanes + 256u + 128u * t;
    const int row = row0 + 128 * t + r;
    const bool live = row < rows;
    const int limit = live ? seen(row) : 0;
    if (t < qtiles) {
      // The warp's queries, D / 4 lanes a row: scaled by a power of two that brings a row's
      // largest into [2^6, 2^7), to f16, eight dims in the order 0 4 1 5 2 6 3 7.
      constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes;
      const float scale = a.scale * 1.4426950408889634f;
      float rowmul = 1.0f;
#pragma unroll 4
      for (int r0 = 0; r0 < 32; r0 += kAtOnce) {
        const int wr = 32 * (warp & 3) + r0 + lane / kLanes, qrow = row0 + 128 * t + wr, d0 = 4 * (lane % kLanes);
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (qrow < rows) {
          const int64_t at = (int64_t)(qs + qrow / G) * a.ldq + (int64_t)(kvh * G + qrow % G) * D + d0;
          if (a.q_wide)
            *reinterpret_cast<float4*>(x) = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at));
          else
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = load_as_f32(a.q, a.q_dtype, at + e);
        }
        float mx = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] *= scale;
          mx = fmaxf(mx, fabsf(x[e]));
        }
#pragma unroll
        for (int o = 1; o < kLanes; o *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        int k2 = 0;
        if (mx > 0.0f && mx < INFINITY) k2 = max(-90, min(90, 6 - ilogbf(mx)));
        const float up = pow2(k2), down = pow2(-k2);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= up;
        const bool odd = lane & 1;
        const float y0 = __shfl_xor_sync(0xffffffffu, odd ? x[0] : x[2], 1), y1 = __shfl_xor_sync(0xffffffffu, odd ? x[1] : x[3], 1);
        const uint32_t w0 = odd ? pack_f16x2(y0, x[2]) : pack_f16x2(x[0], y0), w1 = odd ? pack_f16x2(y1, x[3]) : pack_f16x2(x[1], y1);
        const int d8 = d0 & ~7;
        asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(sm32 + P::offQ + t * P::kTile + (d8 >> 6) * (128 * 128) +
                                                             sw_off(wr, d8 & 63) + (odd ? 8 : 0)),
                     "r"(w0), "r"(w1)
                     : "memory");
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) {
          const float rm = __shfl_sync(0xffffffffu, down, e * kLanes);
          if (lane == r0 + e) rowmul = rm;
        }
      }
      fence_async_shared();
      mbar_arrive(q_full);

      float M = -1e30f, l = 0.0f;
      bool ok = true;
      for (int j = 0; j < nt; ++j) {
        ok = wait(s_full + t, (uint32_t)(j & 1));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const int key0 = j * kKeys;
        const bool masked = __any_sync(0xffffffffu, key0 + kKeys > limit);
        uint32_t p[64];
        float sum, top;
        for (;;) {
          sum = 0.0f;
          top = -INFINITY;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float x[32];
            tmem_ld32(ts + 32u * c, x);
            if (masked) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (key0 + 32 * c + e >= limit) x[e] = -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              top = fmaxf(top, fmaxf(x[e], x[e + 1]));
              const float p0 = ex2(fmaf(x[e], rowmul, -M)), p1 = ex2(fmaf(x[e + 1], rowmul, -M));
              sum += p0 + p1;
              p[16 * c + e / 2] = pack_f16x2(p0, p1);
            }
          }
          const float at = top * rowmul;
          const bool over = at > M + kGrowth;
          if (!__any_sync(0xffffffffu, over)) break;
          // a new maximum: O and l so far in its terms, and these scores once more
          const float to_m = over ? at - kHeadroom : M, f = ex2(M - to_m);
          M = to_m;
          l *= f;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              float x[32];
              tmem_ld32(to + c, x);
              uint32_t y[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) y[e] = __float_as_uint(x[e] * f);
              tmem_st32(to + c, y);
            }
            tmem_wait_st();
          }
        }
        l += sum;
        tmem_st32(ts, p);
        tmem_st32(ts + 32u, p + 32);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(p_full + t);
      }
      if (ok && nt > 0) {
        ok = wait(s_full + t, (uint32_t)(nt & 1));
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      if (misc[2]) l = NAN;  // a block id outside the pool: no number stands for these rows
      const float f = 1.0f / l;
      const int64_t o = (int64_t)(qs + row / G) * a.ldo + (int64_t)(kvh * G + row % G) * D;
      const bool none = nt == 0 || l == 0.0f;
#pragma unroll 1
      for (int c = 0; c < D && ok; c += 32) {
        float x[32];
        __syncwarp();
        if (nt > 0) tmem_ld32(to + c, x);
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = none ? 0.0f : x[e] * f;
        if (!live) {
        } else if (a.o_wide) {
          uint4 q[4];
          uint32_t* w = reinterpret_cast<uint32_t*>(q);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (a.o_dtype == 1) {
              w[e] = pack_f16x2(x[2 * e], x[2 * e + 1]);
            } else {
              const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
              w[e] = *reinterpret_cast<const uint32_t*>(&b);
            }
          }
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.o) + o + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[e] = q[e];
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) store_from_f32(a.o, a.o_dtype, o + c + e, x[e]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

template <int NG>
cudaError_t wide_launch(const Kv4AttnArgs& a, int64_t ctas, int tiles, cudaStream_t st) {
  static std::atomic<uint64_t> configured{0};
  cudaError_t e = configure_once(kv4_wide_kernel<NG>, WidePlan<NG>::kSmem, configured);
  if (e != cudaSuccess) return e;
  count_launch();
  kv4_wide_kernel<NG><<<(unsigned)ctas, kWideThreads, WidePlan<NG>::kSmem, st>>>(a, tiles);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_wide(const Kv4AttnArgs& a, int head_dim, cudaStream_t st) {
  const int64_t tiles = ((int64_t)a.max_q * (a.n_head / a.n_kv) + 255) / 256, ctas = tiles * a.n_kv * a.S;
  if (ctas > INT32_MAX) return cudaErrorInvalidConfiguration;
  return head_dim == 128 ? wide_launch<4>(a, ctas, (int)tiles, st) : wide_launch<2>(a, ctas, (int)tiles, st);
}

}  // namespace rtd
