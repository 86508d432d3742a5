// rtd_kv4_wide.cu -- attention over 4-bit pages for prompt chunks, sm_100a: many query rows
// against the same keys, on the tcgen05 tensor cores.
//
// A CTA takes (sequence, kv head, 256 rows; row = token * G + head of the group) as two
// tiles of 128 rows, and walks the keys in tiles of 64:
//   loader      bulk copies of raw pages, two a stage, in page-table order;
//   8 warps     turn the codes into f16 tiles d * c + m in shared memory, once for both row
//               tiles: K [key][dim] and V transposed [dim][key], both K-major in 128-byte
//               swizzled atoms, four buffers each;
//   MMA thread  S = Q K^T and O += P V, Q and P in tensor memory: with Q in shared memory an
//               MMA took 109 clocks for 64 of work, since both operands and the decoding
//               shared its bandwidth;
//   2 x 4 warps softmax, a thread a row, one row tile each: S from tensor memory, P back over
//               the same columns in f16.  While one tile's softmax runs, the tensor cores
//               work on the other's.
// Tensor memory: S0 S1 (64 columns each), Q0 Q1 (D / 2), O0 O1 (D).
//
// The running maximum moves only when a row's sum of p = 2^(x - max) over a key tile passes
// 2^15: until then every p is below that, and inside f16.  So the maximum is looked for, and O
// rescaled, rarely, and the exponentials come straight from the scores.  P, K, V and the
// queries (scaled by a power of two per row) are rounded to f16's 11 bits: bf16 outputs are 1.75e-3
// off 64 bits (their own rounding 1.65e-3), f16 ones 6e-4 (2e-4).
//
// Keys or values beyond its 65504 have no place in these tiles, and a NaN of V that only some
// rows of a tile see would reach the others as 0 * NaN.  A decoding thread that meets either
// raises the sequence's word in `redo`, and the line kernel, which follows, writes all its rows.
//
// Bound: per 128 x 64 scores 512 clocks of tensor cores (at head_dim 128) and as many of the
// exponential unit; what they take is the chain S -> softmax -> P -> S of a row tile.  2 sequences
// of 4000 with 512 queries, 64/8 heads of 128, bf16: 106 GFLOP, 63 us at the measured rate, 180 here.
#include <algorithm>
#include <cstdint>

#include "rtd_kv4.cuh"
#include "rtd_tcgen05.cuh"

namespace rtd {
namespace {

constexpr int kKeys = 64;              // keys of a tile
constexpr int kBuf = 4;                // buffers of K and V tiles
constexpr int kStageKeys = 2 * kTok;   // keys of a raw stage
constexpr int kRaw = 12;               // raw stages
constexpr int kSoftWarps = 8, kDecodeWarps = 8;
constexpr int kMmaWarp = kSoftWarps + kDecodeWarps, kLoadWarp = kMmaWarp + 1;
constexpr int kWideThreads = 640;  // and two idle warps, for a whole number of warpgroups
// Registers: launched with 96 a thread, 61440 in all; 256 x 128 + 256 x 80 + 128 x 64 are the same.
constexpr int kSoftRegs = 128, kDecodeRegs = 80, kOtherRegs = 64;
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr float kHeadroom = 8.0f, kMostSum = 32768.0f;  // 64 times 2^8 is below it

template <int NG>
struct WidePlan {
  static constexpr int D = 32 * NG, PB = 20 * D;
  static constexpr int kTile = kKeys * D * 2;  // a K or V tile
  static constexpr int offK = 0;
  static constexpr int offV = offK + kBuf * kTile;
  static constexpr int offRaw = offV + kBuf * kTile;
  static constexpr int offQ = 0;               // the queries on their way to tensor memory: before any K and V
  static constexpr int kQTile = 128 * D * 2;
  static_assert(2 * kQTile <= offRaw, "the queries lie where K and V will");
  static constexpr uint32_t colS = 0, colQ = 2 * kKeys, colO = colQ + D;  // tensor-memory columns
  static constexpr int offBar = offRaw + kRaw * 2 * PB;
  static constexpr int kSmem = offBar + 512 + 1024;  // and the alignment of the tiles
};

// 32 columns of this warp's lanes, to be waited for with tmem_wait_ld: the registers pass
// through the wait, so that no use is scheduled before it.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14])
               :
               : "memory");
  asm volatile("" : "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                    "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]));
  asm volatile("" : "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
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

// D (+)= A[tmem] . B[smem desc]^T, f16 in, f32 out.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}

// Nibbles 0 and 4 (ODD = false) or 1 and 5 of w as the f16 pair c, exactly.
template <bool ODD>
__device__ __forceinline__ __half2 code_pair(uint32_t w) {
  const __half2 h = as_h2(lop_and_or(w, ODD ? 0x00F000F0u : 0x000F000Fu, 0x64006400u));
  return ODD ? __hfma2(h, __float2half2_rn(0.0625f), __float2half2_rn(-64.0f)) : __hadd2(h, __float2half2_rn(-1024.0f));
}

__device__ __forceinline__ float2 fma_f32x2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add_f32x2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

template <int NG>
__global__ void __launch_bounds__(kWideThreads, 1) kv4_wide_kernel(const Kv4AttnArgs a) {
  using P = WidePlan<NG>;
  constexpr int D = P::D, PB = P::PB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sm32 = smem_u32(sm);
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(sm + P::offBar);
  uint64_t* raw_empty = raw_full + kRaw;
  uint64_t* kv_full = raw_empty + kRaw;   // [kBuf]
  uint64_t* kv_empty = kv_full + kBuf;    // [kBuf]
  uint64_t* s_full = kv_empty + kBuf;     // [row tile]: S is there, and O of the key tile before
  uint64_t* p_full = s_full + 2;          // [row tile]
  uint64_t* q_full = p_full + 2;
  uint64_t* drained = q_full + 1;
  uint32_t* misc = reinterpret_cast<uint32_t*>(drained + 1);  // tensor-memory base, flags
  volatile uint32_t* abort_flag = misc + 1;

  // ---- the unit: the row tiles of the chunks in one list (the grid's bound on it counts T, not
  // max_q, since one long chunk among many short sequences is the usual batch); of a sequence's
  // the later ones see more keys and come first
  __shared__ int sums[kWideThreads / 32], unit[2];
  __shared__ int64_t row_sums[kWideThreads / 32];
  const int G = a.n_head / a.n_kv;
  const int kvh = (int)(blockIdx.x % a.n_kv), want = (int)(blockIdx.x / a.n_kv);
  {
    const int per = (a.S + kWideThreads - 1) / kWideThreads;
    const int s0 = min(a.S, (int)threadIdx.x * per), s1 = min(a.S, s0 + per);
    int mine = 0;
    int64_t all = 0;
    for (int s = s0; s < s1; ++s) {
      const int n = chunk_rows(a, s);
      mine += (n + 255) / 256;
      all += n;
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if ((int)(threadIdx.x & 31) >= o) inc += y;
      all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    if ((threadIdx.x & 31) == 31) {
      sums[threadIdx.x >> 5] = inc;
      row_sums[threadIdx.x >> 5] = all;
    }
    if (threadIdx.x == 0) unit[0] = -1;
    __syncthreads();
    all = 0;
    for (int k = 0; k < kWideThreads / 32; ++k) {
      if (k < (int)(threadIdx.x >> 5)) inc += sums[k];
      all += row_sums[k];
    }
    int before = inc - mine;
    if (want >= before && want < inc && all * a.n_kv >= a.wide_total)
      for (int s = s0; s < s1; ++s) {
        const int n = (chunk_rows(a, s) + 255) / 256;
        if (want < before + n) {
          unit[0] = s;
          unit[1] = n - 1 - (want - before);
          break;
        }
        before += n;
      }
    __syncthreads();
  }
  const int s = unit[0], tile = unit[1];
  if (s < 0) return;
  const int qs = __ldg(a.q_start + s), nq = __ldg(a.q_start + s + 1) - qs;
  int ctx = __ldg(a.ctx_len + s);
  const int rows = nq * G, row0 = tile * 256;
  if (ctx > a.max_ctx || ctx < 0) ctx = 0;
  auto seen = [&](int row) { return max(0, ctx - nq + row / G + 1); };
  const int least = seen(row0), most = seen(min(row0 + 256, rows) - 1);
  const int nt = (most + kKeys - 1) / kKeys;              // key tiles
  const int pages = (most + kTok - 1) / kTok;
  const int nraw = (pages + 1) / 2;                       // raw stages
  const int qtiles = rows - row0 > 128 ? 2 : 1;

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(misc), 512);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < kRaw; ++i) {
      mbar_init(raw_full + i, 1);
      mbar_init(raw_empty + i, 16 * kDecodeWarps);
    }
    for (int i = 0; i < kBuf; ++i) {
      mbar_init(kv_full + i, 32 * kDecodeWarps);
      mbar_init(kv_empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
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
    // The whole warp walks the loop and one elected lane issues, so that descriptors stay in
    // uniform registers: issued from a one-lane branch an MMA took 118 clocks.
    if (nt > 0) {
      const uint32_t idesc_s = idesc_f16(kKeys), idesc_o = idesc_f16(D);
      const uint64_t k0 = kmajor_desc(sm32 + P::offK), v0 = kmajor_desc(sm32 + P::offV);
      const bool issuer = elect_one();
      auto scores = [&](int t, int buf) {
        const uint64_t b = k0 + (uint64_t)(buf * (P::kTile >> 4));
        const uint32_t d = tmem + P::colS + kKeys * t, q = tmem + P::colQ + (D / 2) * t;
        if (issuer) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_ts(d, q + 8u * k, b + (uint64_t)((k / 4) * (kKeys * 8) + (k % 4) * 2), idesc_s, k > 0);
          umma_commit(s_full + t);
        }
      };
      auto output = [&](int t, int buf, bool more) {
        const uint64_t b = v0 + (uint64_t)(buf * (P::kTile >> 4));
        const uint32_t d = tmem + P::colO + D * t, p = tmem + P::colS + kKeys * t;
        if (issuer) {
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k) umma_ts(d, p + 8u * k, b + (uint64_t)(2 * k), idesc_o, more || k > 0);
        }
      };
      bool ok = wait(q_full, 0) && wait(kv_full, 0);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < qtiles; ++t) scores(t, 0);
        for (int j = 0; j < nt && ok; ++j) {
          for (int t = 0; t < qtiles && ok; ++t) {
            ok = wait(p_full + t, (uint32_t)(j & 1));
            if (t == 0 && j + 1 < nt && ok) ok = wait(kv_full + (j + 1) % kBuf, (uint32_t)(((j + 1) / kBuf) & 1));
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            output(t, j % kBuf, j > 0);
            if (issuer && t == qtiles - 1) umma_commit(kv_empty + j % kBuf);  // both tiles are done with these keys
            if (j + 1 < nt)
              scores(t, (j + 1) % kBuf);  // over P, whose product was issued before
            else if (issuer)
              umma_commit(s_full + t);  // O is there
          }
        }
      }
      // an aborted run leaves MMAs in flight
      if (issuer) {
        umma_commit(drained);
        mbar_wait_ns(drained, 0, kWaitBudgetNs, a.status);
      }
    }
    __syncwarp();
  } else if (warp >= kMmaWarp) {
    // idle
  } else if (warp >= kSoftWarps) {
    // ------------------------------------------------------------ decode
    regs_down<kDecodeRegs>();
    // Four warps take the even stages, four the odd ones; of four, two turn K and two V.
    const int dw = (warp - kSoftWarps) & 3, odd_stage = (warp - kSoftWarps) >> 2;
    bool ok = nt == 0 || wait(q_full, 0);  // the queries have left
    // the largest code's value, which is infinite where f16 is left (the least is f16 itself)
    const __half2 fifteen = __float2half2_rn(15.0f);
    __half2 largest = __float2half2_rn(0.0f);
    bool redo = false;
    for (int j = 0; j < nt && ok; ++j) {
      const int buf = j % kBuf;
      if (j >= kBuf) ok = wait(kv_empty + buf, (uint32_t)((j / kBuf - 1) & 1));
      for (int q = odd_stage; q < kKeys / kStageKeys && ok; q += 2) {
        const int i = j * (kKeys / kStageKeys) + q, st = i % kRaw;
        const uint32_t raw = sm32 + P::offRaw + st * 2 * PB;
        const int key = i * kStageKeys;
        if (i < nraw) {
          ok = wait(raw_full + st, (uint32_t)((i / kRaw) & 1));
          if (!ok) break;
        }
        if (dw < 2) {
          // K, [key][dim]: a thread has a quarter (8 dims) of every group of two tokens; the
          // dims in the order 0 4 1 5 2 6 3 7, as the queries'.  Tokens t and t + 4 share
          // eight lanes, whose stores then fill all banks.
          const int ki = lane & 3;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int kt = 16 * dw + 8 * half + ((lane >> 3) & 3) + 4 * ((lane >> 2) & 1), t = kt & 15;
            const uint32_t page = raw + (kt >> 4) * PB;
            const bool there = key + kt < most;
            const int row = q * kStageKeys + kt;
            uint32_t w[4] = {}, h[4] = {};
            if (there) {
              const uint32_t at = page + t * (D / 2) + ki * NG * 4, head = page + 8 * D + t * NG * 4;
              if constexpr (NG == 4) {
                *reinterpret_cast<uint4*>(w) = lds128(at);
                *reinterpret_cast<uint4*>(h) = lds128(head);
              } else {
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                  w[g] = lds32(at + 4 * g);
                  h[g] = lds32(head + 4 * g);
                }
              }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const __half2 d = __low2half2(as_h2(h[g])), m = __high2half2(as_h2(h[g]));
              largest = __hmax2(largest, __hfma2(fifteen, d, m));
              const int k = 32 * g + 8 * ki;
              sts128(sm32 + P::offK + buf * P::kTile + (k >> 6) * (kKeys * 128) + sw_off(row, k & 63),
                     as_u32(__hfma2(code_pair<false>(w[g]), d, m)), as_u32(__hfma2(code_pair<true>(w[g]), d, m)), as_u32(__hfma2(code_pair<false>(w[g] >> 8), d, m)),
                     as_u32(__hfma2(code_pair<true>(w[g] >> 8), d, m)));
            }
          }
        } else if (2 * (dw - 2) < NG) {
          // V, [dim][key]: a thread has eight keys (an octet) of four dims in each of two
          // groups.  Octets and the parity of n lie in the low lane bits, so that eight lanes'
          // stores fill all banks; odd octets read the tokens of a pair in turn.
          const int oct = lane & 3, n = ((lane >> 2) & 1) | (lane >> 3) << 1, gp = dw - 2, swap = oct & 1;
          const uint32_t page = raw + (oct >> 1) * PB + 10 * D;
          const uint32_t low = swap ? 0x1054u : 0x5410u, high = swap ? 0x3276u : 0x7632u;
          const int t0 = 8 * (oct & 1);
          // every load before the first store: the compiler cannot tell them apart
          uint32_t w[8], h[8][2];
          const bool whole = key + kStageKeys <= most;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int t = t0 + (e ^ swap);
            uint32_t at;
            if constexpr (NG == 4)
              at = (uint32_t)(((n * 2 + gp) ^ (8 * ((t >> 1) & 1))) << 2);
            else
              at = (uint32_t)(n * 4);
            w[e] = lds32(page + t * (D / 2) + at);
            const uint2 hh = lds64(page + 8 * D + (t * NG + 2 * gp) * 4);
            h[e][0] = hh.x;
            h[e][1] = hh.y;
          }
          if (!whole) {  // past the last key, and what was never loaded
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (key + 16 * (oct >> 1) + t0 + (e ^ swap) >= most) w[e] = h[e][0] = h[e][1] = 0;
          }
          if (key + kStageKeys > least) {  // NaN that some rows do not see
#pragma unroll
            for (int e = 0; e < 8; ++e)
              redo |= key + 16 * (oct >> 1) + t0 + (e ^ swap) >= least &&
                      ((h[e][0] & 0x7c00u) == 0x7c00u || (h[e][1] & 0x7c00u) == 0x7c00u);
          }
          const int k = q * kStageKeys + 8 * oct;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint32_t out[4][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t x = prmt(w[2 * e], w[2 * e + 1], g ? high : low);
              const __half2 d = as_h2(prmt(h[2 * e][g], h[2 * e + 1][g], low)), m = as_h2(prmt(h[2 * e][g], h[2 * e + 1][g], high));
              largest = __hmax2(largest, __hfma2(fifteen, d, m));
              out[0][e] = as_u32(__hfma2(code_pair<false>(x), d, m));
              out[1][e] = as_u32(__hfma2(code_pair<true>(x), d, m));
              out[2][e] = as_u32(__hfma2(code_pair<false>(x >> 8), d, m));
              out[3][e] = as_u32(__hfma2(code_pair<true>(x >> 8), d, m));
            }
#pragma unroll
            for (int p = 0; p < 4; ++p)
              sts128(sm32 + P::offV + buf * P::kTile + sw_off(32 * (2 * gp + g) + 4 * n + p, k), out[p][0], out[p][1], out[p][2],
                     out[p][3]);
          }
        }
        if (i < nraw) mbar_arrive(raw_empty + st);
      }
      fence_async_shared();
      mbar_arrive(kv_full + buf);
    }
    redo |= __hisinf(__low2half(largest)) || __hisinf(__high2half(largest));
    if (redo) a.redo[s] = 1;
  } else {
    // ------------------------------------------------------------ softmax, a thread a row
    regs_up<kSoftRegs>();
    const int t = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lanes + P::colS + kKeys * t, to = tmem + lanes + P::colO + D * t;
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
        // 16-byte chunk c of row r at c ^ (r & 7)
        asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(sm32 + P::offQ + t * P::kQTile + wr * (2 * D) +
                                                             (((d0 >> 3) ^ (wr & 7)) << 4) + (odd ? 8 : 0)),
                     "r"(w0), "r"(w1)
                     : "memory");
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) {
          const float rm = __shfl_sync(0xffffffffu, down, e * kLanes);
          if (lane == r0 + e) rowmul = rm;
        }
      }
      __syncwarp();  // the row that a thread takes is its warp's own
#pragma unroll
      for (int c = 0; c < D / 2; c += 32) {
        uint32_t v[32];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint4*>(v + 4 * e) = lds128(sm32 + P::offQ + t * P::kQTile + r * (2 * D) + (((c / 4 + e) ^ (r & 7)) << 4));
        tmem_st32(tmem + lanes + P::colQ + (D / 2) * t + c, v);
      }
      tmem_wait_st();
      tc_fence_before();
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
        uint32_t p[32];
        float sum;
        for (int again = 0;; ++again) {
          const float2 nm = make_float2(-M, -M), rm = make_float2(rowmul, rowmul);
          float2 acc = make_float2(0.0f, 0.0f);
          uint32_t x[2][32];
          tmem_ld32(ts, x[0]);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t(&v)[32] = x[c & 1];
            tmem_wait_ld(v);
            if (c < 1) tmem_ld32(ts + 32u * (c + 1), x[(c + 1) & 1]);
            if (masked) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (key0 + 32 * c + e >= limit) v[e] = 0xff800000u;  // -inf
            }
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 y = fma_f32x2(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), rm, nm);
              const float2 z = make_float2(ex2(y.x), ex2(y.y));
              acc = add_f32x2(acc, z);
              p[16 * c + e / 2] = pack_f16x2(z.x, z.y);
            }
          }
          sum = acc.x + acc.y;
          const bool over = sum > kMostSum;
          if (again == 2 || !__any_sync(0xffffffffu, over)) break;  // once is enough below scores of 2^24
          // a new maximum: O and l so far in its terms, and these scores once more
          float top = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t v[32];
            tmem_ld32(ts + 32u * c, v);
            tmem_wait_ld(v);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (key0 + 32 * c + e < limit) top = fmaxf(top, __uint_as_float(v[e]));
          }
          const float to_m = over ? top * rowmul - kHeadroom : M, f = ex2(M - to_m);
          M = to_m;
          l *= f;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t v[32];
              tmem_ld32(to + c, v);
              tmem_wait_ld(v);
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
              tmem_st32(to + c, v);
            }
            tmem_wait_st();
          }
        }
        l += sum;
        tmem_st32(ts, p);
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
        uint32_t v[32];
        float x[32];
        __syncwarp();
        if (nt > 0) {
          tmem_ld32(to + c, v);
          tmem_wait_ld(v);
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = none ? 0.0f : __uint_as_float(v[e]) * f;
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
cudaError_t wide_launch(const Kv4AttnArgs& a, int64_t ctas, cudaStream_t st) {
  static std::atomic<uint64_t> configured{0};
  static std::atomic<bool> fits{false};
  cudaError_t e = configure_once(kv4_wide_kernel<NG>, WidePlan<NG>::kSmem, configured);
  if (e != cudaSuccess) return e;
  if (!fits.load(std::memory_order_relaxed)) {  // a split beyond the launch's registers would never start
    cudaFuncAttributes at;
    if ((e = cudaFuncGetAttributes(&at, kv4_wide_kernel<NG>)) != cudaSuccess) return e;
    if (at.numRegs * kWideThreads < 32 * (kSoftWarps * kSoftRegs + kDecodeWarps * kDecodeRegs) + 128 * kOtherRegs)
      return cudaErrorInvalidKernelImage;
    fits.store(true, std::memory_order_relaxed);
  }
  count_launch();
  kv4_wide_kernel<NG><<<(unsigned)ctas, kWideThreads, WidePlan<NG>::kSmem, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_wide(const Kv4AttnArgs& a, int head_dim, cudaStream_t st) {
  // n rows have n / 256 whole tiles and a ragged one a chunk, whose chunks have wide_rows at least
  const int64_t rows = (int64_t)a.T * (a.n_head / a.n_kv);
  const int64_t ctas = (rows / 256 + std::min<int64_t>(a.S, rows / a.wide_rows)) * a.n_kv;
  if (ctas == 0) return cudaSuccess;
  if (ctas > INT32_MAX) return cudaErrorInvalidConfiguration;
  return head_dim == 128 ? wide_launch<4>(a, ctas, st) : wide_launch<2>(a, ctas, st);
}

}  // namespace rtd
