// rtd_kv4.cu -- the paged KV cache held in 4 bits, sm_100a: block tables built on the
// device, the quantising append, the attention that reads it and a plain reader.
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
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "rtd_common.cuh"
#include "rtd_kernels.h"

namespace rtd {
namespace {

constexpr int kTok = 16;  // tokens of a page

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

// Byte of the half word with dims 32 g + 4 n .. + 3 of V, within the token's row.
template <int NG>
__device__ __forceinline__ int v_half_byte(int t, int g, int n) {
  if constexpr (NG == 4)
    return ((n * 2 + (g >> 1)) ^ (8 * ((t >> 1) & 1))) * 4 + (g & 1) * 2;
  else
    return ((NG & 1) && g == NG - 1) ? ((NG - 1) * 8 + n) * 2 : n * 4 + (g & 1) * 2;
}

// ------------------------------------------------------------------ block tables
// One cluster serves the call.  Every CTA reads the S lengths and scans three counts per
// sequence (new tokens, blocks taken, blocks given back), so that after one cluster
// barrier -- behind which the state may be overwritten -- each thread finds its share of
// the tokens and blocks by binary search, without a second pass over memory.
// Bound: latency (two loads, three scans, one barrier); the bytes are a few per sequence.
constexpr int kPlanThreads = 1024;

struct PlanArgs {
  const int* want;
  int S;
  int* length;
  int* table;
  int max_blocks;
  int* free_list;
  int* free_count;
  int num_blocks;
  int* q_start;  // null: no token lists
  int* tok_seq;
  int* tok_pos;
  int* tok_slot;
  int max_tokens;
  int* status;
};

// Exclusive sums of three counts over the block's threads; returns the totals.
__device__ __forceinline__ void scan3(int64_t (&v)[3], int64_t (&total)[3], int64_t (*warp_sums)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc[3] = {v[0], v[1], v[2]};
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc[k], o);
      if (lane >= o) inc[k] += y;
    }
  if (lane == 31)
    for (int k = 0; k < 3; ++k) warp_sums[k][warp] = inc[k];
  __syncthreads();
  if (warp < 3) {
    int64_t x = warp_sums[warp][lane], y0 = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncwarp();
    warp_sums[warp][lane] = x - y0;
    if (lane == 31) warp_sums[3 + warp][0] = x;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    v[k] = inc[k] - v[k] + warp_sums[k][warp];
    total[k] = warp_sums[3 + k][0];
  }
}

// The last index s with off[s] <= x, over off[0..n] ascending (off[n] > x).
__device__ __forceinline__ int owner(const int* off, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const PlanArgs a) {
  extern __shared__ int sm[];
  __shared__ int64_t warp_sums[6][32];
  __shared__ int bad;
  const int S = a.S, tid = threadIdx.x;
  int* tok_off = sm;             // [S + 1] first token of each sequence
  int* take_off = tok_off + S + 1;  // [S + 1] first block taken
  int* give_off = take_off + S + 1; // [S + 1] first block given back
  int* old_len = give_off + S + 1;  // [S]
  if (tid == 0) bad = 0;
  __syncthreads();
  const int per = (S + kPlanThreads - 1) / kPlanThreads;
  const int s0 = min(S, tid * per), s1 = min(S, s0 + per);
  const int cap = a.max_blocks * kTok;
  const int count = *a.free_count;
  int64_t sum[3] = {0, 0, 0}, total[3];
  bool wrong = count < 0 || count > a.num_blocks;
  for (int s = s0; s < s1; ++s) {
    const int w = a.want[s], l = a.length[s];
    wrong |= w < 0 || w > cap || l < 0 || l > cap;
    old_len[s] = l;
    const int need = (w + kTok - 1) / kTok, have = (l + kTok - 1) / kTok;
    sum[0] += max(0, w - l);
    sum[1] += max(0, need - have);
    sum[2] += max(0, have - need);
  }
  if (wrong) bad = 1;
  scan3(sum, total, warp_sums);  // its barriers also publish `bad`
  const int64_t left = (int64_t)count + total[2] - total[1];
  const bool fail = bad || left < 0 || left > a.num_blocks || (a.q_start && total[0] > a.max_tokens) ||
                    total[0] > INT32_MAX || total[2] > a.num_blocks;
  if (!fail)
    for (int s = s0; s < s1; ++s) {
      const int w = a.want[s], l = old_len[s];
      const int need = (w + kTok - 1) / kTok, have = (l + kTok - 1) / kTok;
      tok_off[s] = (int)sum[0];
      take_off[s] = (int)sum[1];
      give_off[s] = (int)sum[2];
      sum[0] += max(0, w - l);
      sum[1] += max(0, need - have);
      sum[2] += max(0, have - need);
    }
  if (tid == 0) {
    tok_off[S] = (int)total[0];
    take_off[S] = (int)total[1];
    give_off[S] = (int)total[2];
  }
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  __syncthreads();
  // every CTA has read the state: from here it may be overwritten
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  const int gt = (int)rank * kPlanThreads + tid, NT = (int)ranks * kPlanThreads;
  if (fail) {  // nothing changes; the token lists are empty
    if (gt == 0) raise_status(a.status, kDevCache);
    if (a.q_start) {
      for (int s = gt; s <= S; s += NT) a.q_start[s] = 0;
      for (int t = gt; t < a.max_tokens; t += NT) a.tok_seq[t] = a.tok_pos[t] = a.tok_slot[t] = -1;
    }
    return;
  }
  const int T = (int)total[0], take = (int)total[1], give = (int)total[2];
  // the e-th block given back: sequences in order, each from its last block down
  auto given = [&](int e) {
    const int s = owner(give_off, S, e);
    const int have = (old_len[s] + kTok - 1) / kTok;
    return a.table[(int64_t)s * a.max_blocks + have - 1 - (e - give_off[s])];
  };
  // the j-th block taken: from the top of the stack, the blocks just given back first
  auto taken = [&](int j) {
    const int at = count + give - 1 - j;
    return at < count ? a.free_list[at] : given(at - count);
  };
  for (int j = gt; j < take; j += NT) {
    const int s = owner(take_off, S, j);
    const int have = (old_len[s] + kTok - 1) / kTok;
    a.table[(int64_t)s * a.max_blocks + have + (j - take_off[s])] = taken(j);
  }
  for (int e = gt; e < give - take; e += NT) a.free_list[count + e] = given(e);
  for (int s = gt; s < S; s += NT) a.length[s] = a.want[s];
  if (gt == 0) *a.free_count = (int)left;
  if (!a.q_start) return;
  for (int s = gt; s <= S; s += NT) a.q_start[s] = tok_off[s];
  for (int t = gt; t < a.max_tokens; t += NT) {
    int seq = -1, pos = -1, slot = -1;
    if (t < T) {
      seq = owner(tok_off, S, t);
      const int l = old_len[seq], have = (l + kTok - 1) / kTok;
      pos = l + (t - tok_off[seq]);
      const int b = pos / kTok;
      // a block of this call may not be in the table yet: ask where it comes from
      const int blk = b < have ? a.table[(int64_t)seq * a.max_blocks + b] : taken(take_off[seq] + b - have);
      slot = blk * kTok + pos % kTok;
    }
    a.tok_seq[t] = seq;
    a.tok_pos[t] = pos;
    a.tok_slot[t] = slot;
  }
}

// ------------------------------------------------------------------ rope + quantising append
// A CTA serves one token (and a share of its heads when tokens are few): the rotation
// angles pos * inv_freq[i] are formed and reduced in 64 bits once per CTA -- at position
// 100000 a 32-bit angle is wrong by 6e-3 -- and their cosines and sines, rounded to f32,
// serve every head.  A warp takes a head at a time, lane = dim within the group: the
// group's extremes come from two warp reductions over order-mapped integers, whose ends
// also reveal infinities and NaN.  Bound: HBM (x in, q and the pages out).
constexpr int kAppThreads = 256;

struct AppendArgs {
  const void* q;
  const void* k;
  const void* v;
  int64_t ldq, ldk, ldv;
  int x_dtype;
  int n_head, n_kv, rot_dim;
  const double* inv_freq;
  const int* tok_pos;
  const int* tok_slot;
  uint8_t* pages;
  int64_t num_slots;
  float* q_out;
  int* status;
};

__device__ __forceinline__ int order_map(float x) {
  const int b = __float_as_int(x);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float order_unmap(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }

// One group of 32 dims, a lane each: its header and this lane's code.
__device__ __forceinline__ uint32_t quantise(float x, uint32_t& header) {
  const int i = order_map(x);
  const int lo_i = __reduce_min_sync(0xffffffffu, i), hi_i = __reduce_max_sync(0xffffffffu, i);
  const int inf = 0x7f800000;
  const float lo = order_unmap(lo_i), hi = order_unmap(hi_i);
  const __half d = __float2half_rn(__fdiv_rn(hi - lo, 15.0f)), m = __float2half_rn(lo);
  if (hi_i >= inf || lo_i <= order_map(-INFINITY) || __hisinf(d) || __hisinf(m)) {
    header = 0x7fff7fffu;
    return 0;
  }
  header = (uint32_t)__half_as_ushort(d) | ((uint32_t)__half_as_ushort(m) << 16);
  const float df = __half2float(d);
  if (!(df > 0.0f)) return 0;
  return (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x, __half2float(m)), df)), 0.0f), 15.0f);
}

template <int NG>
__global__ void __launch_bounds__(kAppThreads) rope_kv4_kernel(const AppendArgs a) {
  constexpr int D = 32 * NG;
  __shared__ float2 cs[D / 2];
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  const int slot = __ldg(a.tok_slot + t), pos = __ldg(a.tok_pos + t);
  const int half = a.rot_dim / 2;
  const bool there = slot >= 0 && slot < a.num_slots;
  if (slot >= a.num_slots && tid == 0 && blockIdx.y == 0) raise_status(a.status, kDevCache);
  for (int i = tid; i < half; i += kAppThreads) {
    double s, c;
    sincos((double)pos * a.inv_freq[i], &s, &c);
    cs[i] = make_float2((float)c, (float)s);
  }
  __syncthreads();
  const int heads = a.n_head + 2 * a.n_kv;
  const int warps = gridDim.y * (kAppThreads / 32);
  for (int j = blockIdx.y * (kAppThreads / 32) + (tid >> 5); j < heads; j += warps) {
    const bool is_q = j < a.n_head, is_v = j >= a.n_head + a.n_kv;
    const int h = is_q ? j : (is_v ? j - a.n_head - a.n_kv : j - a.n_head);
    if (!is_q && !there) continue;
    const void* src = is_q ? a.q : (is_v ? a.v : a.k);
    const int64_t base = t * (is_q ? a.ldq : (is_v ? a.ldv : a.ldk)) + (int64_t)h * D;
    float x[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int d = 32 * g + lane;
      float v = load_as_f32(src, a.x_dtype, base + d);
      if (!is_v && d < 2 * half) {
        const bool first = d < half;
        const float o = load_as_f32(src, a.x_dtype, base + (first ? d + half : d - half));
        const float2 r = cs[first ? d : d - half];
        // products rounded first, as rtd_rope_kv_append does
        v = first ? __fsub_rn(__fmul_rn(v, r.x), __fmul_rn(o, r.y)) : __fadd_rn(__fmul_rn(v, r.x), __fmul_rn(o, r.y));
      }
      x[g] = v;
    }
    if (is_q) {
      float* out = a.q_out + (t * a.n_head + h) * (int64_t)D;
#pragma unroll
      for (int g = 0; g < NG; ++g) out[32 * g + lane] = x[g];
      continue;
    }
    uint8_t* page = a.pages + ((int64_t)(slot / kTok) * a.n_kv + h) * (20 * D) + (is_v ? 10 * D : 0);
    const int tk = slot % kTok;
    uint8_t* row = page + tk * (D / 2);
    uint32_t* head = reinterpret_cast<uint32_t*>(page + 8 * D) + tk * NG;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint32_t header;
      uint32_t c = quantise(x[g], header);
      if (lane == 0) head[g] = header;
      if (!is_v) {
        c <<= 4 * (lane & 7);
        c |= __shfl_xor_sync(0xffffffffu, c, 1);
        c |= __shfl_xor_sync(0xffffffffu, c, 2);
        c |= __shfl_xor_sync(0xffffffffu, c, 4);
        if ((lane & 7) == 0) reinterpret_cast<uint32_t*>(row)[(lane >> 3) * NG + g] = c;
      } else {
        c <<= 4 * (lane & 3);
        c |= __shfl_xor_sync(0xffffffffu, c, 1);
        c |= __shfl_xor_sync(0xffffffffu, c, 2);
        if ((lane & 3) == 0) *reinterpret_cast<uint16_t*>(row + v_half_byte<NG>(tk, g, lane >> 2)) = (uint16_t)c;
      }
    }
  }
}

// ------------------------------------------------------------------ reader
// A warp per (slot, kv head): K and V rows as the values their codes stand for.
template <int NG>
__global__ void __launch_bounds__(256) kv4_read_kernel(const int* slots, int64_t n, int n_kv, const uint8_t* pages,
                                                       int64_t num_slots, void* k, void* v, int dt, int* status) {
  constexpr int D = 32 * NG;
  const int lane = threadIdx.x & 31;
  for (int64_t j = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); j < n * n_kv; j += (int64_t)gridDim.x * 8) {
    const int64_t r = j / n_kv;
    const int h = (int)(j - r * n_kv), slot = __ldg(slots + r);
    const bool there = slot >= 0 && slot < num_slots;
    if (slot >= num_slots && lane == 0) raise_status(status, kDevCache);
    const int tk = there ? slot % kTok : 0;
    const uint8_t* page = pages + (there ? ((int64_t)(slot / kTok) * n_kv + h) * (20 * D) : 0);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint8_t* p = page + half * 10 * D;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float x = 0.0f;
        if (there) {
          const uint32_t header = reinterpret_cast<const uint32_t*>(p + 8 * D)[tk * NG + g];
          const uint8_t* row = p + tk * (D / 2);
          const int byte = half ? v_half_byte<NG>(tk, g, lane >> 2) + ((lane & 3) >> 1)
                                : ((lane >> 3) * NG + g) * 4 + ((lane & 7) >> 1);
          const int c = (row[byte] >> (4 * (lane & 1))) & 15;
          x = fmaf(f16_bits_to_f32(header & 0xffffu), (float)c, f16_bits_to_f32(header >> 16));
        }
        store_from_f32(half ? v : k, dt, j * D + 32 * g + lane, x);
      }
    }
  }
}

// ------------------------------------------------------------------ attention
// CTA (sequence s, kv head, tile of 8 rows, chunk of keys); row = token * G + head of the
// group.  Each of its four warps takes every fourth page of the chunk through its own
// ring of bulk copies, with its own running softmax; the warps' states join in shared
// memory, the chunks' in the workspace (the last CTA of a tile joins them in chunk order,
// so the order of arrival changes nothing).
//
// The products run on the tensor cores on the codes themselves, and step and minimum are
// applied to the 32-bit sums of each group:  q.k = sum_g d_g (q_g . c_g) + m_g sum(q_g).
// A nibble masked into an f16 pair under the exponent of 1024 is 1024 + c (or 1024 + 16 c),
// and one packed fma makes it c, exactly: a word of eight codes becomes four operand
// registers with four masks, one shift and four fmas.  (Left as the subnormal c * 2^-24
// the fma would be saved, but the tensor cores align a subnormal's product as if its
// leading zeros counted: measured 2e-5 of the output against 64 bits.)  V takes c - 8, so
// that a long mean of values near zero is a sum of both signs and not a difference of two
// large ones; sum_j p_j (m_jg + 8 d_jg) is added in the end.
// Rows 0..7 of the 16-row MMA hold the queries' f16 heads, rows 8..15 the remainders, so
// that a query enters with 22 bits; likewise p * d_g for V.  Queries are scaled by a power
// of two per row, and p by 2^8, to keep both parts inside f16's range.
constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = 32 * kAttnWarps;
constexpr int kStages = 6;
constexpr int kRows = 8;
constexpr float kHeadroom = 8.0f;  // p = 2^(x - max + 8) right after the maximum is set ...
constexpr float kGrowth = 12.0f;   // ... and the maximum stays until a score would pass 2^12

struct Kv4AttnArgs {
  const void* q;
  int q_dtype;
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
  int64_t ldo;
  int tiles, chunk, chunks;  // 8-row tiles a sequence, keys a chunk, chunks a tile
  float* part;               // [S][n_kv][tiles][chunks][8][D + 2]
  unsigned* count;           // [S][n_kv][tiles], zero between calls
  int* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // |e| <= 126

// Nibbles 0 and 4 (odd = false) or 1 and 5 (odd = true) of w as the f16 pair c - S.
template <int S, bool odd>
__device__ __forceinline__ uint32_t codes(uint32_t w) {
  const uint32_t b = lop_and_or(w, odd ? 0x00F000F0u : 0x000F000Fu, 0x64006400u);
  const __half2 h = *reinterpret_cast<const __half2*>(&b);
  const __half2 r = odd ? __hfma2(h, __float2half2_rn(0.0625f), __float2half2_rn(-64.0f - S))
                        : __hadd2(h, __float2half2_rn(-1024.0f - S));
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <int NG>
__global__ void __launch_bounds__(kAttnThreads) kv4_attn_kernel(const Kv4AttnArgs a) {
  constexpr int D = 32 * NG, PB = 20 * D;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kAttnWarps][kStages];
  __shared__ int last;
  const int G = a.n_head / a.n_kv;
  // tile fastest: CTAs that read the same keys run together
  unsigned bid = blockIdx.x;
  const int tile = a.tiles - 1 - (int)(bid % a.tiles);  // later tiles see more keys: first
  bid /= a.tiles;
  const int chunk = (int)(bid % a.chunks);
  bid /= a.chunks;
  const int kvh = (int)(bid % a.n_kv), s = (int)(bid / a.n_kv);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int qs = __ldg(a.q_start + s), nq = __ldg(a.q_start + s + 1) - qs;
  int ctx = __ldg(a.ctx_len + s);
  if (qs < 0 || nq < 0 || (int64_t)qs + nq > a.T || nq > a.max_q) {
    if (tid == 0) raise_status(a.status, kDevCache);
    return;
  }
  if (ctx > a.max_ctx) {
    if (tid == 0) raise_status(a.status, kDevCache);
    ctx = 0;
  }
  const int row0 = tile * kRows, rows = nq * G;
  if (row0 >= rows) return;
  // keys seen by a row: its position and before
  auto seen = [&](int row) { return max(0, ctx - nq + row / G + 1); };
  const int most = seen(min(row0 + kRows, rows) - 1);
  const int active = max(1, (most + a.chunk - 1) / a.chunk);
  if (chunk >= active) return;
  const int key0 = chunk * a.chunk, key1 = min(most, key0 + a.chunk);
  const int page0 = key0 / kTok, npages = (max(0, key1 - key0) + kTok - 1) / kTok;
  const int mine = npages > warp ? (npages - warp + kAttnWarps - 1) / kAttnWarps : 0;

  // ---- this warp's ring of pages
  uint8_t* ring = smem + warp * (kStages * PB);
  const int* table = a.table + (int64_t)s * a.max_blocks + page0 + warp;
  bool bad = false;
  int ids = 0;
  auto load_ids = [&](int base) {
    const int j = base + lane;
    ids = 0;
    if (j < mine) {
      ids = __ldg(table + j * kAttnWarps);
      if ((unsigned)ids >= (unsigned)a.num_blocks) {
        bad = true;
        ids = 0;
      }
    }
  };
  auto issue = [&](int j) {
    if (j >= mine) return;
    if ((j & 31) == 0) load_ids(j);
    const int blk = __shfl_sync(0xffffffffu, ids, j & 31);
    if (lane == 0) {
      uint64_t* bar = &bars[warp][j % kStages];
      mbar_arrive_expect_tx(bar, PB);
      bulk_g2s(ring + (j % kStages) * PB, a.pages + ((int64_t)blk * a.n_kv + kvh) * PB, PB, bar);
    }
  };
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[warp][i], 1);
    fence_mbar_init();
  }
  __syncwarp();
  for (int j = 0; j < kStages; ++j) issue(j);

  // ---- queries: lane (row r, quad lane i) holds dims 8 i .. 8 i + 7 of every group
  const int r = lane >> 2, qi = lane & 3;
  const int row = row0 + r;
  const bool live = row < rows;
  const int limit = live ? min(seen(row), key1) : 0;
  uint32_t qa[NG][2][4];
  float qsum[NG], rowmul;
  {
    float x[NG][8];
    const int64_t base = live ? (int64_t)(qs + row / G) * a.ldq + (int64_t)(kvh * G + row % G) * D : 0;
    float mx = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = live ? load_as_f32(a.q, a.q_dtype, base + 32 * g + 8 * qi + e) * a.scale * 1.4426950408889634f : 0.0f;
        x[g][e] = v;
        sum += v;
        mx = fmaxf(mx, fabsf(v));
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      qsum[g] = sum;
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // 2^k brings the row's largest into [2^12, 2^13)
    int k = 0;
    if (mx > 0.0f && mx < INFINITY) k = max(-100, min(100, 12 - ilogbf(mx)));
    const float up = pow2(k);
    rowmul = pow2(-k);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      qsum[g] *= up;
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int e = 2 * st + b;  // nibbles e and e + 4
          const float v0 = x[g][e] * up, v1 = x[g][e + 4] * up;
          const __half2 hi = __floats2half2_rn(v0, v1);
          const float2 hf = __half22float2(hi);
          const __half2 lo = __floats2half2_rn(v0 - hf.x, v1 - hf.y);
          qa[g][st][2 * b] = *reinterpret_cast<const uint32_t*>(&hi);
          qa[g][st][2 * b + 1] = *reinterpret_cast<const uint32_t*>(&lo);
        }
    }
  }

  float M = -1e30f, l = 0.0f;
  float z[NG], o[NG][4][4];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    z[g] = 0.0f;
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[g][p][c] = 0.0f;
  }
  auto rescale = [&](float f) {
    l *= f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      z[g] *= f;
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[g][p][c] *= f;
    }
  };

  // ---- pages
  const int kt = ((r & 1) << 2) | (r >> 1);  // token of S column r: columns 2 i, 2 i + 1 are tokens i, i + 4
  for (int j = 0; j < mine; ++j) {
    const int st = j % kStages;
    mbar_wait_bounded(&bars[warp][st], (j / kStages) & 1, a.status);
    const uint8_t* page = ring + st * PB;
    const int key = key0 + (warp + j * kAttnWarps) * kTok;
    float x[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t w[NG], h0[NG], h1[NG];
      const uint32_t* kw = reinterpret_cast<const uint32_t*>(page + (8 * u + kt) * (D / 2)) + qi * NG;
      const uint32_t* kh = reinterpret_cast<const uint32_t*>(page + 8 * D) + (8 * u + qi) * NG;
      if constexpr (NG == 4) {
        *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(kw);
        *reinterpret_cast<uint4*>(h0) = *reinterpret_cast<const uint4*>(kh);
        *reinterpret_cast<uint4*>(h1) = *reinterpret_cast<const uint4*>(kh + 4 * NG);
      } else {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          w[g] = kw[g];
          h0[g] = kh[g];
          h1[g] = kh[4 * NG + g];
        }
      }
      x[u][0] = x[u][1] = 0.0f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t hiw = w[g] >> 8;
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma_f16_acc(acc, qa[g][0][0], qa[g][0][1], qa[g][0][2], qa[g][0][3], codes<0, false>(w[g]),
                    codes<0, true>(w[g]));
        mma_f16_acc(acc, qa[g][1][0], qa[g][1][1], qa[g][1][2], qa[g][1][3], codes<0, false>(hiw),
                    codes<0, true>(hiw));
        const float2 d0 = __half22float2(*reinterpret_cast<__half2*>(&h0[g]));
        const float2 d1 = __half22float2(*reinterpret_cast<__half2*>(&h1[g]));
        x[u][0] = fmaf(d0.x, acc[0] + acc[2], fmaf(d0.y, qsum[g], x[u][0]));
        x[u][1] = fmaf(d1.x, acc[1] + acc[3], fmaf(d1.y, qsum[g], x[u][1]));
      }
    }
    bool vis[2][2];
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        vis[u][c] = key + 8 * u + 4 * c + qi < limit;
        x[u][c] = vis[u][c] ? x[u][c] * rowmul : -INFINITY;
        mx = fmaxf(mx, x[u][c]);
      }
    if (__any_sync(0xffffffffu, mx > M + kGrowth)) {
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      if (mx > M + kGrowth) {
        const float to = mx - kHeadroom;
        rescale(ex2(M - to));
        M = to;
      }
    }
    float p[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) p[u][c] = ex2(x[u][c] - M);
    // V headers of this lane's four tokens
    float pd[NG][4], over = 0.0f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t* vh = reinterpret_cast<const uint32_t*>(page + 18 * D) + (8 * u + 4 * c + qi) * NG;
        uint32_t h[NG];
        if constexpr (NG == 4)
          *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(vh);
        else
#pragma unroll
          for (int g = 0; g < NG; ++g) h[g] = vh[g];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float2 dm = __half22float2(*reinterpret_cast<__half2*>(&h[g]));
          // a key that this row does not see may hold anything
          pd[g][2 * u + c] = vis[u][c] ? p[u][c] * dm.x : 0.0f;
          z[g] = vis[u][c] ? fmaf(p[u][c], dm.y, fmaf(8.0f, pd[g][2 * u + c], z[g])) : z[g];
          over = fmaxf(over, pd[g][2 * u + c]);
        }
      }
    l += (p[0][0] + p[0][1]) + (p[1][0] + p[1][1]);
    if (__any_sync(0xffffffffu, over > 60000.0f)) {  // a step above 16: lower p until it fits f16
      over = fmaxf(over, __shfl_xor_sync(0xffffffffu, over, 1));
      over = fmaxf(over, __shfl_xor_sync(0xffffffffu, over, 2));
      if (over > 60000.0f && over < INFINITY) {
        const int e = ilogbf(over) - 13;
        const float f = pow2(-e);
        M += (float)e;
        rescale(f);
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int c = 0; c < 4; ++c) pd[g][c] *= f;
      }
    }
    // O += (p d) C: pairs of tokens (i, i + 4) and (i + 8, i + 12)
    uint32_t v[4][(NG + 1) / 2];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint8_t* vr = page + 10 * D + (4 * c + qi) * (D / 2);
      if constexpr (NG == 4) {
        *reinterpret_cast<uint2*>(v[c]) = *reinterpret_cast<const uint2*>(vr + (((2 * r) ^ (8 * (qi >> 1))) << 2));
      } else {
        if constexpr (NG >= 2) v[c][0] = *reinterpret_cast<const uint32_t*>(vr + 4 * r);
        if constexpr (NG & 1) v[c][NG / 2] = *reinterpret_cast<const uint16_t*>(vr + ((NG - 1) * 8 + r) * 2);
      }
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const __half2 h0 = __floats2half2_rn(pd[g][0], pd[g][1]), h1 = __floats2half2_rn(pd[g][2], pd[g][3]);
      const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
      const __half2 l0 = __floats2half2_rn(pd[g][0] - f0.x, pd[g][1] - f0.y);
      const __half2 l1 = __floats2half2_rn(pd[g][2] - f1.x, pd[g][3] - f1.y);
      const uint32_t a0 = *reinterpret_cast<const uint32_t*>(&h0), a1 = *reinterpret_cast<const uint32_t*>(&l0);
      const uint32_t a2 = *reinterpret_cast<const uint32_t*>(&h1), a3 = *reinterpret_cast<const uint32_t*>(&l1);
      const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
      const uint32_t b0 = prmt(v[0][g / 2], v[1][g / 2], sel), b1 = prmt(v[2][g / 2], v[3][g / 2], sel);
      mma_f16_acc(o[g][0], a0, a1, a2, a3, codes<8, false>(b0), codes<8, false>(b1));
      mma_f16_acc(o[g][1], a0, a1, a2, a3, codes<8, true>(b0), codes<8, true>(b1));
      mma_f16_acc(o[g][2], a0, a1, a2, a3, codes<8, false>(b0 >> 8), codes<8, false>(b1 >> 8));
      mma_f16_acc(o[g][3], a0, a1, a2, a3, codes<8, true>(b0 >> 8), codes<8, true>(b1 >> 8));
    }
    __syncwarp();
    issue(j + kStages);
  }

  // ---- join the warps (the ring's memory is free once every warp is done)
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  if (__any_sync(0xffffffffu, bad)) {  // a block id outside the pool: no number stands for these rows
    if (lane == 0) raise_status(a.status, kDevCache);
    l = NAN;
  }
  __syncthreads();
  float* st = reinterpret_cast<float*>(smem);  // [warp][8][D + 2]
  {
    float* w = st + (warp * kRows + r) * (D + 2);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float zz = z[g];
      zz += __shfl_xor_sync(0xffffffffu, zz, 1);
      zz += __shfl_xor_sync(0xffffffffu, zz, 2);
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        w[32 * g + 8 * qi + p] = (o[g][p][0] + o[g][p][2]) + zz;
        w[32 * g + 8 * qi + 4 + p] = (o[g][p][1] + o[g][p][3]) + zz;
      }
    }
    if (qi == 0) {
      w[D] = M;
      w[D + 1] = l;
    }
  }
  __syncthreads();
  const int64_t unit = ((int64_t)s * a.n_kv + kvh) * a.tiles + tile;
  float* part = a.part + (unit * a.chunks + chunk) * (kRows * (D + 2));
  auto put = [&](int rr, int d, float v) {
    const int rw = row0 + rr;
    if (rw < rows)
      store_from_f32(a.o, a.o_dtype, (int64_t)(qs + rw / G) * a.ldo + (int64_t)(kvh * G + rw % G) * D + d, v);
  };
  for (int e = tid; e < kRows * D; e += kAttnThreads) {
    const int rr = e / D, d = e - rr * D;
    const float* w = st + rr * (D + 2);
    constexpr int ws = kRows * (D + 2);
    float m = w[D];
#pragma unroll
    for (int k = 1; k < kAttnWarps; ++k) m = fmaxf(m, w[k * ws + D]);
    float ls = 0.0f, os = 0.0f;
#pragma unroll
    for (int k = 0; k < kAttnWarps; ++k) {
      const float f = ex2(w[k * ws + D] - m);
      ls = fmaf(w[k * ws + D + 1], f, ls);
      os = fmaf(w[k * ws + d], f, os);
    }
    if (active == 1) {
      put(rr, d, ls == 0.0f ? 0.0f : os / ls);
    } else {
      part[rr * (D + 2) + d] = os;
      if (d == 0) {
        part[rr * (D + 2) + D] = m;
        part[rr * (D + 2) + D + 1] = ls;
      }
    }
  }
  if (active == 1) return;
  // ---- the last chunk of the tile joins them all, in chunk order
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    last = atomicAdd(a.count + unit, 1u) == (unsigned)active - 1u;
    if (last) a.count[unit] = 0;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  const float* all = a.part + unit * a.chunks * (kRows * (D + 2));
  constexpr int cs = kRows * (D + 2);
  for (int e = tid; e < kRows * D; e += kAttnThreads) {
    const int rr = e / D, d = e - rr * D;
    const float* w = all + rr * (D + 2);
    float m = -1e30f;
    for (int k = 0; k < active; ++k) m = fmaxf(m, __ldcg(w + (int64_t)k * cs + D));
    float ls = 0.0f, os = 0.0f;
    for (int k = 0; k < active; ++k) {
      const float f = ex2(__ldcg(w + (int64_t)k * cs + D) - m);
      ls = fmaf(__ldcg(w + (int64_t)k * cs + D + 1), f, ls);
      os = fmaf(__ldcg(w + (int64_t)k * cs + d), f, os);
    }
    put(rr, d, ls == 0.0f ? 0.0f : os / ls);
  }
}

template <int NG>
cudaError_t attn_launch(const Kv4AttnArgs& a, int64_t blocks, cudaStream_t st) {
  constexpr int D = 32 * NG;
  constexpr int smem = std::max(kAttnWarps * kStages * 20 * D, kAttnWarps * kRows * (D + 2) * 4);
  // per device, and cheap: the attribute belongs to the current context
  cudaError_t e = cudaFuncSetAttribute(kv4_attn_kernel<NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  count_launch();
  kv4_attn_kernel<NG><<<(unsigned)blocks, kAttnThreads, smem, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_plan(const int* want, int S, int* length, int* table, int max_blocks, int* free_list,
                           int* free_count, int num_blocks, int* q_start, int* tok_seq, int* tok_pos, int* tok_slot,
                           int max_tokens, int* status, cudaStream_t st) {
  PlanArgs a{want, S, length, table, max_blocks, free_list, free_count, num_blocks, q_start, tok_seq, tok_pos,
             tok_slot, max_tokens, status};
  const size_t smem = (size_t)(4 * S + 3) * sizeof(int);
  cudaError_t e = cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (4 * kPlanMaxSeqs + 3) * (int)sizeof(int));
  if (e != cudaSuccess) return e;
  const int64_t items = (q_start ? max_tokens : 0) + (int64_t)S;
  const unsigned ctas = items > 4 * kPlanThreads ? 8 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, kv_plan_kernel, a);
}

cudaError_t launch_rope_kv4(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                            int x_dtype, int64_t T, int n_head, int n_kv, int head_dim, int rot_dim,
                            const double* inv_freq, const int* tok_pos, const int* tok_slot, uint8_t* pages,
                            int num_blocks, float* q_out, int sm_count, int* status, cudaStream_t st) {
  AppendArgs a{q, k, v, ldq, ldk, ldv, x_dtype, n_head, n_kv, rot_dim, inv_freq, tok_pos, tok_slot, pages,
               (int64_t)num_blocks * kTok, q_out, status};
  const int heads = n_head + 2 * n_kv, warps = kAppThreads / 32;
  const dim3 grid((unsigned)T, T < 2 * sm_count ? (unsigned)((heads + warps - 1) / warps) : 1u);
  count_launch();
  switch (head_dim / 32) {
    case 1: rope_kv4_kernel<1><<<grid, kAppThreads, 0, st>>>(a); break;
    case 2: rope_kv4_kernel<2><<<grid, kAppThreads, 0, st>>>(a); break;
    case 3: rope_kv4_kernel<3><<<grid, kAppThreads, 0, st>>>(a); break;
    default: rope_kv4_kernel<4><<<grid, kAppThreads, 0, st>>>(a); break;
  }
  return cudaGetLastError();
}

cudaError_t launch_kv4_read(const int* slots, int64_t n, int n_kv, int head_dim, const uint8_t* pages, int num_blocks,
                            void* k, void* v, int dtype, int* status, cudaStream_t st) {
  const unsigned blocks = (unsigned)std::min<int64_t>((n * n_kv + 7) / 8, 1 << 16);
  const int64_t ns = (int64_t)num_blocks * kTok;
  count_launch();
  switch (head_dim / 32) {
    case 1: kv4_read_kernel<1><<<blocks, 256, 0, st>>>(slots, n, n_kv, pages, ns, k, v, dtype, status); break;
    case 2: kv4_read_kernel<2><<<blocks, 256, 0, st>>>(slots, n, n_kv, pages, ns, k, v, dtype, status); break;
    case 3: kv4_read_kernel<3><<<blocks, 256, 0, st>>>(slots, n, n_kv, pages, ns, k, v, dtype, status); break;
    default: kv4_read_kernel<4><<<blocks, 256, 0, st>>>(slots, n, n_kv, pages, ns, k, v, dtype, status); break;
  }
  return cudaGetLastError();
}

cudaError_t launch_kv4_attention(const Kv4Attention& c, int* plan_error) {
  *plan_error = 0;
  const int G = c.n_head / c.n_kv;
  const int64_t tiles = ((int64_t)c.max_q * G + kRows - 1) / kRows;
  const int64_t units = (int64_t)c.S * c.n_kv * tiles;
  // Chunks: enough CTAs for two per SM when (sequence, head, tile) alone are fewer, and at
  // most 2048 keys where lengths differ; none below 256 keys (four pages a warp).
  int64_t chunk = 2048;
  const int64_t want = (2 * (int64_t)c.sm_count + units - 1) / units;
  if (want > 1) chunk = std::min<int64_t>(chunk, ((c.max_ctx + want - 1) / want + 63) / 64 * 64);
  chunk = std::max<int64_t>(chunk, 256);
  if ((c.max_ctx + chunk - 1) / chunk > 64) chunk = ((c.max_ctx + 63) / 64 + 63) / 64 * 64;
  const int64_t slot = (int64_t)kRows * (c.head_dim + 2) * 4;
  while (chunk < c.max_ctx && (units > c.count_words || units * ((c.max_ctx + chunk - 1) / chunk) * slot > (int64_t)c.ws_bytes))
    chunk = units > c.count_words ? (c.max_ctx + 63) / 64 * 64 : 2 * chunk;
  const int64_t chunks = (c.max_ctx + chunk - 1) / chunk;
  const int64_t blocks = units * chunks;
  if (blocks > INT32_MAX) {
    *plan_error = 1;
    return cudaSuccess;
  }
  Kv4AttnArgs a{c.q, c.q_dtype, c.ldq, (int)c.T, c.n_head, c.n_kv, c.scale, c.q_start, c.ctx_len, c.S, c.block_table,
                c.max_blocks, c.max_q, c.max_ctx, c.pages, c.num_blocks, c.o, c.o_dtype, c.ldo, (int)tiles, (int)chunk,
                (int)chunks, c.ws, c.count, c.status};
  switch (c.head_dim / 32) {
    case 1: return attn_launch<1>(a, blocks, c.stream);
    case 2: return attn_launch<2>(a, blocks, c.stream);
    case 3: return attn_launch<3>(a, blocks, c.stream);
    default: return attn_launch<4>(a, blocks, c.stream);
  }
}

}  // namespace rtd
