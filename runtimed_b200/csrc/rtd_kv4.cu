// rtd_kv4.cu -- the paged KV cache held in 4 bits, sm_100a: block tables built on the
// device, the quantising append, the attention that reads it and a plain reader.  The pages'
// layout stands in rtd_kv4.cuh; prompt chunks with 16-bit outputs run in rtd_kv4_wide.cu.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "rtd_kv4.cuh"

namespace rtd {
namespace {


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
// serve every head.  Queries whose whole head turns go by quads of neighbouring dims of
// either half, asked for before the angles are formed.  Of the other heads a warp takes one
// at a time, lane = dim within the group: the group's extremes come from two warp reductions
// over order-mapped integers, whose ends also reveal infinities and NaN.
// Bound: HBM.  2000 tokens of 64/8 heads of 128 in f32 move 150 MB, 23 us at the copy rate; 38 us
// here (bf16 and f16, 109 MB, 17 us: 36).  The angles' 64-bit sines hold up a CTA for 2 us, with
// four or five CTAs on an SM.  With a lane per dim for the queries too (4-byte accesses) append
// and reader together took 59 us, 44 as they are.
constexpr int kAppThreads = 256;
constexpr int kAppQuads = 2;  // those 44 us; 1: 47; 4: 51, since fewer CTAs fit

struct AppendArgs {
  const void* q;
  const void* k;
  const void* v;
  int64_t ldq, ldk, ldv;
  int x_dtype;
  int q_wide;  // queries in whole quads of both halves
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

// Four neighbouring values: 16 bytes of f32 or 8 of 16 bits.
__device__ __forceinline__ uint4 load_quad(const void* p, int dt, int64_t i) {
  if (dt == 0) return *reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
  const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
  return make_uint4(v.x, v.y, 0u, 0u);
}
__device__ __forceinline__ float4 quad_as_f32(uint4 v, int dt) {
  if (dt == 0) return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
  float2 lo, hi;
  if (dt == 1) {
    lo = __half22float2(as_h2(v.x));
    hi = __half22float2(as_h2(v.y));
  } else {
    lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x));
    hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
  }
  return make_float4(lo.x, lo.y, hi.x, hi.y);
}
// A pair of dims turned by an angle, products rounded first, as rtd_rope_kv_append does.
__device__ __forceinline__ void turn(float x, float y, float2 r, float& a, float& b) {
  a = __fsub_rn(__fmul_rn(x, r.x), __fmul_rn(y, r.y));
  b = __fadd_rn(__fmul_rn(y, r.x), __fmul_rn(x, r.y));
}

template <int NG>
__global__ void __launch_bounds__(kAppThreads) rope_kv4_kernel(const AppendArgs a) {
  constexpr int D = 32 * NG;
  __shared__ __align__(16) float2 cs[D / 2];
  const int64_t t = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  const int slot = __ldg(a.tok_slot + t), pos = __ldg(a.tok_pos + t);
  const int half = a.rot_dim / 2;
  const bool there = slot >= 0 && slot < a.num_slots;
  if (slot >= a.num_slots && tid == 0 && blockIdx.y == 0) raise_status(a.status, kDevCache);
  // queries by quads of each half, if whole heads turn: kAppQuads are on their way before the
  // angles are formed
  constexpr int QD = D / 8;  // quads of a head's first half
  const int quads = a.q_wide ? a.n_head * QD : 0, step = gridDim.y * kAppThreads;
  int e = blockIdx.y * kAppThreads + tid;
  uint4 qa[kAppQuads], qb[kAppQuads];
  auto ask = [&]() {
#pragma unroll
    for (int k = 0; k < kAppQuads; ++k) {
      const int i = e + k * step;
      if (i >= quads) continue;
      const int64_t at = t * a.ldq + (i / QD) * D + 4 * (i % QD);
      qa[k] = load_quad(a.q, a.x_dtype, at);
      qb[k] = load_quad(a.q, a.x_dtype, at + D / 2);
    }
  };
  ask();
  for (int i = tid; i < half; i += kAppThreads) {
    double s, c;
    sincos((double)pos * a.inv_freq[i], &s, &c);
    cs[i] = make_float2((float)c, (float)s);
  }
  __syncthreads();
  for (; e < quads; e += kAppQuads * step, ask()) {
#pragma unroll
    for (int k = 0; k < kAppQuads; ++k) {
      const int i = e + k * step;
      if (i >= quads) continue;
      const float4 x = quad_as_f32(qa[k], a.x_dtype), y = quad_as_f32(qb[k], a.x_dtype);
      const float4* r = reinterpret_cast<const float4*>(cs + 4 * (i % QD));
      const float4 r0 = r[0], r1 = r[1];
      float4 u, v;
      turn(x.x, y.x, make_float2(r0.x, r0.y), u.x, v.x);
      turn(x.y, y.y, make_float2(r0.z, r0.w), u.y, v.y);
      turn(x.z, y.z, make_float2(r1.x, r1.y), u.z, v.z);
      turn(x.w, y.w, make_float2(r1.z, r1.w), u.w, v.w);
      float* out = a.q_out + (t * a.n_head + i / QD) * (int64_t)D + 4 * (i % QD);
      *reinterpret_cast<float4*>(out) = u;
      *reinterpret_cast<float4*>(out + D / 2) = v;
    }
  }
  // the other heads a warp each, a lane per dim of a group
  const int heads = a.n_head + 2 * a.n_kv, warps = gridDim.y * (kAppThreads / 32);
  for (int j = (a.q_wide ? a.n_head : 0) + blockIdx.y * (kAppThreads / 32) + (tid >> 5); j < heads; j += warps) {
    const bool is_q = j < a.n_head, is_v = j >= a.n_head + a.n_kv;
    const int h = is_q ? j : (is_v ? j - a.n_head - a.n_kv : j - a.n_head);
    if (!is_q && !there) continue;
    const void* src = is_q ? a.q : (is_v ? a.v : a.k);
    const int64_t base = t * (is_q ? a.ldq : (is_v ? a.ldv : a.ldk)) + (int64_t)h * D;
    float x[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) x[g] = load_as_f32(src, a.x_dtype, base + 32 * g + lane);
    if (!is_v && NG % 2 == 0 && half == D / 2) {
#pragma unroll
      for (int g = 0; g < NG / 2; ++g) {
        float u, v;
        turn(x[g], x[g + NG / 2], cs[32 * g + lane], u, v);
        x[g] = u;
        x[g + NG / 2] = v;
      }
    } else if (!is_v) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int d = 32 * g + lane;
        if (d >= 2 * half) continue;
        const float o = load_as_f32(src, a.x_dtype, base + (d < half ? d + half : d - half));
        float u;
        if (d < half)
          turn(x[g], o, cs[d], x[g], u);
        else
          turn(o, x[g], cs[d - half], u, x[g]);
      }
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
// Work: a unit is (sequence s, kv head, tile of 8 rows; row = token * G + head of the
// group), its cost the pages of its keys.  The units' pages form one line, which the
// resident CTAs share evenly, whatever the lengths; a unit that crosses a border is joined
// from its CTAs' partial states by the last of them, in CTA order, so equal calls give
// equal bits.  Each CTA finds its place from the lengths (S loads and a scan).  Within a
// CTA every fourth page goes to a warp, which streams it through its own ring of bulk
// copies and keeps its own running softmax; the warps' states join in shared memory.
//
// The products run on the tensor cores on the codes themselves, and step and minimum are
// applied to the 32-bit sums of each group:  q.k = sum_g d_g (q_g . c_g) + m_g sum(q_g),
// the minima's part as one more MMA over the groups.  For V the weights p * d_g multiply
// the codes, and one MMA of p with the headers gives the minima's part.
//
// EXACT (f32 and f16 outputs): rows 0..7 of the 16-row MMA hold the f16 heads of q and p d, rows
// 8..15 the remainders, so that both enter with 22 bits (p d is split by an exact fma).  A
// nibble masked into an f16 pair under the exponent of 1024 is 1024 + c (or 1024 + 16 c)
// and one packed addition makes it c (16 c, against a 16th of the query), exactly; V takes
// c - 8, so that a long mean of values near zero is a sum of both signs and not a
// difference of two large ones.
// Otherwise (bf16 outputs): the rows enter rounded to 11 bits and the nibble stays the
// f16 subnormal c * 2^-24, which saves the addition; the tensor cores align a subnormal's
// product as if its leading zeros counted, which costs 2e-5 of the output.  bf16 outputs come out
// 1.77e-3 off 64 bits, where their own rounding is 1.65e-3; f16 ones were 5e-4 off in this form,
// where rounding them costs 2e-4.
//
// Bound: 64 sequences of up to 4096 tokens, 64 query heads on 8 (f32 outputs) read 240 MB,
// 37 us at the copy rate; the kernel takes 97 us (2.5 TB/s), 3 sequences of up to 60000 in
// bf16 (184 MB, 28 us) 69 us, in f16 78.  Neither the bytes nor the issue slots (57 % of a
// scheduler's cycles; 600 instructions a page) bound it but a page's chain scores -> softmax ->
// values, which three warps a scheduler do not hide: fixed latencies, and the ALU (44 %) and
// FMA (39 %) pipes in bursts.  Of an earlier version's 111 us the scores were 31, the values 26.
// Two CTAs an SM with rings of eight pages and four with rings of three were no faster, nor was
// a loop over page pairs; five stages cost 4 us with f32 outputs.
constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = 32 * kAttnWarps;
constexpr int kStages = 4;  // even: pages are asked for in pairs (six do not fit three CTAs)
constexpr int kRows = 8;
constexpr int kCtasPerSm = 3;
constexpr int kMaxCtas = 512;
constexpr unsigned kArrive = 1u << 20;  // more than CTAs
// Sequences with so many rows (queries x heads of the group) are prompt chunks.  With other chunks
// filling the GPU (16 sequences of 2000, 64/8 heads of 128) 64 rows take 83 us there, 121 here with
// bf16 outputs and 137 with f16, 48 rows 83 against 94 and 109; of 64 dims (64 sequences of 1000)
// 64 rows 150 against 154 and 180, 48 rows 150 against 118 and 139.  f16 outputs, whose queries and
// weights have 22 bits here and 11 there, stay longer: 80 rows take 83 us there, 165 here.
constexpr int kWideRowsBf16 = 64, kWideRowsF16 = 96;
// A chunk tile takes its time however few there are, so all chunks together need so many rows
// (queries x n_head).  One sequence of 4000, 64/8 heads: of 128, 2048 rows take 98 us there and
// 58 here, 4096 98 and 103; of 64, 4096 take 85 and 66, 8192 85 and 121.
constexpr int64_t kWideTotal128 = 4096, kWideTotal64 = 6144;
// What a unit costs beside its pages (queries, joins), in pages.  In an earlier version 8 took
// 106 us for the first of the cases above and 74 for the second, 16 104 and 72, 24 the same.
constexpr int kUnitCost = 16;
// Units of up to so many pages are not split: the join costs 6 us (one sequence of 160 tokens:
// 7 us whole, 13 split); 32 pages took 33 us for 8 sequences of 2000 and 4 queries, 16 31.
constexpr int kWholePages = 16;

__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unf2(uint64_t a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// Nibbles 0 and 4 (ODD = false) or 1 and 5 of w as an f16 pair, odd ones times 16: c - S
// when EXACT, else the subnormals c * 2^-24.
template <bool EXACT, int S, bool ODD>
__device__ __forceinline__ uint32_t codes(uint32_t w) {
  constexpr uint32_t mask = ODD ? 0x00F000F0u : 0x000F000Fu;
  if constexpr (!EXACT) return w & mask;
  const __half2 h = as_h2(lop_and_or(w, mask, 0x64006400u));
  return as_u32(__hadd2(h, __float2half2_rn(ODD ? -1024.0f - 16 * S : -1024.0f - S)));
}

// Shared memory by 32-bit address: through a generic pointer every load would pay for the
// address space.  Volatile, since bulk copies change what lies there.
__device__ __forceinline__ void lds(uint32_t at, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
}
__device__ __forceinline__ void lds(uint32_t at, uint32_t (&v)[2]) {
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(at));
}
__device__ __forceinline__ uint32_t lds(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_half(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
  return v;
}
// NG words of a row.
template <int NG>
__device__ __forceinline__ void lds_row(uint32_t at, uint32_t (&v)[NG]) {
  if constexpr (NG == 4 || NG == 2) {
    lds(at, v);
  } else {
#pragma unroll
    for (int g = 0; g < NG; ++g) v[g] = lds(at + 4 * g);
  }
}
// D = A B (+ C), m16n8k16, f16 in, f32 out.
__device__ __forceinline__ void mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The line of work: this CTA's range of it and where that begins.
struct Place {
  int64_t total, share;
  int64_t pos, end;  // this CTA's pages
  int s;             // the sequence of the first, and
  int64_t off;       // its place among that sequence's pages
};

template <int NG, bool EXACT>
struct Attn {
  static constexpr int D = 32 * NG, PB = 20 * D;
  static constexpr int kPitch = D + 4;                          // a row of a warp's state in the join buffer
  static constexpr int kState = kRows * kPitch + 2 * kRows;     // the rows, their maxima and denominators
  static constexpr int kPart = kRows * (D + 2);
  static constexpr int kJoinBytes = kAttnWarps * kState * 4;
  static constexpr int kCols = EXACT ? 2 : 4;  // sums of a fragment: of both row halves, or as the MMA has them
  static constexpr int kSmem = kAttnWarps * kStages * PB + kJoinBytes + NG * 1024 + 4 * NG * kAttnWarps;
  const Kv4AttnArgs& a;
  uint8_t* ring;      // this warp's pages
  uint32_t ring32;
  uint64_t* bars;     // and their barriers
  float* join;        // the warps' states
  uint32_t qfrag;     // this lane's query fragments, [group][k step][lane][16 bytes]; behind them the warps' scales
  int G, lane, warp;
  int wide_rows = INT32_MAX;    // a.wide_rows where the chunks are many enough
  unsigned get = 0, phase = 0;  // the ring's next page to use, and its parity
  unsigned put_at = 0;          // the ring's next page to ask for

  // A unit that other CTAs share: CTAs c0 .. c1 hold parts of it (c0 = -1: none).
  struct Open {
    int qs, rows, kvh, row0, c0, c1, last;
  };
  // A stretch of one unit: what its sequence is, and this warp's pages in it.
  struct Seg {
    int s, qs, nq, ctx, kvh, tile;
    int cost;     // the unit's length on the line: kUnitCost + its pages
    int off, n;   // the stretch on it
    int first, mine;  // this warp's first page, and how many
    const int* table;
    int ids;      // block ids of 32 of them, a lane each
    bool bad;
  };

  __device__ int seq_info(int s, int& qs, int& nq, int& ctx, bool tell) const {
    qs = __ldg(a.q_start + s);
    nq = __ldg(a.q_start + s + 1) - qs;
    ctx = __ldg(a.ctx_len + s);
    bool bad = qs < 0 || nq < 0 || (int64_t)qs + nq > a.T || nq > a.max_q;
    if (bad) nq = 0;
    if (ctx < 0 || ctx > a.max_ctx) {
      bad |= nq > 0;
      ctx = 0;
    }
    // the wide kernel's, which leaves the telling to this one, unless it met values beyond f16
    if (nq * G >= wide_rows && !__ldg(a.redo + s)) nq = 0;
    if (bad && tell) raise_status(a.status, kDevCache);
    return kUnitCost + (ctx + kTok - 1) / kTok;
  }

  // keys that a row of the sequence sees: those before and at its position
  __device__ int seen(const Seg& g, int row) const { return max(0, g.ctx - g.nq + row / G + 1); }

  __device__ int load_ids(const Seg& g, int j) const {  // 32 of this warp's block ids from the j-th on
    return j + lane < g.mine ? __ldg(g.table + (j + lane) * kAttnWarps) : 0;
  }
  // Asks for this warp's j-th and j + 1-st pages (j even), a lane each.
  __device__ void issue(Seg& g, int j) {
    if (j >= g.mine) return;
    if ((j & 31) == 0) {
      if (j > 0) g.ids = load_ids(g, j);
      if ((unsigned)g.ids >= (unsigned)a.num_blocks) {
        g.bad = true;
        g.ids = 0;
      }
    }
    const int blk = __shfl_sync(0xffffffffu, g.ids, (j + lane) & 31);
    if (lane < 2 && j + lane < g.mine) {
      unsigned at = put_at + lane;
      if (at >= kStages) at -= kStages;
      mbar_arrive_expect_tx(bars + at, PB);
      bulk_g2s(ring + at * PB, a.pages + ((int64_t)blk * a.n_kv + g.kvh) * PB, PB, bars + at);
    }
    put_at += min(2, g.mine - j);
    if (put_at >= kStages) put_at -= kStages;
  }

  // This warp's pages of the stretch [off, off + n) of a unit's line, and the first block ids.
  __device__ void open(Seg& g) const {
    const int row0 = g.tile * kRows, rows = g.nq * G;
    const int need = (seen(g, min(row0 + kRows, rows) - 1) + kTok - 1) / kTok;
    g.first = max(0, g.off - kUnitCost) + warp;
    const int last = min(g.off + g.n - kUnitCost, need);
    g.mine = last > g.first ? (last - g.first + kAttnWarps - 1) / kAttnWarps : 0;
    g.table = a.table + (int64_t)g.s * a.max_blocks + g.first;
  }
  __device__ void begin(Seg& g) {
    g.bad = false;
    for (int j = 0; j < kStages; j += 2) issue(g, j);
  }

  __device__ void run(Place& w, Seg* next, Open* left) {
    Seg g;
    g.s = w.s;
    g.cost = seq_info(g.s, g.qs, g.nq, g.ctx, false);
    int tiles = (g.nq * G + kRows - 1) / kRows;
    int64_t unit = w.off / g.cost;  // within the sequence: kv head * tiles + tile
    g.off = (int)(w.off - unit * g.cost);
    auto locate = [&](Seg& g, int64_t pos) {
      while (unit >= (int64_t)a.n_kv * tiles) {  // on to the next sequence with queries
        unit = 0;
        ++g.s;
        g.cost = seq_info(g.s, g.qs, g.nq, g.ctx, false);
        tiles = (g.nq * G + kRows - 1) / kRows;
      }
      g.kvh = (int)(unit / tiles);
      g.tile = (int)(unit - (int64_t)g.kvh * tiles);
      g.n = (int)min((int64_t)(g.cost - g.off), w.end - pos);
    };
    locate(g, w.pos);
    open(g);
    g.ids = load_ids(g, 0);
    begin(g);
    if (threadIdx.x == 0) left[0].c0 = left[1].c0 = -1;
    for (;;) {
      const int64_t at = w.pos - g.off;  // the unit's place on the line
      w.pos += g.n;
      const bool more = w.pos < w.end;
      int ids = 0;
      if (more) {
        // the next stretch: where it lies, kept in shared memory, its first block ids and its
        // queries on their way while this one is worked on
        Seg n = g;
        n.off = 0;
        ++unit;
        locate(n, w.pos);
        open(n);
        ids = load_ids(n, 0);
        const int row = n.tile * kRows + (lane >> 2), es = a.q_dtype == 0 ? 4 : 2;
        if (row < n.nq * G && (lane & 3) * 128 < D * es) {
          const char* q = static_cast<const char*>(a.q) +
                          ((int64_t)(n.qs + row / G) * a.ldq + (int64_t)(n.kvh * G + row % G) * D) * es + (lane & 3) * 128;
          asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
        }
        if (lane == 0) *next = n;
      }
      float M, l, o[NG][4][kCols], z[4];
      pages(g, M, l, o, z);
      const Seg done = g;
      if (more) {
        __syncwarp();
        g = *next;
        g.ids = ids;
        begin(g);
      }
      finish(w, done, at, M, l, o, z, left);
      if (!more) break;
    }
    join_parts(left);
  }

  // Scores of tokens 8 u + i and 8 u + 4 + i of a page (quad lane i), in the row's scale.
  __device__ uint64_t scores(uint32_t page, int u, int kt, int qi, const uint32_t (&qm)[3]) const {
    uint32_t kw[NG], h0[NG], h1[NG], hm[2] = {0, 0};
    const uint32_t ph = page + 8 * D + 8 * u * (4 * NG);
    lds_row<NG>(page + (8 * u + kt) * (D / 2) + qi * (4 * NG), kw);
    lds_row<NG>(ph + qi * (4 * NG), h0);
    lds_row<NG>(ph + (4 + qi) * (4 * NG), h1);
    if constexpr (NG == 4) {
      lds(ph + kt * 16 + 8 * (qi & 1), hm);
    } else {
      if (2 * qi < NG) hm[0] = lds(ph + kt * (4 * NG) + 8 * qi);
      if (2 * qi + 1 < NG) hm[1] = lds(ph + kt * (4 * NG) + 8 * qi + 4);
    }
    float acc[4];
    uint32_t bm = prmt(hm[0], hm[1], 0x7632u);
    if (qi >= 2) bm = 0;
    mma0(acc, qm[0], EXACT ? qm[1] : 0u, EXACT ? qm[2] : 0u, 0u, bm, EXACT ? bm : 0u);
    uint64_t x2 = EXACT ? add2(f2(acc[0], acc[1]), f2(acc[2], acc[3])) : f2(acc[0], acc[1]);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint32_t hw = kw[g] >> 8;
      float e[4];
      uint32_t qa[4];
      lds(qfrag + g * 1024, qa);
      mma0(e, qa[0], EXACT ? qa[1] : 0u, qa[2], EXACT ? qa[3] : 0u, codes<EXACT, 0, false>(kw[g]), codes<EXACT, 0, true>(kw[g]));
      lds(qfrag + g * 1024 + 512, qa);
      mma(e, qa[0], EXACT ? qa[1] : 0u, qa[2], EXACT ? qa[3] : 0u, codes<EXACT, 0, false>(hw), codes<EXACT, 0, true>(hw));
      float d0 = __low2float(as_h2(h0[g])), d1 = __low2float(as_h2(h1[g]));
      uint64_t sum = f2(e[0], e[1]);
      if constexpr (EXACT) {
        sum = add2(sum, f2(e[2], e[3]));
      } else {
        d0 *= 16777216.0f;  // the codes' 2^-24
        d1 *= 16777216.0f;
      }
      x2 = fma2(f2(d0, d1), sum, x2);
    }
    return x2;
  }

  // o += hi C and lo C.  The tensor cores truncate their sums always towards zero, and codes
  // about 8 lean to one side: summed there, 16 pages at a time, 13000 keys came out 2e-6 off.
  // Added here, rounded, a page at a time, 4e-7, as sums in 32 bits throughout.
  __device__ static void add(float (&o)[kCols], const uint32_t (&hi)[2], const uint32_t (&lo)[2], uint32_t b0, uint32_t b1) {
    if constexpr (EXACT) {
      float t[4];
      mma0(t, hi[0], lo[0], hi[1], lo[1], b0, b1);
      const float2 sum = unf2(add2(f2(o[0], o[1]), add2(f2(t[0], t[1]), f2(t[2], t[3]))));
      o[0] = sum.x;
      o[1] = sum.y;
    } else {
      mma(o, hi[0], lo[0], hi[1], lo[1], b0, b1);
    }
  }

  // O += (p d) C and the header sums z of a page, p = ph + pl of pairs of tokens (i, i + 4) and
  // (i + 8, i + 12).
  template <bool SECOND>
  __device__ void values(uint32_t page, int r, int qi, const uint32_t (&ph)[2], const uint32_t (&pl)[2],
                         float (&o)[NG][4][kCols], float (&z)[4]) const {
    // ---- sums of p times what a group's codes add to: its minimum, or, about code 8, the
    // middle m + 8 d.  The middles lie around zero, where the sums of the minima and of the
    // steps would each grow and then cancel; column g takes the middle as f16, column 4 + g
    // the rest (two-sum).  On a second attempt a 16th where m + 8 d would pass f16's range.
    const uint32_t vh = page + 18 * D;
    {
      const int g = min(r & 3, NG - 1);
      const uint32_t at = vh + 4 * (qi * NG + g);
      uint32_t b[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t w0 = lds(at + 32 * NG * u), w1 = lds(at + 32 * NG * u + 16 * NG);
        b[u] = prmt(w0, w1, 0x7632u);
        if constexpr (EXACT) {
          __half2 s8 = __float2half2_rn(8.0f), s1 = __float2half2_rn(1.0f);
          if constexpr (SECOND) {
            s1 = __high2half2(as_h2(lds(scales_at() + 4 * g)));
            s8 = __hmul2_rn(s8, s1);
          }
          const __half2 x = __hmul2_rn(as_h2(prmt(w0, w1, 0x5410u)), s8), y = __hmul2_rn(as_h2(b[u]), s1);
          const __half2 sum = __hadd2_rn(x, y), v = __hsub2_rn(sum, x);
          const __half2 rest = __hadd2_rn(__hsub2_rn(x, __hsub2_rn(sum, v)), __hsub2_rn(y, v));
          b[u] = as_u32(r < 4 ? sum : rest);
        }
      }
      if constexpr (EXACT) {
        float t[4];
        mma0(t, ph[0], pl[0], ph[1], pl[1], b[0], b[1]);
        if constexpr (SECOND) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (lds(scales_at() + 4 * min(2 * (qi & 1) + (c & 1), NG - 1)) >> 16 != 0x3c00u) t[c] *= 16.0f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) z[c] += t[c];
      } else {
        mma(z, ph[0], pl[0], ph[1], pl[1], b[0], b[1]);
      }
    }
    // ---- O += (p d) C: pairs of tokens (i, i + 4) and (i + 8, i + 12)
    uint32_t vd[4][NG], vw[4][(NG + 1) / 2];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t vr = page + 10 * D + (4 * c + qi) * (D / 2);
      lds_row<NG>(vh + (4 * c + qi) * (4 * NG), vd[c]);
      if constexpr (NG == 4) {
        lds(vr + (((2 * r) ^ (8 * (qi >> 1))) << 2), vw[c]);
      } else {
        if constexpr (NG >= 2) vw[c][0] = lds(vr + 4 * r);
        if constexpr (NG & 1) vw[c][NG / 2] = lds_half(vr + ((NG - 1) * 8 + r) * 2);
      }
    }
    // one for all groups, or one each
    uint32_t scales[NG] = {};
    if constexpr (SECOND)
      lds_row<NG>(scales_at(), scales);
    else if constexpr (EXACT)
      scales[0] = lds(scales_at());
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        __half2 d = as_h2(prmt(vd[2 * u][g], vd[2 * u + 1][g], 0x5410u));
        if constexpr (SECOND || EXACT) d = __hmul2(d, __low2half2(as_h2(scales[SECOND ? g : 0])));
        const __half2 p = as_h2(ph[u]), h = __hmul2(p, d);
        hi[u] = as_u32(h);
        lo[u] = EXACT ? as_u32(__hfma2(as_h2(pl[u]), d, __hfma2(p, d, __hneg2(h)))) : 0u;
      }
      const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
      const uint32_t b0 = prmt(vw[0][g / 2], vw[1][g / 2], sel), b1 = prmt(vw[2][g / 2], vw[3][g / 2], sel);
      add(o[g][0], hi, lo, codes<EXACT, 8, false>(b0), codes<EXACT, 8, false>(b1));
      add(o[g][1], hi, lo, codes<EXACT, 8, true>(b0), codes<EXACT, 8, true>(b1));
      add(o[g][2], hi, lo, codes<EXACT, 8, false>(b0 >> 8), codes<EXACT, 8, false>(b1 >> 8));
      add(o[g][3], hi, lo, codes<EXACT, 8, true>(b0 >> 8), codes<EXACT, 8, true>(b1 >> 8));
    }
  }

  // Steps are lifted by a power of two, at most 2^15: the rest of p d lies on f16's grid of 2^-24,
  // which with p d of 2^-7 was 4e-6 of it.  The largest step of a warp's first page that holds any
  // (of the keys that some row sees) goes to 2^-4 at least, and later ones may be 256 times as
  // large; on the second attempt, with p at most 1, every group of every page goes to 2^14 where
  // 2^15 suffice.
  // A warp's words, f16 pairs: 2^lift of a group's steps, and what its middles are multiplied by.
  // In shared memory, since the loop over the pages has no register left.
  __device__ uint32_t scales_at() const { return qfrag - 16 * lane + NG * 1024 + 4 * NG * warp; }
  __device__ int lift_now(int g) const { return (int)(lds(scales_at() + 4 * g) >> 10 & 31u) - 15; }
  __device__ void set_scales(int g, uint32_t factors) const {
    if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(scales_at() + 4 * g), "r"(factors) : "memory");
  }
  // False: the page holds no step above zero.
  __device__ bool first_scales(uint32_t vh, int keys) const {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < (16 * NG + 31) / 32; ++i) {
      const int at = 32 * i + lane;
      const uint32_t d = at < NG * min(kTok, keys) ? lds(vh + 4 * at) & 0x7fffu : 0u;
      if (d < 0x7c00u) most = max(most, d);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (!most) return false;
    const uint32_t by = (uint32_t)max(0, min(15, -4 - ilogbf(f16_bits_to_f32(most))));
#pragma unroll
    for (int g = 0; g < NG; ++g) set_scales(g, (by + 15) << 10 | 0x3c000000u);
    __syncwarp();
    return true;
  }
  // The second attempt's, and the sums so far in their terms.
  __device__ void page_scales(uint32_t vh, int keys, float (&o)[NG][4][kCols]) const {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint32_t h = lane < min(kTok, keys) ? lds(vh + 4 * (lane * NG + g)) & 0x7fff7fffu : 0u;
      const bool number = (h & 0x7fffu) < 0x7c00u && h >> 16 < 0x7c00u;
      const float d = f16_bits_to_f32(__reduce_max_sync(0xffffffffu, number ? h & 0xffffu : 0u));
      const float m = f16_bits_to_f32(__reduce_max_sync(0xffffffffu, number ? h >> 16 : 0u));
      const int now = lift_now(g), to = d > 0.0f ? min(now, max(0, 14 - ilogbf(d))) : now;
      if (to < now) {
        const float f = pow2(to - now);
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int c = 0; c < kCols; ++c) o[g][p][c] *= f;
      }
      __syncwarp();
      set_scales(g, (uint32_t)(to + 15) << 10 | (fmaf(8.0f, d, m) > 32768.0f ? 0x2c000000u : 0x3c000000u));
    }
    __syncwarp();
  }

  // A page with keys that some row does not see: such keys weigh nothing, whatever they hold,
  // so V headers that are not finite are zeroed, since 0 * NaN would reach every row of the
  // MMA; a row that does see such a header gets its group's NaN here.  Headers of keys that no row
  // of the tile sees are zeroed too: the steps are scaled by the others'.
  __device__ void sanitise(uint32_t vh, int key, int most, int limit, float (&o)[NG][4][kCols]) const {
    uint64_t nan_at = 0;
#pragma unroll
    for (int i = 0; i < (16 * NG + 31) / 32; ++i) {
      const int at = 32 * i + lane;
      bool no = false;
      if (at < 16 * NG) {
        const uint32_t h = lds(vh + 4 * at);
        no = (h & 0x7c00u) == 0x7c00u || (h & 0x7c000000u) == 0x7c000000u;
        if (no || key + at / NG >= most) asm volatile("st.shared.u32 [%0], %1;" ::"r"(vh + 4 * at), "r"(0u) : "memory");
      }
      nan_at |= (uint64_t)__ballot_sync(0xffffffffu, no) << (32 * i);
    }
    if (nan_at) {
      const int cnt = max(0, min(kTok, limit - key));
      for (int t = 0; t < cnt; ++t)
#pragma unroll
        for (int g = 0; g < NG; ++g)
          if ((nan_at >> (t * NG + g)) & 1)
#pragma unroll
            for (int p = 0; p < 4; ++p) o[g][p][0] = o[g][p][1] = NAN;
    }
    // the next bulk copy into this page follows these stores
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
  }

  // One attempt: p = 2^(x - max + headroom) right after a maximum is set, which stays until a score
  // would pass 2^growth.
  template <bool SECOND>
  __device__ void walk(Seg& sg, const uint32_t (&qm)[3], float rowmul, int least, int most, int limit, float& M, float& l,
                       float (&o)[NG][4][kCols], float (&z)[4]) {
    const int mine = sg.mine, first = sg.first;
    const int r = lane >> 2, qi = lane & 3;
    const int kt = ((r & 1) << 2) | (r >> 1);  // token of S column r: columns 2 i, 2 i + 1 are tokens i, i + 4
    constexpr float headroom = SECOND ? 0.0f : 8.0f, growth = SECOND ? 0.0f : 12.0f;
    __syncwarp();
#pragma unroll
    for (int g = 0; g < NG; ++g) set_scales(g, SECOND || EXACT ? 0x3c007800u : 0x3c003c00u);  // 2^15 or 1, and 1
    __syncwarp();
    bool scaled = false;
    M = -1e30f;
    l = 0.0f;
#pragma unroll
    for (int c = 0; c < 4; ++c) z[c] = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[g][p][c] = 0.0f;
    for (int j = 0; j < mine; ++j) {
      mbar_wait_bounded(bars + get, phase, a.status);
      const uint32_t page = ring32 + get * PB;
      if (++get == kStages) {
        get = 0;
        phase ^= 1;
      }
      const int key = (first + j * kAttnWarps) * kTok;
      // ---- scores
      float x[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) *reinterpret_cast<float2*>(x[u]) = unf2(scores(page, u, kt, qi, qm));
      if (key + kTok > least) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (key + 8 * u + 4 * c + qi >= limit) x[u][c] = -INFINITY;
        sanitise(page + 18 * D, key, most, limit, o);
      }
      // ---- running softmax
      float mx = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1])) * rowmul;
      if (__any_sync(0xffffffffu, mx > M + growth)) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (mx > M + growth) {
          const float to = mx - headroom, f = ex2(M - to);
          M = to;
          l *= f;
#pragma unroll
          for (int c = 0; c < 4; ++c) z[c] *= f;
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
              for (int c = 0; c < kCols; ++c) o[g][p][c] *= f;
        }
      }
      uint32_t ph[2], pl[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float p0 = ex2(fmaf(x[u][0], rowmul, -M)), p1 = ex2(fmaf(x[u][1], rowmul, -M));
        l += p0 + p1;
        const __half2 h = __floats2half2_rn(p0, p1);
        ph[u] = as_u32(h);
        pl[u] = 0;
        if constexpr (EXACT) {
          const float2 f = __half22float2(h);
          pl[u] = as_u32(__floats2half2_rn(p0 - f.x, p1 - f.y));
        }
      }
      if constexpr (SECOND)
        page_scales(page + 18 * D, most - key, o);
      else if (EXACT && !scaled)
        scaled = first_scales(page + 18 * D, most - key);
      values<SECOND>(page, r, qi, ph, pl, o, z);
      __syncwarp();
      if (j & 1) issue(sg, j + kStages - 1);  // the two pages just used
    }
  }

  // This warp's pages of the stretch: per row the running maximum M and sum l, and in
  // fragments the products o and the header sums z.
  __device__ void pages(Seg& sg, float& M, float& l, float (&o)[NG][4][kCols], float (&z)[4]) {
    const int qs = sg.qs, kvh = sg.kvh, mine = sg.mine;
    const int row0 = sg.tile * kRows, rows = sg.nq * G;
    const int least = seen(sg, row0), most = seen(sg, min(row0 + kRows, rows) - 1);
    // ---- queries: lane (row r, quad lane i) holds dims 8 i .. 8 i + 7 of every group
    const int r = lane >> 2, qi = lane & 3;
    const int row = row0 + r;
    const bool live = row < rows;
    const int limit = live ? seen(sg, row) : most;
    uint32_t qm[3] = {};
    float rowmul;
    {
      float x[NG][8], qsum[NG];
      const int64_t base = live ? (int64_t)(qs + row / G) * a.ldq + (int64_t)(kvh * G + row % G) * D : 0;
      float mx = 0.0f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float sum = 0.0f;
        const int64_t at = base + 32 * g + 8 * qi;
        if (a.q_wide) {
          *reinterpret_cast<float4*>(x[g]) = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at));
          *reinterpret_cast<float4*>(x[g] + 4) = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at + 4));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[g][e] = load_as_f32(a.q, a.q_dtype, at + e);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = live ? x[g][e] * a.scale * 1.4426950408889634f : 0.0f;
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
      // 2^k brings the row's largest into [2^6, 2^7): the group sums fit f16 too
      int k = 0;
      if (mx > 0.0f && mx < INFINITY) k = max(-90, min(90, 6 - ilogbf(mx)));
      const float up = pow2(k);
      rowmul = pow2(-k);
      auto split = [](float v0, float v1, uint32_t& hi, uint32_t& lo) {
        const __half2 h = __floats2half2_rn(v0, v1);
        const float2 f = __half22float2(h);
        hi = as_u32(h);
        lo = as_u32(__floats2half2_rn(v0 - f.x, v1 - f.y));
      };
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          uint32_t frag[4];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int e = 2 * st + b;  // nibbles e and e + 4; odd ones carry a factor 16
            const float f = b ? up * 0.0625f : up;
            split(x[g][e] * f, x[g][e + 4] * f, frag[2 * b], frag[2 * b + 1]);
          }
          // every warp has the same queries and writes the same words
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(qfrag + (g * 2 + st) * 512), "r"(frag[0]), "r"(frag[1]),
                       "r"(frag[2]), "r"(frag[3])
                       : "memory");
        }
      // the sums of groups 2 i and 2 i + 1, against the minima
      float q0 = 0.0f, q1 = 0.0f;
#pragma unroll
      for (int g = 0; g < NG; ++g)
        if (g / 2 == qi) {
          if (g & 1)
            q1 = qsum[g] * up;
          else
            q0 = qsum[g] * up;
        }
      // (three parts: they meet minima of several steps, and their error would not average out)
      split(q0, q1, qm[0], qm[1]);
      if constexpr (EXACT) {
        const float2 h = __half22float2(as_h2(qm[0])), m = __half22float2(as_h2(qm[1]));
        qm[2] = as_u32(__floats2half2_rn((q0 - h.x) - m.x, (q1 - h.y) - m.y));
      }
    }

    walk<false>(sg, qm, rowmul, least, most, limit, M, l, o, z);
    if (mine == 0) return;
    // if p d or a middle left f16's range after all (a step above 16, or 256 times the first page's),
    // the pages are read once more with p at most 1 and the scales found for every page
    float probe = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int c = 0; c < kCols; ++c) probe = fmaf(o[g][p][c], 0.0f, probe);
#pragma unroll
    for (int c = 0; c < 4; ++c) probe = fmaf(z[c], 0.0f, probe);
    if (!__any_sync(0xffffffffu, probe != 0.0f)) return;  // NaN where anything was not finite
    // from the start: the ring is empty, and an odd number of pages may have used it
    sg.ids = load_ids(sg, 0);
    for (int j = 0; j < kStages; j += 2) issue(sg, j);
    walk<true>(sg, qm, rowmul, least, most, limit, M, l, o, z);
  }

  // Joins the warps' states into the output or, where the unit goes on in other CTAs, into a
  // part of it.
  __device__ void finish(const Place& w, const Seg& sg, int64_t begin, float M, float l, const float (&o)[NG][4][kCols],
                         const float (&z)[4], Open* left) {
    const int r = lane >> 2, qi = lane & 3;
    const int qs = sg.qs, kvh = sg.kvh, row0 = sg.tile * kRows, rows = sg.nq * G;
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (__any_sync(0xffffffffu, sg.bad)) {  // a block id outside the pool: no number stands for these rows
      if (lane == 0) raise_status(a.status, kDevCache);
      l = NAN;
    }
    {
      float* out = join + warp * kState + r * kPitch + 8 * qi;
      const float z0 = z[0] + z[2], z1 = z[1] + z[3];  // quad lanes 0, 1: middles or minima; 2, 3: their rests
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int from = (lane & ~3) + g / 2;
        const float zm = __shfl_sync(0xffffffffu, (g & 1) ? z1 : z0, from);
        const float zd = __shfl_sync(0xffffffffu, (g & 1) ? z1 : z0, from + 2);
        const float zz = EXACT ? zm + zd : zm;
        const float down = pow2((EXACT ? 0 : 24) - lift_now(g));
        float v[8];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const float f = down * ((p & 1) ? 0.0625f : 1.0f);  // the odd nibbles' 16
          v[p] = fmaf(o[g][p][0] + (EXACT ? 0.0f : o[g][p][kCols - 2]), f, zz);
          v[4 + p] = fmaf(o[g][p][1] + (EXACT ? 0.0f : o[g][p][kCols - 1]), f, zz);
        }
        *reinterpret_cast<float4*>(out + 32 * g) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(out + 32 * g + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
      if (qi == 0) {
        join[warp * kState + kRows * kPitch + r] = M;
        join[warp * kState + kRows * kPitch + kRows + r] = l;
      }
    }
    __syncthreads();
    const int tid = threadIdx.x;
    const int cta = blockIdx.x;
    const int c0 = (int)(begin / w.share), c1 = (int)((begin + sg.cost - 1) / w.share);
    const Open u{qs, rows, kvh, row0, c0, c1, 0};
    if (c0 != c1 && tid == 0) left[c0 == cta ? 1 : 0] = u;
    for (int e = tid; e < kRows * D / 4; e += kAttnThreads) {
      const int rr = e / (D / 4), d = 4 * (e - rr * (D / 4));
      const float* ml = join + kRows * kPitch + rr;
      float m = ml[0];
#pragma unroll
      for (int k = 1; k < kAttnWarps; ++k) m = fmaxf(m, ml[k * kState]);
      float ls = 0.0f;
      float4 os = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < kAttnWarps; ++k) {
        const float f = ex2(ml[k * kState] - m);
        const float4 v = *reinterpret_cast<const float4*>(join + k * kState + rr * kPitch + d);
        ls = fmaf(ml[k * kState + kRows], f, ls);
        os = make_float4(fmaf(v.x, f, os.x), fmaf(v.y, f, os.y), fmaf(v.z, f, os.z), fmaf(v.w, f, os.w));
      }
      if (c0 == c1) {
        put(u, rr, d, os, ls);
      } else {
        float* p = part(u, cta);
        *reinterpret_cast<float4*>(p + rr * D + d) = os;
        if (d == 0) {
          p[kRows * D + rr] = m;
          p[kRows * D + kRows + rr] = ls;
        }
      }
    }
    __syncthreads();  // the join buffer is used again
  }

  // a part: [8][D] sums, [8] maxima, [8] denominators
  __device__ float* part(const Open& u, int c) const { return a.part + ((int64_t)c * 2 + (c == u.c0 ? 1 : 0)) * kPart; }
  __device__ void put(const Open& u, int rr, int d, float4 v, float ls) const {
    const int rw = u.row0 + rr;
    if (rw >= u.rows) return;
    const float f = ls == 0.0f ? 0.0f : 1.0f / ls;
    if (ls == 0.0f) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int64_t at = (int64_t)(u.qs + rw / G) * a.ldo + (int64_t)(u.kvh * G + rw % G) * D + d;
    if (a.o_wide && a.o_dtype == 0) {
      *reinterpret_cast<float4*>(static_cast<float*>(a.o) + at) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
    } else {
      store_from_f32(a.o, a.o_dtype, at, v.x * f);
      store_from_f32(a.o, a.o_dtype, at + 1, v.y * f);
      store_from_f32(a.o, a.o_dtype, at + 2, v.z * f);
      store_from_f32(a.o, a.o_dtype, at + 3, v.w * f);
    }
  }

  // The units that this CTA shares (the one begun before it, the one it leaves open): the last
  // CTA of a unit to come here joins its parts, in CTA order.  Once, at the end of the CTA's
  // stretch: the fence and the atomics cost 3 us a time.  A unit's CTAs add a whole kArrive in all
  // to its word, which only the last to arrive fills up.  Nobody clears it: calls that overlapped
  // spoil one another's parts, but leave whole multiples behind, and later calls count as ever.
  __device__ void join_parts(Open* left) {
    const int tid = threadIdx.x;
    if (tid < 2) {
      Open& u = left[tid];
      u.last = 0;
      if (u.c0 >= 0) {
        __threadfence();
        const unsigned add = (int)blockIdx.x == u.c0 ? kArrive - (unsigned)(u.c1 - u.c0) : 1u;
        u.last = (atomicAdd(a.count + u.c0, add) + add) % kArrive == 0;
        __threadfence();
      }
    }
    __syncthreads();
    for (int i = 0; i < 2; ++i) {
      if (!left[i].last) continue;
      const Open u = left[i];
      // a thread takes four dims of a row; the loads of eight parts do not wait for one another
      for (int e = tid; e < kRows * D / 4; e += kAttnThreads) {
        const int er = e / (D / 4), d = 4 * (e - er * (D / 4));
        float m = -1e30f, ls = 0.0f;
        float4 os = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int c = u.c0; c <= u.c1; c += 8) {
          float mc[8], lc[8];
          float4 v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const bool in = c + k <= u.c1;
            const float* p = part(u, in ? c + k : c);
            mc[k] = in ? __ldcg(p + kRows * D + er) : -1e30f;
            lc[k] = in ? __ldcg(p + kRows * D + kRows + er) : 0.0f;
            v[k] = in ? __ldcg(reinterpret_cast<const float4*>(p + er * D + d)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          }
          float top = m;
#pragma unroll
          for (int k = 0; k < 8; ++k) top = fmaxf(top, mc[k]);
          const float f = ex2(m - top);
          m = top;
          ls *= f;
          os = make_float4(os.x * f, os.y * f, os.z * f, os.w * f);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float w = ex2(mc[k] - top);
            ls = fmaf(lc[k], w, ls);
            os = make_float4(fmaf(v[k].x, w, os.x), fmaf(v[k].y, w, os.y), fmaf(v[k].z, w, os.z), fmaf(v[k].w, w, os.w));
          }
        }
        put(u, er, d, os, ls);
      }
    }
  }
};

template <int NG, bool EXACT>
__global__ void __launch_bounds__(kAttnThreads, kCtasPerSm) kv4_attn_kernel(const Kv4AttnArgs a) {
  constexpr int D = 32 * NG, PB = 20 * D;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kAttnWarps][kStages];
  __shared__ int64_t sums[kAttnWarps];
  __shared__ Place place;
  __shared__ typename Attn<NG, EXACT>::Seg next[kAttnWarps];
  __shared__ typename Attn<NG, EXACT>::Open left[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Attn<NG, EXACT> at{a, smem + warp * (kStages * PB), smem_u32(smem + warp * (kStages * PB)), bars[warp], reinterpret_cast<float*>(smem + kAttnWarps * kStages * PB),
                     smem_u32(smem + kAttnWarps * kStages * PB + Attn<NG, EXACT>::kJoinBytes) + 16 * lane,
                     a.n_head / a.n_kv, lane, warp};
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[warp][i], 1);
    fence_mbar_init();
  }
  // ---- the line of work and this CTA's place on it
  const int per = (a.S + kAttnThreads - 1) / kAttnThreads;
  const int s0 = min(a.S, tid * per), s1 = min(a.S, s0 + per);
  if (a.wide_rows < INT32_MAX) {
    int64_t all = 0;
    for (int s = s0; s < s1; ++s) all += chunk_rows(a, s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) sums[warp] = all;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int k = 0; k < kAttnWarps; ++k) all += sums[k];
    __syncthreads();
    if (all * a.n_kv >= a.wide_total) at.wide_rows = a.wide_rows;
  }
  auto cost = [&](int s) -> int64_t {
    int qs, nq, ctx;
    const int unit = at.seq_info(s, qs, nq, ctx, blockIdx.x == 0);
    return (int64_t)a.n_kv * ((nq * at.G + kRows - 1) / kRows) * unit;
  };
  int64_t mine = 0;
  for (int s = s0; s < s1; ++s) mine += cost(s);
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int k = 0; k < kAttnWarps; ++k) {
    if (k < warp) inc += sums[k];
    total += sums[k];
  }
  const int64_t share = max((int64_t)a.min_share, (total + gridDim.x - 1) / gridDim.x);
  const int64_t pos = share * blockIdx.x;
  if (pos >= total) return;
  int64_t before = inc - mine;
  if (pos >= before && pos < inc)
    for (int s = s0; s < s1; ++s) {
      const int64_t c = cost(s);
      if (pos < before + c) {
        place = Place{total, share, pos, min(total, pos + share), s, pos - before};
        break;
      }
      before += c;
    }
  __syncthreads();
  Place w = place;
  at.run(w, next + warp, left);
}

template <int NG, bool EXACT>
cudaError_t attn_launch(Kv4AttnArgs a, int sm_count, cudaStream_t st) {
  constexpr int smem = Attn<NG, EXACT>::kSmem;
  static std::atomic<uint64_t> configured{0};
  cudaError_t e = configure_once(kv4_attn_kernel<NG, EXACT>, smem, configured);
  if (e != cudaSuccess) return e;
  // never more CTAs than the bounds on the lengths can give work to
  const int64_t tiles = ((int64_t)a.max_q * (a.n_head / a.n_kv) + kRows - 1) / kRows;
  const double most = (double)a.S * a.n_kv * tiles * (kUnitCost + (a.max_ctx + kTok - 1) / kTok);
  const double want = most / a.min_share + 1.0;
  const unsigned grid = (unsigned)std::min<double>(want, (double)std::min(kMaxCtas, kCtasPerSm * sm_count));
  count_launch();
  kv4_attn_kernel<NG, EXACT><<<grid, kAttnThreads, smem, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_plan(const int* want, int S, int* length, int* table, int max_blocks, int* free_list,
                           int* free_count, int num_blocks, int* q_start, int* tok_seq, int* tok_pos, int* tok_slot,
                           int max_tokens, int* status, cudaStream_t st) {
  PlanArgs a{want, S, length, table, max_blocks, free_list, free_count, num_blocks, q_start, tok_seq, tok_pos,
             tok_slot, max_tokens, status};
  const size_t smem = (size_t)(4 * S + 3) * sizeof(int);
  static std::atomic<uint64_t> configured{0};
  cudaError_t e = configure_once(kv_plan_kernel, (4 * kPlanMaxSeqs + 3) * (int)sizeof(int), configured);
  if (e != cudaSuccess) return e;
  const int64_t items = (q_start ? max_tokens : 0) + (int64_t)S;
  const unsigned ctas = items > 4 * kPlanThreads ? 8 : 1;
  count_launch();
  if (ctas == 1) {
    kv_plan_kernel<<<1, kPlanThreads, smem, st>>>(a);
    return cudaGetLastError();
  }
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
  return cudaLaunchKernelEx(&cfg, kv_plan_kernel, a);
}

cudaError_t launch_rope_kv4(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                            int x_dtype, int64_t T, int n_head, int n_kv, int head_dim, int rot_dim,
                            const double* inv_freq, const int* tok_pos, const int* tok_slot, uint8_t* pages,
                            int num_blocks, float* q_out, int sm_count, int* status, cudaStream_t st) {
  const int q_wide = rot_dim == head_dim && ldq % 4 == 0 && reinterpret_cast<uintptr_t>(q) % (x_dtype == 0 ? 16 : 8) == 0 &&
                     reinterpret_cast<uintptr_t>(q_out) % 16 == 0;
  AppendArgs a{q, k, v, ldq, ldk, ldv, x_dtype, q_wide, n_head, n_kv, rot_dim, inv_freq, tok_pos, tok_slot, pages,
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

cudaError_t launch_kv4_attention(const Kv4Attention& c) {
  const int wide = c.q_dtype == 0 && c.ldq % 4 == 0 && reinterpret_cast<uintptr_t>(c.q) % 16 == 0;
  const int wide_o = c.ldo % (c.o_dtype == 0 ? 4 : 8) == 0 && reinterpret_cast<uintptr_t>(c.o) % 16 == 0;
  Kv4AttnArgs a{c.q, c.q_dtype, wide, c.ldq, (int)c.T, c.n_head, c.n_kv, c.scale, c.q_start, c.ctx_len, c.S, c.block_table,
                c.max_blocks, c.max_q, c.max_ctx, c.pages, c.num_blocks, c.o, c.o_dtype, wide_o,
                c.ldo, INT32_MAX, c.head_dim == 128 ? kWideTotal128 : kWideTotal64, c.redo, kUnitCost + std::min(kWholePages, (c.max_ctx + kTok - 1) / kTok), c.ws, c.count, c.status};
  const bool exact = c.o_dtype != 2;  // bf16 rounds by 2^-9 what the other form rounds by 2^-11
  const int64_t rows = (int64_t)c.max_q * (c.n_head / c.n_kv);
  const int wide_rows = c.o_dtype == 2 ? kWideRowsBf16 : kWideRowsF16;
  // outputs written over the queries are the line kernel's: it may have to read a chunk's again
  auto bytes = [&](int dt, int64_t ld) { return ((c.T - 1) * ld + (int64_t)c.n_head * c.head_dim) * (dt == 0 ? 4 : 2); };
  const uintptr_t q0 = reinterpret_cast<uintptr_t>(c.q), o0 = reinterpret_cast<uintptr_t>(c.o);
  const bool apart = q0 + bytes(c.q_dtype, c.ldq) <= o0 || o0 + bytes(c.o_dtype, c.ldo) <= q0;
  if (c.o_dtype != 0 && (c.head_dim == 64 || c.head_dim == 128) && rows >= wide_rows && c.T * c.n_head >= a.wide_total &&
      apart && c.S <= c.redo_words) {
    a.wide_rows = wide_rows;
    cudaError_t e = cudaMemsetAsync(c.redo, 0, (size_t)c.S * sizeof(int), c.stream);
    if (e == cudaSuccess) e = launch_kv4_wide(a, c.head_dim, c.stream);
    if (e != cudaSuccess) return e;  // what follows is for the others, if any
  }
  switch (c.head_dim / 32) {
    case 1: return exact ? attn_launch<1, true>(a, c.sm_count, c.stream) : attn_launch<1, false>(a, c.sm_count, c.stream);
    case 2: return exact ? attn_launch<2, true>(a, c.sm_count, c.stream) : attn_launch<2, false>(a, c.sm_count, c.stream);
    case 3: return exact ? attn_launch<3, true>(a, c.sm_count, c.stream) : attn_launch<3, false>(a, c.sm_count, c.stream);
    default: return exact ? attn_launch<4, true>(a, c.sm_count, c.stream) : attn_launch<4, false>(a, c.sm_count, c.stream);
  }
}

size_t kv4_attention_ws_bytes(int sm_count) { return (size_t)kCtasPerSm * sm_count * 2 * kRows * (128 + 2) * sizeof(float); }
size_t kv4_attention_count_bytes(int sm_count) { return (size_t)kCtasPerSm * sm_count * sizeof(unsigned); }

}  // namespace rtd
