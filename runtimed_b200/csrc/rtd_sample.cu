// rtd_sample.cu -- temperature, top-k, top-p and min-p sampling of a row of logits from a
// given random number, sm_100a.
//
// A cluster of CTAs serves a row.  Nothing is sorted: each filter is a threshold (a value,
// and how many of the entries equal to it stay, lowest index first), found by histograms
// over the row, and the pick is a prefix sum in index order over what the thresholds keep.
//
// Weights are whole numbers, w = rint(2^44 exp((x - max) / t)), formed in 64 bits: sums of
// whole numbers do not depend on their order, so the atomics and the split over CTAs
// cannot change a result, and every CTA of the cluster decides alike from the same
// totals.  2^44 leaves room for 2^19 entries and drops what is below 2^-45 of the largest.
//
// A histogram over 1024 equal steps of (max - x) / t spreads any row's upper end over many
// bins.  With top-k, the bins that hold the k largest usually hold few more: they are
// gathered into one CTA, which sorts them and decides alone.  Where they are too many, and
// for a nucleus over the whole row, a select finds the exact threshold: the bin where the
// count or weight is reached, then, if at most 255 entries share it, their ranks, else splits
// of it by the bits of the value's order map.
//
// Bound: for few rows the latency of the passes (three to five, the first from memory, the
// others from L1) and of a cluster barrier after each: 1 row of 151936 with top-k 50 and top-p
// 11 us.  64 rows of 152064 f32 with top-p alone take 74 us, of which in one row 4 the
// maximum (at the memory's rate), 11 the histogram's shared-memory atomics, 18 the 64-bit
// exponentials, and the steps between the passes 2 to 4 each.  200 rows in bf16 with every
// filter take 27 us, 8 of them the maximum.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "rtd_common.cuh"
#include "rtd_kernels.h"

namespace rtd {
namespace {

namespace cg = cooperative_groups;

constexpr int kBins = 1024;
constexpr int kList = 255;   // entries of a bin that are ranked against one another
constexpr int kLanes = 4;    // threads that share an entry's comparisons
constexpr int kCand = 1024;  // candidates that one CTA ranks
constexpr int kMaxRanks = 8;
constexpr int kNT = 512;
constexpr int kWarps = kNT / 32;
constexpr int kFar = 4;  // a chunk: so many of a lane's 16-byte vectors
constexpr int kResident = 296;  // CTAs: more rows than fill the SMs get fewer CTAs each
constexpr double kUnit = 17592186044416.0;  // 2^44

struct SampleArgs {
  const void* x;
  int64_t ldx;
  int V;
  int per_warp;  // entries of a warp, a multiple of 256
  int wide;      // rows on 16-byte boundaries
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int* ids;
};

template <int DT>
__device__ __forceinline__ float load(const void* p, int64_t i) {
  if constexpr (DT == 0) return static_cast<const float*>(p)[i];
  if constexpr (DT == 1) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Order map onto unsigned: larger value, larger key; -0 as +0; NaN below everything.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

struct Shared {
  uint32_t cnt[2][kBins], lo[2][kBins], hi[2][kBins];
  uint64_t cand[kCand];  // candidates of the row (in rank 0): key << 32 | ~index
  uint32_t keys[kCand];  // a bin's entries
  uint64_t weights[kCand];
  uint32_t list[kList + 1];
  uint64_t red[32];
  uint64_t red2[32];
  uint64_t xch[3][2];  // values for the other CTAs, a slot per exchange
  uint32_t cand_n, list_n, first;
  uint32_t found, found_cnt;
  uint64_t found_above, found_total;
  double pow2[64];            // 2^(44 - i / 64)
  float queue[kWarps][64];     // kept values waiting for a full warp of exponentials
  uint16_t hits[kWarps][64];   // chunks waiting to be looked at
  __nv_bfloat16 marks[];       // the chunks' maxima, rounded up
};

template <int DT>
struct Row {
  static constexpr int kPer = kBins / kNT;       // bins, or candidates, of a thread
  static constexpr int kVec = DT == 0 ? 4 : 8;  // entries of 16 bytes
  static constexpr int kAhead = DT == 0 ? 4 : 2;  // loads in flight where every entry is looked at
  const SampleArgs& a;
  Shared& sm;
  cg::cluster_group cluster;
  const void* x;
  int rank, ranks, tid, lane, warp, w0, w1;
  float top, c;      // the row's maximum; histogram steps per unit of (max - x)
  double topd, scale;  // log2(e) / t
  uint32_t sk;       // kept: keys above sk ...
  uint64_t sm_ties;  // ... and the first sm_ties entries with key sk
  int buf;

  // The weight of a value, rint(2^44 2^-y) with y = (max - v) log2(e) / t, in 64 bits:
  // 2^(44 - i / 64) e^(-r ln 2) with i / 64 the 64th nearest y, the first from a table, the
  // second by its Taylor series for |r| <= 2^-7, whose sixth term is below 2^-54.  40 cycles a
  // warp, against 56 with exp().  From y = 46 on (-inf and NaN too) it is 0, without a branch.
  __device__ uint64_t weight(float v) const {
    const double y = fmin((topd - (double)v) * scale, 47.0);
    const double magic = 6755399441055744.0;  // 1.5 * 2^52
    const double at = fma(y, 64.0, magic);
    const int i = __double2loint(at);
    const double r = fma(at - magic, -0.015625, y) * -0.69314718055994530942;
    double e = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    e = fma(r, e, 1.0 / 6.0);
    e = fma(r, e, 0.5);
    e = fma(r, e, 1.0);
    e = fma(r, e, 1.0);
    const double f = sm.pow2[i & 63];
    const double w = fma(__hiloint2double(__double2hiint(f) - ((i >> 6) << 20), __double2loint(f)), e, 4503599627370496.0);
    return (uint64_t)__double_as_longlong(w) & 0xFFFFFFFFFFFFFull;  // rounded, in the mantissa under 2^52
  }
  // miss(value) at least for the entries that are not below `low`, and f(value, weight) for those
  // above it: where that is not all, few lanes of a warp hold one, and they wait for a full warp
  // of exponentials.
  template <typename F, typename G>
  __device__ void weigh(float low, G miss, F f) {
    if (low == -INFINITY) {
      each<1>([&](int, float v) { f(v, weight(v)); });
      return;
    }
    float* q = sm.queue[warp];
    int waiting = 0;
    each_from(low, [&](int, float v) {
      miss(v);
      const bool in = v > low;
      const uint32_t late = __ballot_sync(0xffffffffu, in);
      if (!late) return;
      if (in) q[waiting + __popc(late & ((1u << lane) - 1u))] = v;
      waiting += __popc(late);
      __syncwarp();
      if (waiting >= 32) {
        const float x = q[lane];
        f(x, weight(x));
        waiting -= 32;
        const float next = lane < waiting ? q[32 + lane] : 0.0f;
        __syncwarp();
        if (lane < waiting) q[lane] = next;
        __syncwarp();
      }
    });
    if (lane < waiting) f(q[lane], weight(q[lane]));
    __syncwarp();
  }
  __device__ int bin(float v) const {
    const float t = (top - v) * c;
    return t < (float)(kBins - 1) ? (int)t : kBins - 1;
  }
  // The 16 bytes from index i on; NaN past this warp's entries.
  __device__ uint4 raw_at(int i) const {
    if (i + kVec <= w1) {
      if constexpr (DT == 0)
        return *reinterpret_cast<const uint4*>(static_cast<const float*>(x) + i);
      else
        return *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + i);
    }
    uint32_t w[4] = {~0u, ~0u, ~0u, ~0u};  // NaN in every type
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      if (i + e < w1) {
        if constexpr (DT == 0)
          w[e] = static_cast<const uint32_t*>(x)[i + e];
        else
          w[e / 2] = (e & 1) ? (w[e / 2] & 0xffffu) | ((uint32_t) static_cast<const uint16_t*>(x)[i + e] << 16)
                             : (w[e / 2] & 0xffff0000u) | static_cast<const uint16_t*>(x)[i + e];
      }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ static void unpack(uint4 q, float (&v)[kVec]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == 0) {
        v[e] = __uint_as_float(w[e]);
      } else {
        float2 y;
        if constexpr (DT == 1)
          y = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
        else
          y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]));
        v[2 * e] = y.x;
        v[2 * e + 1] = y.y;
      }
    }
  }
  // The largest of them that is no NaN.
  __device__ static float largest(uint4 q) {
    if constexpr (DT == 0) {
      return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
    } else if constexpr (DT == 1) {
      auto h = [](uint32_t u) { return *reinterpret_cast<__half2*>(&u); };
      const float2 m = __half22float2(__hmax2(__hmax2(h(q.x), h(q.y)), __hmax2(h(q.z), h(q.w))));
      return fmaxf(m.x, m.y);
    } else {
      auto h = [](uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); };
      const float2 m = __bfloat1622float2(__hmax2(__hmax2(h(q.x), h(q.y)), __hmax2(h(q.z), h(q.w))));
      return fmaxf(m.x, m.y);
    }
  }
  // f(index, value) over this warp's entries, the whole warp in every call: lanes without
  // an entry bring NaN.  AHEAD loads are in flight before the first use.
  template <int AHEAD, typename F>
  __device__ void each(F f) const {
    if (a.wide) {
#pragma unroll 1
      for (int i = w0 + lane * kVec; i - lane * kVec < w1; i += AHEAD * 32 * kVec) {
        uint4 q[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) q[k] = raw_at(i + k * 32 * kVec);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          float v[kVec];
          unpack(q[k], v);
#pragma unroll
          for (int e = 0; e < kVec; ++e) f(i + k * 32 * kVec + e, v[e]);
        }
      }
    } else {
      for (int i = w0 + lane; i - lane < w1; i += 32) f(i, i < w1 ? load<DT>(x, i) : NAN);
    }
  }

  __device__ __nv_bfloat16* marks_of_warp() const { return sm.marks + warp * (chunk_steps(a.per_warp) * 32); }
  // Steps of a chunk a lane over n entries.
  __host__ __device__ static constexpr int chunk_steps(int n) { return (n + kFar * 32 * kVec - 1) / (kFar * 32 * kVec); }

  // The largest of this lane's entries that is no NaN; leaves the chunks' maxima in marks.
  __device__ float row_max() const {
    float most = -INFINITY;
    if (a.wide) {
      __nv_bfloat16* mark = marks_of_warp() + lane;
#pragma unroll 1
      for (int i = w0 + lane * kVec; i - lane * kVec < w1; i += kFar * 32 * kVec, mark += 32) {
        uint4 q[kFar];
#pragma unroll
        for (int k = 0; k < kFar; ++k) q[k] = raw_at(i + k * 32 * kVec);
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < kFar; ++k) m = fmaxf(m, largest(q[k]));
        *mark = __float2bfloat16_ru(m);
        most = fmaxf(most, m);
      }
    } else {
      for (int i = w0 + lane; i < w1; i += 32) most = fmaxf(most, load<DT>(x, i));
    }
    return most;
  }
  // f(index, value) at least for the entries that are not below `low`, the whole warp in every
  // call (lanes without an entry bring NaN).  The marks tell which chunks hold any; 32 of those
  // at a time are shared out, a vector of eight of them a lane.
  template <typename F>
  __device__ void each_from(float low, F f) const {
    if (!a.wide) {
      each<1>(f);
      return;
    }
    const __nv_bfloat16* mark = marks_of_warp() + lane;
    uint16_t* hits = sm.hits[warp];
    const int steps = chunk_steps(w1 - w0);
    int waiting = 0;
#pragma unroll 1
    for (int it = 0; it <= steps; ++it) {
      const bool in = it < steps && __bfloat162float(mark[it < steps ? it * 32 : 0]) >= low;
      const uint32_t late = __ballot_sync(0xffffffffu, in);
      if (in) hits[waiting + __popc(late & ((1u << lane) - 1u))] = (uint16_t)(it * 32 + lane);
      waiting += __popc(late);
      __syncwarp();
      if (waiting >= 32 || (it == steps && waiting > 0)) {
        uint4 q[kFar];
        int at[kFar];
#pragma unroll
        for (int k = 0; k < kFar; ++k) {
          const int n = (lane >> 2) + 8 * k, chunk = hits[n];
          at[k] = n < waiting ? w0 + ((chunk >> 5) * (kFar * 32) + (lane & 3) * 32 + (chunk & 31)) * kVec : w1;
          q[k] = raw_at(at[k]);
        }
#pragma unroll
        for (int k = 0; k < kFar; ++k) {
          if (8 * k >= waiting || !__any_sync(0xffffffffu, largest(q[k]) >= low)) continue;
          float v[kVec];
          unpack(q[k], v);
#pragma unroll
          for (int e = 0; e < kVec; ++e) f(at[k] + e, v[e]);
        }
        waiting = max(0, waiting - 32);
        const uint16_t next = hits[32 + lane];
        __syncwarp();
        hits[lane] = next;
        __syncwarp();
      }
    }
  }

  __device__ uint64_t block_sum(uint64_t v, uint64_t* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = lane < kWarps ? red[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    return v;
  }

  // Merge the cluster's histograms (buffer `buf`, already synchronised) and find the bin
  // where need(total) >= 1 is reached, counts or weights; `tie_bin` holds `tie_n` more
  // entries of weight `tie_w`.  Thread t has kPer bins, from kPer t on.
  template <bool W, typename F>
  __device__ void find(F need_of, int tie_bin, uint64_t tie_n, uint64_t tie_w) {
    uint64_t n[kPer] = {}, v[kPer] = {};
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = cluster.map_shared_rank(&sm, r);
#pragma unroll
      for (int e = 0; e < kPer; e += 2) {
        const uint2 q = *reinterpret_cast<const uint2*>(o->cnt[buf] + kPer * tid + e);
        n[e] += q.x;
        n[e + 1] += q.y;
        if (W) {
          const uint2 l = *reinterpret_cast<const uint2*>(o->lo[buf] + kPer * tid + e);
          const uint2 h = *reinterpret_cast<const uint2*>(o->hi[buf] + kPer * tid + e);
          v[e] += (uint64_t)l.x + ((uint64_t)h.x << 32);
          v[e + 1] += (uint64_t)l.y + ((uint64_t)h.y << 32);
        }
      }
    }
    uint64_t mine = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (kPer * tid + e == tie_bin) {
        n[e] += tie_n;
        v[e] += tie_n * tie_w;
      }
      if (!W) v[e] = n[e];
      mine += v[e];
    }
    uint64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) sm.red[warp] = inc;
    __syncthreads();
    uint64_t before = lane < warp ? sm.red[lane] : 0, total = lane < kWarps ? sm.red[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    inc += before;
    if (tid == 0) sm.found_total = total;
    const uint64_t need = need_of(total);
    uint64_t at = inc - mine;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (at < need && at + v[e] >= need) {
        sm.found = (uint32_t)(kPer * tid + e);
        sm.found_cnt = (uint32_t)n[e];
        sm.found_above = at;
      }
      at += v[e];
    }
    __syncthreads();
  }

  __device__ void clear_hist(int b) {
    for (int i = tid; i < kBins; i += kNT) sm.cnt[b][i] = sm.lo[b][i] = sm.hi[b][i] = 0;
  }

  template <bool W>
  __device__ void count_in(int b, uint64_t w) {
    atomicAdd(&sm.cnt[buf][b], 1u);
    if (W) {
      const uint32_t l = (uint32_t)w, old = atomicAdd(&sm.lo[buf][b], l);
      const uint32_t h = (uint32_t)(w >> 32) + (old + l < old ? 1u : 0u);
      if (h) atomicAdd(&sm.hi[buf][b], h);
    }
  }

  // The kept set becomes its first entries, by value and then by index, that reach
  // need_of(the kept set's count or, when W, weight).  All CTAs of the cluster call it
  // together.
  template <bool W, typename F>
  __device__ void select(F need_of) {
    const uint32_t sk0 = sk;
    const uint64_t ties = sm_ties;
    const float tie_x = value_of(sk0), tie_v = sk0 ? tie_x : -INFINITY;  // a weight of -inf is 0
    const uint64_t tie_w = (W && ties) ? weight(tie_x) : 0;
    uint64_t above = 0, target = 0;
    int level = 0, b0 = 0;
    uint32_t prefix = 0;
    const int shifts[5] = {0, 22, 12, 2, 0};
    auto digit = [&](uint32_t k, int lv) -> int {  // larger keys first
      return lv == 4 ? 3 - (int)(k & 3u) : 1023 - (int)((k >> shifts[lv]) & 1023u);
    };
    auto matches = [&](float v, uint32_t k, int lv) {
      if (lv == 0) return true;
      if (bin(v) != b0) return false;
      if (lv == 1) return true;
      return (k >> shifts[lv - 1]) == prefix;
    };
    for (;;) {
      each<1>([&](int, float v) {
        if (!(v > tie_v)) return;  // NaN too
        const uint32_t k = key_of(v);
        if (!matches(v, k, level)) return;
        count_in<W>(level == 0 ? bin(v) : digit(k, level), W ? weight(v) : 0);
      });
      cluster.sync();
      const bool tie_in = W && ties && matches(tie_x, sk0, level);
      find<W>([&](uint64_t total) { return level == 0 ? need_of(total) : target - above; },
              tie_in ? (level == 0 ? bin(tie_x) : digit(sk0, level)) : -1, ties, tie_w);
      clear_hist(buf ^ 1);  // the other buffer was last read before this step's barrier
      buf ^= 1;
      if (level == 0) target = need_of(sm.found_total);
      const int f = (int)sm.found;
      const uint32_t n = sm.found_cnt;
      above += sm.found_above;
      if (level == 0)
        b0 = f;
      else if (level == 4)
        prefix = (prefix << 2) | (uint32_t)(3 - f);
      else
        prefix = (prefix << 10) | (uint32_t)(1023 - f);
      __syncthreads();
      ++level;
      if (level == 5) {  // the whole key is known
        sk = prefix;
        sm_ties = W ? (target - above + weight(value_of(sk)) - 1) / weight(value_of(sk)) : target - above;
        return;
      }
      if (n <= (uint32_t)kList) break;
    }
    // gather the bin's entries and rank them
    if (tid == 0) sm.list_n = 0;
    __syncthreads();
    each<1>([&](int, float v) {
      if (!(v > tie_v) || bin(v) != b0) return;
      const uint32_t k = key_of(v);
      if (!matches(v, k, level)) return;
      const uint32_t at = atomicAdd(&sm.list_n, 1u);
      if (at < (uint32_t)kList) sm.list[at] = k;
    });
    cluster.sync();
    settle<W>(above, target, W && ties && matches(tie_x, sk0, level), sk0, ties);
  }

  // Ranks the entries that the CTAs' lists hold (already synchronised), at most kList in
  // all, and `ties` more of key tie_key where tie_in: the threshold where `target` is
  // reached, `above` lying before them.
  template <bool W>
  __device__ void settle(uint64_t above, uint64_t target, bool tie_in, uint32_t tie_key, uint64_t ties) {
    uint32_t total = 0;
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = cluster.map_shared_rank(&sm, r);
      const uint32_t m = min(o->list_n, (uint32_t)kList);
      for (uint32_t i = tid; i < m && total + i < (uint32_t)kCand; i += kNT) sm.keys[total + i] = o->list[i];
      total += m;
    }
    if (tie_in && tid == 0 && total < (uint32_t)kCand) sm.keys[total] = tie_key;
    if (tie_in) ++total;
    total = min(total, (uint32_t)kCand);
    __syncthreads();
    for (uint32_t i = tid; i < total; i += kNT) {
      const uint64_t w = W ? weight(value_of(sm.keys[i])) : 1;
      sm.weights[i] = (tie_in && i == total - 1) ? ties * w : w;
    }
    __syncthreads();
    for (uint32_t i0 = 0; i0 < total; i0 += kNT / kLanes) {
      const uint32_t i = i0 + tid / kLanes;
      const uint32_t k = i < total ? sm.keys[i] : 0;
      uint64_t gt = 0, eq = 0;
#pragma unroll 4
      for (uint32_t j = tid % kLanes; j < total; j += kLanes) {
        const uint32_t kj = sm.keys[j];
        const uint64_t wj = sm.weights[j];
        gt += kj > k ? wj : 0;
        eq += kj == k ? wj : 0;
      }
#pragma unroll
      for (int o = 1; o < kLanes; o *= 2) {
        gt += __shfl_xor_sync(0xffffffffu, gt, o);
        eq += __shfl_xor_sync(0xffffffffu, eq, o);
      }
      gt += above;
      if (i < total && gt < target && gt + eq >= target) {
        const uint64_t w = W ? weight(value_of(k)) : 1;
        sm.found = k;
        sm.found_above = (target - gt + w - 1) / w;
      }
    }
    __syncthreads();
    sk = sm.found;
    sm_ties = sm.found_above;
    __syncthreads();
  }

  // The nucleus of the whole row.  A histogram of counts and of places within the bins
  // brackets each bin's weight: with f the mean place, n e^(-step f) is a lower bound (the
  // exponential is convex) and 1 + step^2 / 8 < 1.0003 times that an upper one.  The exact
  // pass then sums what lies before the bins that may hold the threshold, and the whole,
  // and gathers those bins' entries, or, where they are too many, a finer histogram of them.
  // False: too many even so.
  __device__ bool nucleus_of_row(float p) {
    constexpr double kStep = 31.9 / kBins;
    each<kAhead>([&](int, float v) {
      const float t = (top - v) * c;
      if (!(t < (float)kBins)) return;  // NaN, and what weighs nothing
      const uint32_t fixed = (uint32_t)(t * 4096.0f);
      atomicAdd(&sm.cnt[buf][fixed >> 12], 1u);
      atomicAdd(&sm.lo[buf][fixed >> 12], fixed & 4095u);
    });
    if (tid == 0) sm.list_n = 0;
    cluster.sync();
    uint64_t n[kPer] = {}, f[kPer] = {};
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = cluster.map_shared_rank(&sm, r);
#pragma unroll
      for (int e = 0; e < kPer; e += 2) {
        const uint2 q = *reinterpret_cast<const uint2*>(o->cnt[buf] + kPer * tid + e);
        const uint2 g = *reinterpret_cast<const uint2*>(o->lo[buf] + kPer * tid + e);
        n[e] += q.x;
        n[e + 1] += q.y;
        f[e] += g.x;
        f[e + 1] += g.y;
      }
    }
    // the lower bounds in units of 2^-40 of the largest weight: whole numbers again, so that
    // every CTA finds the same bins
    uint64_t w[kPer], inc[2] = {0, 0}, mine[2];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      w[e] = n[e] ? (uint64_t)((double)n[e] * exp(-kStep * ((double)(kPer * tid + e) + (double)f[e] / (4096.0 * (double)n[e]))) *
                               1099511627776.0)
                  : 0;
      inc[0] += w[e];
      inc[1] += n[e];
    }
    mine[0] = inc[0];
    mine[1] = inc[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, inc[e], o);
        if (lane >= o) inc[e] += y;
      }
    if (lane == 31) {
      sm.red[warp] = inc[0];
      sm.red2[warp] = inc[1];
    }
    __syncthreads();
    uint64_t all = 0;
    for (int k = 0; k < kWarps; ++k) {
      if (k < warp) {
        inc[0] += sm.red[k];
        inc[1] += sm.red2[k];
      }
      all += sm.red[k];
    }
    const double part = (double)p * (double)all;
    const uint64_t low = max((uint64_t)1, (uint64_t)(part * 0.9996)), high = max(low, min(all, (uint64_t)(part * 1.0004) + 1));
    uint64_t at = inc[0] - mine[0], many = inc[1] - mine[1];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (at < low && at + w[e] >= low) {
        sm.found = (uint32_t)(kPer * tid + e);
        sm.found_above = many;
      }
      if (at < high && at + w[e] >= high) {
        sm.found_cnt = (uint32_t)(kPer * tid + e);
        sm.found_total = many + n[e];
      }
      at += w[e];
      many += n[e];
    }
    __syncthreads();
    const float from = (float)sm.found, upto = (float)(sm.found_cnt + 1);
    const bool few = sm.found_total - sm.found_above <= (uint64_t)kList;
    buf ^= 1;
    const float fine = (float)kBins / (upto - from);
    auto fine_bin = [&](float t) { return min((int)((t - from) * fine), kBins - 1); };
    uint64_t z = 0, before = 0;
    weigh(-INFINITY, [](float) {}, [&](float v, uint64_t e) {
      const float t = (top - v) * c;
      z += e;
      before += t < from ? e : 0;
      if (t >= from && t < upto) {
        if (few) {
          const uint32_t at = atomicAdd(&sm.list_n, 1u);
          if (at < (uint32_t)kList) sm.list[at] = key_of(v);
        } else {
          count_in<true>(fine_bin(t), e);
        }
      }
    });
    z = block_sum(z, sm.red);
    before = block_sum(before, sm.red);
    if (tid == 0) {
      sm.xch[2][0] = z;
      sm.xch[2][1] = before;
    }
    cluster.sync();
    z = before = 0;
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = cluster.map_shared_rank(&sm, r);
      z += o->xch[2][0];
      before += o->xch[2][1];
    }
    const uint64_t target = nucleus(p, z);
    if (!few) {
      find<true>([&](uint64_t) { return target - before; }, -1, 0, 0);
      const int fb = (int)sm.found;
      before += sm.found_above;
      const bool fits = sm.found_cnt <= (uint32_t)kList;
      clear_hist(buf ^ 1);
      buf ^= 1;
      __syncthreads();
      if (!fits) return false;
      each<kAhead>([&](int, float v) {
        const float t = (top - v) * c;
        if (!(t >= from && t < upto) || fine_bin(t) != fb) return;
        const uint32_t at = atomicAdd(&sm.list_n, 1u);
        if (at < (uint32_t)kList) sm.list[at] = key_of(v);
      });
      cluster.sync();
    }
    settle<true>(before, target, false, 0, 0);
    return true;
  }

  // floor(u * total), within 0 .. total - 1
  __device__ static uint64_t drawn(float u, uint64_t total) {
    const double e = floor((double)(u > 0.0f ? u : 0.0f) * (double)total);
    return e < (double)total ? min((uint64_t)e, total - 1) : total - 1;
  }
  __device__ static uint64_t nucleus(float p, uint64_t total) {
    const double e = floor((double)p * (double)total);
    return e >= 1.0 ? min(total, (uint64_t)e) : 1;
  }

  // Sorts n <= kCand different values above zero (in shared memory, complete), the largest first.
  // Up to 128 by counting the larger ones, kLanes threads a value: 0.4 us there against 1.0;
  // more by a bitonic network on the next power of two, whose steps of up to 32 places stay
  // within a warp's 64 values: for 265, 1.5 us against 10.
  template <typename U>
  __device__ void sort(U* v, int n) const {
    if (n <= kNT / kLanes) {
      const int i = tid / kLanes;
      const U x = i < n ? v[i] : 0;
      int place = 0;
#pragma unroll 4
      for (int j = tid % kLanes; j < n; j += kLanes) place += v[j] > x;
#pragma unroll
      for (int o = 1; o < kLanes; o *= 2) place += __shfl_xor_sync(0xffffffffu, place, o);
      __syncthreads();
      if (i < n && tid % kLanes == 0) v[place] = x;
      __syncthreads();
      return;
    }
    const int all = 1 << (32 - __clz(n - 1));
    for (int i = n + tid; i < all; i += kNT) v[i] = 0;
    __syncthreads();
    for (int size = 2; size <= all; size *= 2)
      for (int j = size / 2; j > 0; j /= 2) {
        if (tid < all / 2) {
          const int i = 2 * tid - (tid & (j - 1));
          const U x = v[i], y = v[i + j];
          if ((x < y) == ((i & size) == 0)) {
            v[i] = y;
            v[i + j] = x;
          }
        }
        if (j > 32 || (j == 1 && size > 32))
          __syncthreads();
        else
          __syncwarp();
      }
  }

  // The sum of the threads' values before this one's, and of all.
  __device__ uint64_t scan(uint64_t mine, uint64_t& total) const {
    uint64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    __syncthreads();
    if (lane == 31) sm.red[warp] = inc;
    __syncthreads();
    uint64_t before = lane < warp ? sm.red[lane] : 0;
    total = lane < kWarps ? sm.red[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    return before + inc - mine;
  }

  // The k largest are among n <= kCand candidates: rank 0 decides on them alone.  Two sorts: by
  // rank for the filters, which each keep the first so many, and those by index for the pick.
  __device__ void among(int n, int k, float p, uint64_t least, float u, int row) {
    const int most = min(n, k);
    sort(sm.cand, n);
    uint64_t w[kPer], mine = 0, total;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int r = kPer * tid + e;
      w[e] = r < most ? weight(value_of((uint32_t)(sm.cand[r] >> 32))) : 0;
      mine += w[e];
    }
    if (p < 1.0f) {  // those before which `enough` is not reached yet
      uint64_t before = scan(mine, total);
      const uint64_t enough = nucleus(p, total);
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const uint64_t next = before + w[e];
        if (before >= enough) w[e] = 0;
        before = next;
      }
    }
    int kept = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (w[e] < least) w[e] = 0;
      sm.weights[kPer * tid + e] = w[e];
      kept += __syncthreads_count(w[e] > 0);
    }
    // the largest complement of (index, rank) first: the lowest index
    for (int r = tid; r < kept; r += kNT) sm.keys[r] = ~((~(uint32_t)sm.cand[r] << 10) | (uint32_t)r);
    __syncthreads();
    sort(sm.keys, kept);
    mine = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int r = kPer * tid + e;
      w[e] = r < kept ? sm.weights[~sm.keys[r] & 1023u] : 0;
      mine += w[e];
    }
    uint64_t before = scan(mine, total);
    const uint64_t at = drawn(u, total);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (before <= at && at < before + w[e]) a.ids[row] = (int)(~sm.keys[kPer * tid + e] >> 10);
      before += w[e];
    }
  }

  __device__ void run(int row) {
    // ---- the largest value and its lowest index
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float mp = a.min_p ? a.min_p[row] : 0.0f;
    const float u = a.u[row];
    const float mine = row_max();
    uint64_t best = key_of(mine);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sm.red[warp] = best;
    if (tid == 0) sm.cand_n = 0, sm.first = 0x7fffffffu;
    if (tid < 64) sm.pow2[tid] = exp2(44.0 - (double)tid / 64.0);
    buf = 0;
    clear_hist(0);
    clear_hist(1);
    __syncthreads();
    if (warp == 0) {
      uint64_t b = lane < kWarps ? sm.red[lane] : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
      if (lane == 0) sm.xch[0][0] = b;
    }
    cluster.sync();
    best = 0;
    for (int r = 0; r < ranks; ++r) best = max(best, cluster.map_shared_rank(&sm, r)->xch[0][0]);
    top = value_of((uint32_t)best);
    if (!(fabsf(top) < INFINITY) || !(t > 0.0f) || k == 1) {  // the maximum's lowest index
      uint32_t first = 0x7fffffffu;
      each_from(top, [&](int i, float v) {
        if (v == top) first = min(first, (uint32_t)i);  // NaN past the row's end
      });
      first = __reduce_min_sync(0xffffffffu, first);
      if (lane == 0) atomicMin(&cluster.map_shared_rank(&sm, 0)->first, first);
      cluster.sync();
      if (rank == 0 && tid == 0) a.ids[row] = sm.first == 0x7fffffffu ? 0 : (int)sm.first;  // NaN alone: 0
      return;
    }
    topd = (double)top;
    scale = 1.4426950408889634074 / (double)t;
    c = fminf((float)kBins / 31.9f / t, 1e30f);  // 46 ln 2: beyond it a weight is zero
    sk = 0;
    sm_ties = 0;
    const uint64_t least = mp > 0.0f ? (uint64_t)ceil((double)fminf(mp, 1.0f) * kUnit) : 0;
    // ---- filters
    if (k > 0 && k < a.V) {
      // The lanes' maxima bound the k-th largest from below: at least k entries lie in the
      // bins up to the one where the maxima reach k, and with many more lanes than k few
      // others do.
      bool few = 2 * k <= ranks * kNT;
      if (few) {
        if (mine > -INFINITY) atomicAdd(&sm.cnt[0][bin(mine)], 1u);
        cluster.sync();
        find<false>([&](uint64_t total) { return total >= (uint64_t)k ? (uint64_t)k : 0; }, -1, 0, 0);
        few = sm.found_total >= (uint64_t)k && sm.found < (uint32_t)kBins - 1;
        buf = 1;  // zero since the start: clearing it here would race with the select's counting, which may follow at once
      }
      if (few) {
        const float upto = (float)(sm.found + 1);
        Shared* o = cluster.map_shared_rank(&sm, 0);
        // a little below the last value that qualifies: the exact test follows
        const float from = top - upto / c - 1e-5f * (upto / c + fabsf(top));
        each_from(from, [&](int i, float v) {
          if (!((top - v) * c < upto)) return;
          const uint32_t at = atomicAdd(&o->cand_n, 1u);
          if (at < (uint32_t)kCand) o->cand[at] = (uint64_t)key_of(v) << 32 | (uint32_t)~i;
        });
        cluster.sync();
        const uint32_t n = o->cand_n;
        if (n <= (uint32_t)kCand) {
          if (rank == 0) among((int)n, k, p, least, u, row);
          return;
        }
      }
      select<false>([&](uint64_t total) { return min((uint64_t)k, total); });
    }
    if (p < 1.0f && (sk || !nucleus_of_row(p))) select<true>([&](uint64_t total) { return nucleus(p, total); });
    auto kept_weight = [&](float v) -> uint64_t {
      const uint64_t w = weight(v);
      return w >= least ? w : 0;
    };
    // ---- the pick
    const uint64_t tie_w = sm_ties ? kept_weight(value_of(sk)) : 0;
    const float kept_above = sk ? value_of(sk) : -INFINITY;  // a weight of -inf is 0
    uint64_t z = 0;
    uint32_t ties = 0;
    weigh(kept_above, [&](float v) { ties += v == kept_above; }, [&](float, uint64_t w) { z += w >= least ? w : 0; });
    if (!sm_ties) ties = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      z += __shfl_xor_sync(0xffffffffu, z, o);
      ties += __shfl_xor_sync(0xffffffffu, ties, o);
    }
    if (lane == 0) {
      sm.red[warp] = z;
      sm.red2[warp] = ties;
    }
    __syncthreads();
    if (warp == 0) {
      uint64_t zz = lane < kWarps ? sm.red[lane] : 0, tt = lane < kWarps ? sm.red2[lane] : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        zz += __shfl_xor_sync(0xffffffffu, zz, o);
        tt += __shfl_xor_sync(0xffffffffu, tt, o);
      }
      if (lane == 0) {
        sm.xch[1][0] = zz;
        sm.xch[1][1] = tt;
      }
    }
    cluster.sync();
    uint64_t total = 0, base = 0, tie_base = 0;
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = cluster.map_shared_rank(&sm, r);
      if (r < rank) {
        base += o->xch[1][0];
        tie_base += o->xch[1][1];
      }
      total += o->xch[1][0];
    }
    total += sm_ties * tie_w;
    const uint64_t at = drawn(u, total);
    // weight kept before an entry = what lies above sk + the ties kept so far
    auto ties_kept = [&](uint64_t n) { return min(n, sm_ties) * tie_w; };
    if (tid == 0) sm.found = kWarps;
    __syncthreads();
    if (lane == 0) {
      for (int w = 0; w < warp; ++w) {
        base += sm.red[w];
        tie_base += sm.red2[w];
      }
      if (at >= base + ties_kept(tie_base) && at < base + sm.red[warp] + ties_kept(tie_base + sm.red2[warp])) {
        sm.found = (uint32_t)warp;
        sm.found_above = base;
        sm.found_total = tie_base;
      }
    }
    __syncthreads();
    if (sm.found == kWarps) return;
    // the CTA shares the entries of that warp, a stretch a thread, and scans them
    base = sm.found_above;
    tie_base = sm.found_total;
    const int64_t start = (int64_t)(rank * kWarps + (int)sm.found) * a.per_warp;
    const int per = a.per_warp / 256, stop = (int)min(start + a.per_warp, (int64_t)a.V);
    const int i0 = (int)min(start + (int64_t)tid * per, (int64_t)stop), i1 = tid < 256 ? min(i0 + per, stop) : i0;
    uint64_t w = 0, tied = 0;
    for (int i = i0; i < i1; ++i) {
      const float v = load<DT>(x, i);
      if (v > kept_above) w += kept_weight(v);
      tied += sm_ties && v == kept_above;
    }
    uint64_t w_in = w, t_in = tied;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, w_in, o), t = __shfl_up_sync(0xffffffffu, t_in, o);
      if (lane >= o) {
        w_in += y;
        t_in += t;
      }
    }
    __syncthreads();
    if (lane == 31) {
      sm.red[warp] = w_in;
      sm.red2[warp] = t_in;
    }
    __syncthreads();
    for (int k = 0; k < warp; ++k) {
      base += sm.red[k];
      tie_base += sm.red2[k];
    }
    base += w_in - w;
    tie_base += t_in - tied;
    if (at < base + ties_kept(tie_base) || at >= base + w + ties_kept(tie_base + tied)) return;
    for (int i = i0; i < i1; ++i) {
      const float v = load<DT>(x, i);
      if (v > kept_above) base += kept_weight(v);
      tie_base += sm_ties && v == kept_above;
      if (base + ties_kept(tie_base) > at) {
        a.ids[row] = i;
        return;
      }
    }
  }
};

template <int DT>
__global__ void __launch_bounds__(kNT, 2) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sm = *reinterpret_cast<Shared*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = (int)(blockIdx.x / ranks);
  const int tid = threadIdx.x, warp = tid >> 5;
  const int64_t first = (int64_t)(rank * (kNT / 32) + warp) * a.per_warp;
  constexpr int es = DT == 0 ? 4 : 2;
  Row<DT> r{a, sm, cluster, static_cast<const uint8_t*>(a.x) + (int64_t)row * a.ldx * es, rank, ranks, tid, tid & 31, warp,
                (int)min(first, (int64_t)a.V), (int)min(first + a.per_warp, (int64_t)a.V)};
  r.run(row);
  cluster.sync();  // no CTA leaves while another may read its shared memory
}

template <int DT>
constexpr int smem_bytes(int per_warp) {
  return (int)(sizeof(Shared) + kWarps * Row<DT>::chunk_steps(per_warp) * 32 * sizeof(__nv_bfloat16));
}

template <int DT>
cudaError_t sample_launch(SampleArgs a, int64_t T, int ranks, cudaStream_t st) {
  static std::atomic<uint64_t> configured{0};  // devices whose attribute is set
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load(std::memory_order_relaxed) & bit)) {
    cudaError_t e = cudaFuncSetAttribute(sample_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<DT>((int)(kSampleMaxVocab / kWarps)));
    if (e != cudaSuccess) return e;
    configured.fetch_or(bit, std::memory_order_relaxed);
  }
  const int64_t warps = (int64_t)ranks * (kNT / 32);
  a.per_warp = (int)((a.V + warps - 1) / warps + 255) / 256 * 256;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(T * ranks));
  cfg.blockDim = dim3(kNT);
  cfg.dynamicSmemBytes = smem_bytes<DT>(a.per_warp);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&cfg, sample_kernel<DT>, a);
}

}  // namespace

cudaError_t launch_sample(const void* x, int dt, int64_t ldx, int64_t T, int64_t V, const float* temperature,
                          const int* top_k, const float* top_p, const float* min_p, const float* u, int* ids,
                          cudaStream_t st) {
  if (T <= 0) return cudaSuccess;
  const int es = dt == 0 ? 4 : 2;
  const int wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (T == 1 || ldx * es % 16 == 0);
  const SampleArgs a{x, ldx, (int)V, 0, wide, temperature, top_k, top_p, min_p, u, ids};
  int ranks = 1;
  while (ranks < kMaxRanks && V > (int64_t)ranks * 4096 && 2 * ranks * T <= kResident) ranks *= 2;
  return dt == 0 ? sample_launch<0>(a, T, ranks, st) : dt == 1 ? sample_launch<1>(a, T, ranks, st) : sample_launch<2>(a, T, ranks, st);
}

}  // namespace rtd
