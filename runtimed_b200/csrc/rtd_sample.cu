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
// A select finds the threshold where a count (top-k) or a weight (top-p) is reached:
// first a histogram over 1024 equal steps of (max - x) / t, which spreads any row's upper
// end over many bins; then, if at most 1023 entries share the bin, they are gathered and
// ranked against one another, else the bin is split by the bits of the value's order map.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "rtd_common.cuh"
#include "rtd_kernels.h"

namespace rtd {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kBins = 1024;
constexpr int kList = 1023;
constexpr int kMaxRanks = 8;
constexpr double kUnit = 17592186044416.0;  // 2^44

struct SampleArgs {
  const void* x;
  int64_t ldx;
  int V;
  int per_warp;  // entries of a warp, a multiple of 32
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
  uint32_t list[kList + 1];
  uint32_t keys[kList + 1];
  uint64_t weights[kList + 1];
  uint64_t red[32];
  uint64_t red2[32];
  uint64_t xch[4][2];  // values for the other CTAs, a slot per exchange
  uint32_t list_n;
  uint32_t found, found_cnt;
  uint64_t found_above;
};

template <int DT>
struct Row {
  const SampleArgs& a;
  Shared& sm;
  cg::cluster_group cluster;
  const void* x;
  int rank, ranks, tid, lane, warp, w0, w1;
  float top, c;      // the row's maximum; histogram steps per unit of (max - x)
  double inv_t, topd;
  uint32_t sk;       // kept: keys above sk ...
  uint64_t sm_ties;  // ... and the first sm_ties entries with key sk
  int buf = 0;

  __device__ uint64_t weight(float v) const {
    if (v == -INFINITY) return 0;
    return (uint64_t)__double2ll_rn(exp(((double)v - topd) * inv_t) * kUnit);
  }
  __device__ int bin(float v) const {
    const float t = (top - v) * c;
    return t < (float)(kBins - 1) ? (int)t : kBins - 1;
  }
  template <typename F>
  __device__ void each(F f) const {
#pragma unroll 4
    for (int i = w0 + lane; i < w1; i += 32) f(i, load<DT>(x, i));
  }

  __device__ uint64_t block_sum(uint64_t v, uint64_t* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = red[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    return v;
  }

  // Merge the cluster's histograms (buffer `buf`, already synchronised) and find the bin
  // where `need` (>= 1) is reached; `tie_bin` holds `tie_n` more entries of weight `tie_w`.
  template <bool W>
  __device__ void find(uint64_t need, int tie_bin, uint64_t tie_n, uint64_t tie_w) {
    uint64_t n = 0, v = 0;
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = cluster.map_shared_rank(&sm, r);
      n += o->cnt[buf][tid];
      if (W) v += (uint64_t)o->lo[buf][tid] + ((uint64_t)o->hi[buf][tid] << 32);
    }
    if (tid == tie_bin) {
      n += tie_n;
      v += tie_n * tie_w;
    }
    if (!W) v = n;
    uint64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) sm.red[warp] = inc;
    __syncthreads();
    uint64_t before = lane < warp ? sm.red[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    inc += before;
    if (inc >= need && inc - v < need) {
      sm.found = (uint32_t)tid;
      sm.found_cnt = (uint32_t)n;
      sm.found_above = inc - v;
    }
    __syncthreads();
  }

  __device__ void clear_hist(int b) {
    sm.cnt[b][tid] = 0;
    sm.lo[b][tid] = 0;
    sm.hi[b][tid] = 0;
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
  // `target` (a count, or a weight when W); entries lighter than `floor_w` cannot be among
  // them.  All CTAs of the cluster call it together.
  template <bool W>
  __device__ void select(uint64_t target, uint64_t floor_w) {
    const uint32_t sk0 = sk;
    const uint64_t ties = sm_ties;
    const float tie_x = value_of(sk0);
    const uint64_t tie_w = (W && ties) ? weight(tie_x) : 0;
    // a value below which no weight reaches floor_w, with room for the roundings
    float floor_x = -INFINITY;
    if (W && floor_w > 1)
      floor_x = top + (logf((float)floor_w * 5.6843418860808015e-14f) - 1e-3f) / (float)inv_t - 1e-6f * fabsf(top);
    if (!(floor_x < top)) floor_x = -INFINITY;
    uint64_t above = 0;
    int level = 0, b0 = 0;
    uint32_t prefix = 0, n = 0;
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
      each([&](int, float v) {
        const uint32_t k = key_of(v);
        if (k <= sk0 || v < floor_x || !matches(v, k, level)) return;
        uint64_t w = 0;
        if (W) {
          w = weight(v);
          if (w < floor_w) return;
        }
        count_in<W>(level == 0 ? bin(v) : digit(k, level), w);
      });
      cluster.sync();
      const bool tie_in = W && ties && matches(tie_x, sk0, level);
      find<W>(target - above, tie_in ? (level == 0 ? bin(tie_x) : digit(sk0, level)) : -1, ties, tie_w);
      const int f = (int)sm.found;
      n = sm.found_cnt;
      above += sm.found_above;
      clear_hist(buf ^ 1);  // the other buffer was last read before this step's barrier
      buf ^= 1;
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
    each([&](int, float v) {
      const uint32_t k = key_of(v);
      if (k <= sk0 || v < floor_x || !matches(v, k, level)) return;
      if (W && floor_w > 1 && weight(v) < floor_w) return;
      const uint32_t at = atomicAdd(&sm.list_n, 1u);
      if (at < (uint32_t)kList) sm.list[at] = k;
    });
    cluster.sync();
    uint32_t total = 0;
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = cluster.map_shared_rank(&sm, r);
      const uint32_t m = min(o->list_n, (uint32_t)kList);
      if (tid < (int)m && total + tid <= (uint32_t)kList) sm.keys[total + tid] = o->list[tid];
      total += m;
    }
    const bool tie_in = W && ties && matches(tie_x, sk0, level);
    if (tie_in && tid == 0 && total <= (uint32_t)kList) sm.keys[total] = sk0;
    if (tie_in) ++total;
    total = min(total, (uint32_t)kList + 1u);
    __syncthreads();
    const bool mine = tid < (int)total;
    const uint32_t k = mine ? sm.keys[tid] : 0;
    const uint64_t w1 = mine ? (W ? weight(value_of(k)) : 1) : 0;
    if (mine) sm.weights[tid] = (tie_in && tid == (int)total - 1) ? ties * w1 : w1;
    __syncthreads();
    if (mine) {
      uint64_t gt = above, eq = 0;
      for (uint32_t j = 0; j < total; ++j) {
        const uint32_t kj = sm.keys[j];
        const uint64_t wj = sm.weights[j];
        if (kj > k) gt += wj;
        if (kj == k) eq += wj;
      }
      if (gt < target && gt + eq >= target) {
        sm.found = k;
        sm.found_above = (target - gt + w1 - 1) / w1;
      }
    }
    __syncthreads();
    sk = sm.found;
    sm_ties = sm.found_above;
    __syncthreads();
  }

  __device__ void run(int row) {
    // ---- the largest value and its lowest index
    uint64_t best = 0, valid = 0;
    each([&](int i, float v) {
      const uint32_t k = key_of(v);
      valid += k != 0;
      const uint64_t p = ((uint64_t)k << 32) | (uint32_t)(0xffffffffu - (uint32_t)i);
      if (k && p > best) best = p;
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sm.red2[warp] = best;
    clear_hist(0);
    clear_hist(1);
    valid = block_sum(valid, sm.red);
    best = sm.red2[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (tid == 0) {
      sm.xch[0][0] = best;
      sm.xch[0][1] = valid;
    }
    cluster.sync();
    valid = 0;
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = cluster.map_shared_rank(&sm, r);
      best = max(best, o->xch[0][0]);
      valid += o->xch[0][1];
    }
    top = value_of((uint32_t)(best >> 32));
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const int k = a.top_k ? a.top_k[row] : 0;
    if (best == 0 || !(fabsf(top) < INFINITY) || !(t > 0.0f) || k == 1) {
      if (rank == 0 && tid == 0) a.ids[row] = best == 0 ? 0 : (int)(0xffffffffu - (uint32_t)best);
      return;
    }
    topd = (double)top;
    inv_t = 1.0 / (double)t;
    c = fminf((float)kBins / 31.9f / t, 1e30f);  // 46 ln 2: beyond it a weight is zero
    sk = 0;
    sm_ties = 0;
    // ---- filters
    if (k > 0 && (uint64_t)k < valid) select<false>((uint64_t)k, 0);
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    if (p < 1.0f) {
      uint64_t z = 0;
      each([&](int, float v) {
        if (key_of(v) > sk) z += weight(v);
      });
      z = block_sum(z, sm.red);
      if (tid == 0) sm.xch[1][0] = z;
      cluster.sync();
      z = sm_ties ? sm_ties * weight(value_of(sk)) : 0;
      for (int r = 0; r < ranks; ++r) z += cluster.map_shared_rank(&sm, r)->xch[1][0];
      const double e = floor((double)p * (double)z);
      const uint64_t target = e >= 1.0 ? min(z, (uint64_t)e) : 1;
      select<true>(target, (z - target) / (uint64_t)a.V);
    }
    const float mp = a.min_p ? a.min_p[row] : 0.0f;
    const double least = mp > 0.0f ? (double)fminf(mp, 1.0f) * kUnit : 0.0;
    auto kept_weight = [&](float v) -> uint64_t {
      const uint64_t w = weight(v);
      return (double)w >= least ? w : 0;
    };
    // ---- the pick
    const uint64_t tie_w = sm_ties ? kept_weight(value_of(sk)) : 0;
    uint64_t z = 0, ties = 0;
    each([&](int, float v) {
      const uint32_t key = key_of(v);
      if (key > sk) z += kept_weight(v);
      if (sm_ties && key == sk) ++ties;
    });
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
      uint64_t zz = sm.red[lane], tt = sm.red2[lane];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        zz += __shfl_xor_sync(0xffffffffu, zz, o);
        tt += __shfl_xor_sync(0xffffffffu, tt, o);
      }
      if (lane == 0) {
        sm.xch[2][0] = zz;
        sm.xch[2][1] = tt;
      }
    }
    cluster.sync();
    uint64_t total = 0, base = 0, tie_base = 0;
    for (int r = 0; r < ranks; ++r) {
      const Shared* o = cluster.map_shared_rank(&sm, r);
      if (r < rank) {
        base += o->xch[2][0];
        tie_base += o->xch[2][1];
      }
      total += o->xch[2][0];
    }
    total += sm_ties * tie_w;
    const float u = a.u[row];
    const double e = floor((double)(u > 0.0f ? u : 0.0f) * (double)total);
    const uint64_t at = e < (double)total ? min((uint64_t)e, total - 1) : total - 1;
    for (int w = 0; w < warp; ++w) {
      base += sm.red[w];
      tie_base += sm.red2[w];
    }
    // weight kept before an entry = what lies above sk + the ties kept so far
    auto ties_kept = [&](uint64_t n) { return min(n, sm_ties) * tie_w; };
    const uint64_t from = base + ties_kept(tie_base);
    const uint64_t to = base + sm.red[warp] + ties_kept(tie_base + sm.red2[warp]);
    if (at < from || at >= to) return;
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      const float v = i < w1 ? load<DT>(x, i) : NAN;
      const uint32_t key = key_of(v);
      const bool tie = sm_ties && key == sk && i < w1;
      uint64_t w = key > sk ? kept_weight(v) : 0;
      const uint32_t tied = __ballot_sync(0xffffffffu, tie);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
      }
      const uint64_t reached = base + w + ties_kept(tie_base + __popc(tied & (0xffffffffu >> (31 - lane))));
      const uint32_t past = __ballot_sync(0xffffffffu, reached > at);
      if (past) {
        if (lane == __ffs(past) - 1) a.ids[row] = i;
        return;
      }
      base += __shfl_sync(0xffffffffu, w, 31);
      tie_base += __popc(tied);
    }
  }
};

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& sm = *reinterpret_cast<Shared*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = (int)(blockIdx.x / ranks);
  const int tid = threadIdx.x, warp = tid >> 5;
  const int64_t first = (int64_t)(rank * (kThreads / 32) + warp) * a.per_warp;
  constexpr int es = DT == 0 ? 4 : 2;
  Row<DT> r{a, sm, cluster, static_cast<const uint8_t*>(a.x) + (int64_t)row * a.ldx * es, rank, ranks, tid, tid & 31, warp,
            (int)min(first, (int64_t)a.V), (int)min(first + a.per_warp, (int64_t)a.V)};
  r.run(row);
  cluster.sync();  // no CTA leaves while another may read its shared memory
}

}  // namespace

cudaError_t launch_sample(const void* x, int dt, int64_t ldx, int64_t T, int64_t V, const float* temperature,
                          const int* top_k, const float* top_p, const float* min_p, const float* u, int* ids,
                          cudaStream_t st) {
  if (T <= 0) return cudaSuccess;
  int ranks = 1;
  while (ranks < kMaxRanks && V > (int64_t)ranks * 8 * kThreads) ranks *= 2;
  const int64_t warps = (int64_t)ranks * (kThreads / 32);
  SampleArgs a{x, ldx, (int)V, (int)(((V + warps - 1) / warps + 31) / 32 * 32), temperature, top_k, top_p, min_p, u, ids};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(T * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  auto go = [&](auto k) {
    return cudaLaunchKernelEx(&cfg, k, a);
  };
  return dt == 0 ? go(sample_kernel<0>) : dt == 1 ? go(sample_kernel<1>) : go(sample_kernel<2>);
}

}  // namespace rtd
