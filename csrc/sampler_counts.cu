// Sampling one token per row from given random numbers (sm_100a): temperature, top-k, min-p and top-p,
// exact to 64 bits, from one read of the logits.
//
// A 16-bit logit has only 65,536 values. The kernel counts how often a row holds each of them; everything
// the sampler asks is then a function of the counts. In the order of descending value (ties by index) the
// candidates are a prefix of the row: the first top_k tokens, of these the ones with
// exp((x - max) / T) >= min_p, of these the ones whose preceding mass is below top_p times their mass. So
// each cut is one search for a position by count or by cumulative mass, and the draw is a fourth: the first
// position whose cumulative mass exceeds u times the mass that is left. It names a value and a rank among the
// tokens of that value; a second look at the row (from L2) finds that token. There is no sort, one 64-bit
// exponential per value that occurs, and only integer atomics, so a result does not depend on their order.
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"

namespace accerl {

constexpr int kCntThreads = 1024;
constexpr int kCntWarps = kCntThreads / 32;
constexpr int kCntWords = 32768;              // 65,536 16-bit counters, two to a word
constexpr int kCntGroups = 1024;              // of 64 neighbouring values
constexpr int kCntMaxSlice = 65528;           // elements a CTA may count without overflowing 16 bits
constexpr int kCntMaxCluster = 8;
constexpr uint32_t kKeyZero = 0x8000u;        // +0; -0 is the key below and counts as +0

template <typename T>
struct Key16;  // order-preserving 16-bit keys: valid ones lie in (kNegInf, kPosInf]
template <>
struct Key16<__nv_bfloat16> {
  static constexpr uint32_t kPosInf = 0xff80u, kNegInf = 0x007fu;
  static ACCERL_DEVINL float value(uint32_t bits) { return __uint_as_float(bits << 16); }
};
template <>
struct Key16<__half> {
  static constexpr uint32_t kPosInf = 0xfc00u, kNegInf = 0x03ffu;
  static ACCERL_DEVINL float value(uint32_t bits) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  }
};
ACCERL_DEVINL uint32_t key_bits(uint32_t key) { return (key & 0x8000u) ? key ^ 0x8000u : key ^ 0xffffu; }

// 0xffff in each half whose sign bit is set
ACCERL_DEVINL uint32_t sign_masks(uint32_t v) {
  uint32_t r;
  asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(r) : "r"(v));
  return r;
}

ACCERL_DEVINL uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
ACCERL_DEVINL double ld_cluster_f64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}
ACCERL_DEVINL void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
ACCERL_DEVINL void st_cluster_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}

ACCERL_DEVINL double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
ACCERL_DEVINL double warp_scan_f64(double v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  return v;
}
ACCERL_DEVINL uint32_t warp_scan_u32(uint32_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  return v;
}

struct CountShared {
  uint32_t cnt[kCntGroups];  // leader: tokens per group, then up to the group's end
  double own[kCntGroups];    // leader: their mass
  double mass[kCntGroups];   // leader: the mass up to the group's end
  double lse[kCntMaxCluster][kCntWarps];  // leader: partial sums of exp(x - max)
  uint32_t warp_u[kCntWarps];
  double warp_d[kCntWarps];
  uint32_t max_key;               // of this CTA's slice
  uint32_t sel_key, sel_rank;     // leader: the drawn value and the rank among its tokens
  float logprob;                  // leader
};

// The row's settings and how a value turns into a weight.
template <typename T>
struct RowWeights {
  double t;
  double min_p;
  float max;
  uint32_t max_key;
  ACCERL_DEVINL double weight(uint32_t key) const {
    if (key == max_key) return 1.0;
    if (isinf(max)) return 0.0;
    return exp((static_cast<double>(Key16<T>::value(key_bits(key))) - static_cast<double>(max)) / t);
  }
  ACCERL_DEVINL bool kept(uint32_t key, double w) const { return key == max_key || !(min_p > 0.0) || w >= min_p; }
  ACCERL_DEVINL double plain(uint32_t key) const {  // exp(x - max): the mass at temperature 1
    if (key == max_key) return 1.0;
    if (isinf(max)) return 0.0;
    return exp(static_cast<double>(Key16<T>::value(key_bits(key))) - static_cast<double>(max));
  }
};

// Tokens of keys (2 w + 1, 2 w) of counter word w over the whole cluster.
template <typename T>
ACCERL_DEVINL uint2 cluster_counts(uint32_t hist_addr, uint32_t w, int csize) {
  uint32_t hi = 0, lo = 0;
  for (int c = 0; c < csize; ++c) {
    uint32_t base;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(base) : "r"(hist_addr), "r"(c));
    const uint32_t v = ld_cluster_u32(base + w * 4);
    lo += v & 0xffffu;
    hi += v >> 16;
    if (w == (kKeyZero >> 1)) lo += ld_cluster_u32(base + (w - 1) * 4) >> 16;  // -0 counts as +0
  }
  if (w == (kKeyZero >> 1) - 1) hi = 0;
  return make_uint2(hi, lo);
}

// A group's 64 values, two per lane in descending order: counts of the kept tokens and weights.
template <typename T>
struct GroupLane {
  uint32_t c0, c1;
  double w0, w1;
};
template <typename T>
ACCERL_DEVINL GroupLane<T> load_group(const RowWeights<T>& rw, uint32_t hist_addr, int g, int lane, int csize) {
  GroupLane<T> o;
  const uint32_t word = static_cast<uint32_t>(kCntGroups - 1 - g) * 32 + 31 - lane;
  const uint2 c = cluster_counts<T>(hist_addr, word, csize);
  o.w0 = o.w1 = 0.0;
  o.c0 = o.c1 = 0;
  if (c.x) {
    o.w0 = rw.weight(2 * word + 1);
    if (rw.kept(2 * word + 1, o.w0)) o.c0 = c.x;
  }
  if (c.y) {
    o.w1 = rw.weight(2 * word);
    if (rw.kept(2 * word, o.w1)) o.c1 = c.y;
  }
  return o;
}

// One row per cluster of CTAs, each counting a slice of it.
template <typename T>
__global__ void __launch_bounds__(kCntThreads, 1)
    sample_counts_kernel(const T* __restrict__ logits, long long ld, int V, const float* __restrict__ u,
                         const float* __restrict__ temperature, const int* __restrict__ top_k,
                         const float* __restrict__ top_p, const float* __restrict__ min_p,
                         long long* __restrict__ out_tokens, float* __restrict__ out_logprobs, int csize) {
  extern __shared__ uint4 dyn[];
  uint32_t* hist = reinterpret_cast<uint32_t*>(dyn);
  __shared__ CountShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();
  const long long row = blockIdx.x / csize;
  const unsigned short* x = reinterpret_cast<const unsigned short*>(logits) + row * ld;
  // positions are counted from the 16-byte boundary at or before the row, in chunks of 8
  const int head = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) >> 1);
  const int chunks = (head + V + 7) / 8;
  const int per = (chunks + csize - 1) / csize;
  const int ch0 = min(chunks, static_cast<int>(rank) * per), ch1 = min(chunks, ch0 + per);
  // chunk ch of the row; elements outside it read as negative NaN, which is below every valid key
  auto load8 = [&](int ch) -> uint4 {
    const int i0 = ch * 8 - head;
    if (i0 >= 0 && i0 + 8 <= V) return *reinterpret_cast<const uint4*>(x + i0);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int a = i0 + 2 * j, b = a + 1;
      const uint32_t lo = (a >= 0 && a < V) ? x[a] : 0xffffu, hi = (b >= 0 && b < V) ? x[b] : 0xffffu;
      w[j] = lo | (hi << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };

  for (int i = tid; i < kCntWords / 4; i += kCntThreads) dyn[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();

  // ---- count the slice ----
  uint32_t maxk = 0;
  auto count = [&](uint32_t key) {
    if (key > Key16<T>::kNegInf && key <= Key16<T>::kPosInf) {
      maxk = max(maxk, key);
      atomicAdd(&hist[key >> 1], (key & 1u) ? 0x10000u : 1u);
    }
  };
  for (int ch = ch0 + tid; ch < ch1; ch += kCntThreads) {
    const uint4 v = load8(ch);
    const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // per half: complement a negative pattern, set the top bit of a positive one
      const uint32_t key2 = vw[j] ^ (sign_masks(vw[j]) | 0x80008000u);
      count(key2 & 0xffffu);
      count(key2 >> 16);
    }
  }
  maxk = __reduce_max_sync(0xffffffffu, maxk);
  if (lane == 0) sh.warp_u[warp] = maxk;
  __syncthreads();
  if (warp == 0) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, sh.warp_u[lane]);
    if (lane == 0) sh.max_key = m;
  }
  __syncthreads();
  cluster_sync();

  RowWeights<T> rw;
  uint32_t mk = 0;
  for (int c = 0; c < csize; ++c) mk = max(mk, ld_cluster_u32(map_shared_rank(&sh.max_key, c)));
  if (mk == kKeyZero - 1) mk = kKeyZero;
  rw.max_key = mk;
  rw.max = Key16<T>::value(key_bits(mk));
  const float t = temperature[row];
  const bool greedy = !(t > 0.f);
  rw.t = greedy ? 1.0 : static_cast<double>(t);
  rw.min_p = min_p ? static_cast<double>(min_p[row]) : 0.0;
  const uint32_t hist_addr = smem_u32(hist);

  // ---- tokens and mass of every group of 64 values ----
  double lse = 0.0;
  const int gper = kCntGroups / csize;
  for (int i = warp; i < gper; i += kCntWarps) {
    const int g = static_cast<int>(rank) * gper + i;  // 0 holds the largest values
    const uint32_t word = static_cast<uint32_t>(kCntGroups - 1 - g) * 32 + 31 - lane;
    const uint2 c = cluster_counts<T>(hist_addr, word, csize);
    uint32_t n = 0;
    double m = 0.0;
    if (__any_sync(0xffffffffu, (c.x | c.y) != 0u)) {
      if (c.x) {
        const double w = rw.weight(2 * word + 1);
        lse += c.x * (t == 1.f ? w : rw.plain(2 * word + 1));
        if (rw.kept(2 * word + 1, w)) {
          n += c.x;
          m += c.x * w;
        }
      }
      if (c.y) {
        const double w = rw.weight(2 * word);
        lse += c.y * (t == 1.f ? w : rw.plain(2 * word));
        if (rw.kept(2 * word, w)) {
          n += c.y;
          m += c.y * w;
        }
      }
      n = __reduce_add_sync(0xffffffffu, n);
      m = warp_sum_f64(m);
    }
    if (lane == 0) {
      st_cluster_u32(map_shared_rank(&sh.cnt[g], 0), n);
      st_cluster_f64(map_shared_rank(&sh.own[g], 0), m);
    }
  }
  lse = warp_sum_f64(lse);
  if (lane == 0) st_cluster_f64(map_shared_rank(&sh.lse[rank][warp], 0), lse);
  __syncthreads();
  cluster_sync();

  if (rank == 0 && mk != 0u) {
    // ---- prefix sums over the groups ----
    const uint32_t c = sh.cnt[tid];
    const double m = sh.own[tid];
    const uint32_t ci = warp_scan_u32(c, lane);
    const double mi = warp_scan_f64(m, lane);
    if (lane == 31) {
      sh.warp_u[warp] = ci;
      sh.warp_d[warp] = mi;
    }
    __syncthreads();
    uint32_t cb = 0;
    double mb = 0.0;
    for (int w = 0; w < warp; ++w) {
      cb += sh.warp_u[w];
      mb += sh.warp_d[w];
    }
    sh.cnt[tid] = cb + ci;   // inclusive
    sh.mass[tid] = mb + mi;
    __syncthreads();
    if (warp == 0) {
      // first group whose inclusive prefix satisfies `f`; kCntGroups when none does
      auto find_group = [&](auto f) -> int {
        for (int g0 = 0; g0 < kCntGroups; g0 += 32) {
          const uint32_t hit = __ballot_sync(0xffffffffu, f(g0 + lane));
          if (hit) return g0 + __ffs(hit) - 1;
        }
        return kCntGroups;
      };
      const uint32_t n_all = sh.cnt[kCntGroups - 1];
      double kept = sh.mass[kCntGroups - 1];
      int k = top_k ? top_k[row] : 0;
      if (greedy || rw.min_p > 1.0) k = 1;  // the first candidate stays whatever min_p asks
      if (k > 0 && static_cast<uint32_t>(k) < n_all) {
        const int g = find_group([&](int i) { return sh.cnt[i] >= static_cast<uint32_t>(k); });
        const GroupLane<T> gl = load_group<T>(rw, hist_addr, g, lane, csize);
        const uint32_t own = gl.c0 + gl.c1;
        const uint32_t before = (g ? sh.cnt[g - 1] : 0u) + warp_scan_u32(own, lane) - own;
        // of this lane's tokens the first `take` are among the k
        const uint32_t take = static_cast<uint32_t>(max(0, min(static_cast<int>(own), k - static_cast<int>(before))));
        const uint32_t take0 = min(take, gl.c0);
        kept = (g ? sh.mass[g - 1] : 0.0) + warp_sum_f64(take0 * gl.w0 + (take - take0) * gl.w1);
      }
      // position whose cumulative mass first reaches (strict: exceeds) `limit`
      auto find_mass = [&](double limit, bool strict, uint32_t& key, uint32_t& nth, double& cum) {
        int g = find_group([&](int i) {
          return sh.own[i] > 0.0 && (strict ? sh.mass[i] > limit : sh.mass[i] >= limit);
        });
        if (g == kCntGroups)  // rounding at the very end: the last group that has mass
          for (int g0 = kCntGroups - 32; g0 >= 0 && g == kCntGroups; g0 -= 32) {
            const uint32_t hit = __ballot_sync(0xffffffffu, sh.own[g0 + lane] > 0.0);
            if (hit) g = g0 + 31 - __clz(hit);
          }
        const GroupLane<T> gl = load_group<T>(rw, hist_addr, g, lane, csize);
        const double m0 = gl.c0 * gl.w0, m1 = gl.c1 * gl.w1;
        const double incl = warp_scan_f64(m0 + m1, lane);
        double at = __shfl_up_sync(0xffffffffu, incl, 1);
        at = (g ? sh.mass[g - 1] : 0.0) + (lane ? at : 0.0);
        const bool first = m0 > 0.0 && (strict ? at + m0 > limit : at + m0 >= limit);
        const bool second = m1 > 0.0 && (strict ? at + m0 + m1 > limit : at + m0 + m1 >= limit);
        uint32_t hit = __ballot_sync(0xffffffffu, first || second);
        bool clamp = false;
        int src;
        if (hit) {
          src = __ffs(hit) - 1;
        } else {  // rounding inside the group: its last value that has mass
          src = 31 - __clz(__ballot_sync(0xffffffffu, m0 > 0.0 || m1 > 0.0));
          clamp = true;
        }
        const bool use0 = clamp ? !(m1 > 0.0) : first;
        const uint32_t cc = use0 ? gl.c0 : gl.c1;
        const double ww = use0 ? gl.w0 : gl.w1, a = use0 ? at : at + m0;
        const double q = (limit - a) / ww;
        double j = strict ? floor(q) : ceil(q) - 1.0;  // 0-based position among the equal tokens
        j = clamp ? static_cast<double>(cc) - 1.0 : fmin(fmax(j, 0.0), static_cast<double>(cc) - 1.0);
        const uint32_t word = static_cast<uint32_t>(kCntGroups - 1 - g) * 32 + 31 - lane;
        key = __shfl_sync(0xffffffffu, 2 * word + (use0 ? 1u : 0u), src);
        nth = __shfl_sync(0xffffffffu, static_cast<uint32_t>(j), src);
        cum = __shfl_sync(0xffffffffu, a + (j + 1.0) * ww, src);
      };
      uint32_t key, nth;
      double cum;
      const double p = top_p ? static_cast<double>(top_p[row]) : 1.0;
      if (p < 1.0 && !greedy) {
        find_mass(fmax(p, 0.0) * kept, false, key, nth, cum);
        kept = fmin(cum, kept);
      }
      const double uu = fmin(fmax(static_cast<double>(u[row]), 0.0), 1.0 - 0x1p-53);  // NaN: 0
      find_mass(greedy ? 0.0 : uu * kept, true, key, nth, cum);
      double s = 0.0;
      for (int i = 0; i < csize; ++i) s += sh.lse[i][lane];
      s = warp_sum_f64(s);
      if (lane == 0) {
        sh.sel_key = key;
        sh.sel_rank = nth;
        const double d = key == mk ? 0.0 : static_cast<double>(Key16<T>::value(key_bits(key))) - static_cast<double>(rw.max);
        sh.logprob = static_cast<float>(d - log(s));
      }
    }
  }
  __syncthreads();
  cluster_sync();

  // ---- the token: the sel_rank-th of the row with the drawn value ----
  const uint32_t key = ld_cluster_u32(map_shared_rank(&sh.sel_key, 0));
  const uint32_t nth = ld_cluster_u32(map_shared_rank(&sh.sel_rank, 0));
  const float lp = __uint_as_float(ld_cluster_u32(map_shared_rank(&sh.logprob, 0)));
  uint32_t before = 0, own = 0;
  if (mk != 0u) {
    for (int c = 0; c <= static_cast<int>(rank); ++c) {
      const uint32_t base = map_shared_rank(hist, c);
      uint32_t n = ld_cluster_u32(base + (key >> 1) * 4);
      n = (key & 1u) ? n >> 16 : n & 0xffffu;
      if (key == kKeyZero) n += ld_cluster_u32(base + ((key >> 1) - 1) * 4) >> 16;
      if (c < static_cast<int>(rank)) before += n;
      else own = n;
    }
  }
  __syncthreads();
  cluster_sync();  // no CTA leaves while another may read its counts
  if (mk == 0u) {  // nothing to choose from
    if (rank == 0 && tid == 0) {
      out_tokens[row] = 0;
      out_logprobs[row] = -INFINITY;
    }
    return;
  }
  if (nth < before || nth >= before + own) return;
  const uint32_t want = key_bits(key), mask = key == kKeyZero ? 0x7fffu : 0xffffu;
  auto matches = [&](uint4 v) -> uint32_t {  // bit i: element i of the chunk is one of them
    const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
    uint32_t b = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      b |= ((vw[j] & mask) == want ? 1u : 0u) << (2 * j);
      b |= (((vw[j] >> 16) & mask) == want ? 1u : 0u) << (2 * j + 1);
    }
    return b;
  };
  // each warp counts a contiguous part of the slice; the one that holds the token goes through its part again
  const int wper = (ch1 - ch0 + kCntWarps - 1) / kCntWarps;
  const int w0 = min(ch1, ch0 + warp * wper), w1 = min(ch1, w0 + wper);
  uint32_t n = 0;
  for (int ch = w0 + lane; ch < w1; ch += 32) n += __popc(matches(load8(ch)));
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();
  if (lane == 0) sh.warp_u[warp] = n;
  __syncthreads();
  uint32_t at = before;
  for (int w = 0; w < warp; ++w) at += sh.warp_u[w];
  if (nth < at || nth >= at + n) return;
  for (int c0 = w0; c0 < w1; c0 += 32) {
    const uint32_t b = c0 + lane < w1 ? matches(load8(c0 + lane)) : 0u;
    const uint32_t mine = __popc(b);
    const uint32_t incl = warp_scan_u32(mine, lane);
    const uint32_t excl = at + incl - mine;
    if (nth >= excl && nth < excl + mine) {
      uint32_t bits = b;
      for (uint32_t i = excl; i < nth; ++i) bits &= bits - 1;
      out_tokens[row] = static_cast<long long>(c0 + lane) * 8 - head + __ffs(bits) - 1;
      out_logprobs[row] = lp;
    }
    at += __shfl_sync(0xffffffffu, incl, 31);
    if (nth < at) break;
  }
}

namespace {
template <typename T>
int launch_sample_counts(const void* logits, long long ld, int rows, int V, const float* u, const float* temperature,
                         const int* top_k, const float* top_p, const float* min_p, long long* tokens, float* logprobs,
                         int csize, cudaStream_t s) {
  constexpr int smem = kCntWords * 4;
  auto kern = sample_counts_kernel<T>;
  cudaError_t e = smem_attr_once<sample_counts_kernel<T>>(smem);
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = csize;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * csize, 1, 1);
  cfg.blockDim = dim3(kCntThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, reinterpret_cast<const T*>(logits), ld, V, u, temperature,
                                             top_k, top_p, min_p, tokens, logprobs, csize));
}
}  // namespace
}  // namespace accerl

// One token per row of logits [rows, V] (half: 0 bf16, 1 fp16; row stride ld) from u [rows]. top_k, top_p and
// min_p may be null (off). -2: V above what a cluster can count.
extern "C" int accerl_sample_counts(const void* logits, long long ld, int half, int rows, int V, const float* u,
                                    const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                                    long long* tokens, float* logprobs, cudaStream_t s) {
  using namespace accerl;
  if (rows <= 0) return 0;
  if (V <= 0) return -1;
  // a slice holds its chunks of 8 and may start 7 elements before the row
  auto slice = [&](int c) { return ((V + 14) / 8 + c - 1) / c * 8; };
  int csize = 1;
  while (csize < kCntMaxCluster && slice(csize) > kCntMaxSlice) csize *= 2;
  if (slice(csize) > kCntMaxSlice) return -2;
  if (static_cast<long long>(rows) * csize > 0x7fffffffll) return -3;
  // few rows: spread each over more SMs while its slices stay long enough to count
  while (csize < kCntMaxCluster && static_cast<long long>(rows) * csize * 2 <= device_sm_count() && slice(csize) > 8192)
    csize *= 2;
  if (half) return launch_sample_counts<__half>(logits, ld, rows, V, u, temperature, top_k, top_p, min_p, tokens, logprobs, csize, s);
  return launch_sample_counts<__nv_bfloat16>(logits, ld, rows, V, u, temperature, top_k, top_p, min_p, tokens, logprobs, csize, s);
}
