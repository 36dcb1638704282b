// Sampling one token per row from given random numbers (sm_100a): temperature, top-k, min-p and top-p,
// exact to 64 bits, from one read of the logits.
//
// A 16-bit logit has only 65,536 values. The kernel counts how often a row holds each of them; everything
// the sampler asks is then a function of the counts. In the order of descending value (ties by index) the
// candidates are a prefix of the row: the first top_k tokens, of these the ones with
// exp((x - max) / T) >= min_p, of these the ones whose preceding mass is below top_p times their mass. So
// each cut is one search for a position by count or by cumulative mass, and the draw is a last one: the first
// position whose cumulative mass exceeds u times the mass that is left. It names a value and a rank among the
// tokens of that value; a second look at the row (from L2) finds that token. There is no sort, one 64-bit
// exponential per four neighbouring values (the others follow by the ratio of evenly spaced ones), and only integer
// atomics, so a result does not depend on their order.
//
// Counters for all values would not fit an SM. The kernel counts a window of the values that logits take (bf16: zero
// and 2^-40 to 2^24; fp16: below 128, each sign) in 64 KB (176 KB). Lower values, masks of the type's lowest value
// among them, are left out where they weigh nothing; a row with any other value takes the slow path, which counts
// all values, window by window.
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"

namespace accerl {

constexpr int kCntGroups = 1024;              // at most: groups of 64 neighbouring values
constexpr int kCntMaxCluster = 8;
// tokens further below the largest logit than this many temperatures weigh nothing: each holds less than e^-60 = 9e-27
// of the largest one's mass, all of a row's together less than 2e-17 even at 2^31 tokens (1.4e-21 at 151936), below
// half a step of a 64-bit sum
constexpr double kCntNegligible = 60.0;

// Order-preserving 16-bit keys of the finite values and +inf: (kNegInf, kPosInf].
// The window holds kSlots magnitude patterns from kBase on (fp16: without the first, zero). Its bins ascend with
// the value: [64, 64 + kSlots) negative, then as many positive ones; bin 0, whose group of 64 has no other use, is
// zero's. kBase and kSlots are multiples of 4, so four neighbouring bins from a multiple of 4 on are evenly spaced.
template <typename T>
struct Key16;
template <>
struct Key16<__nv_bfloat16> {
  static constexpr uint32_t kInf = 0x7f80u, kPosInf = 0xff80u, kNegInf = 0x007fu;
  static constexpr uint32_t kBase = (127u - 40u) << 7, kSlots = 64u << 7, kMantissa = 7;
  static constexpr bool kOneRow = false;  // the counters leave room for two blocks on an SM
  static ACCERL_DEVINL float value(uint32_t bits) { return __uint_as_float(bits << 16); }
  static ACCERL_DEVINL uint32_t bits(float v) { return __float_as_uint(v) >> 16; }  // of a neighbour: cut off
  static ACCERL_DEVINL uint32_t max2(uint32_t a, uint32_t b) {  // of both halves; a NaN loses
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  // n += elements of the 8 words' halves equal to the value in both halves of `want` (0 equals -0, NaN nothing)
  static ACCERL_DEVINL void count_equal(const uint4 (&v)[8], uint32_t want, uint32_t& n) {
    const __nv_bfloat162 k = *reinterpret_cast<__nv_bfloat162*>(&want);
    __nv_bfloat162 sum = __float2bfloat162_rn(0.f);  // at most 32 a half: exact
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) sum = __hadd2(sum, __heq2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), k));
    }
    n += static_cast<uint32_t>(__low2float(sum) + __high2float(sum));
  }
  static ACCERL_DEVINL uint32_t min2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmin2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  // halves that are not 0 where w, whose magnitude is t - 0x8000 + kBase, is not in the window
  static ACCERL_DEVINL uint32_t outside(uint32_t w, uint32_t t) { return (t & 0xe000e000u) ^ 0x80008000u; }
  // top bit of the halves whose magnitude lies below the window
  static ACCERL_DEVINL uint32_t below(uint32_t t) { return ~t; }
};
template <>
struct Key16<__half> {
  static constexpr uint32_t kInf = 0x7c00u, kPosInf = 0xfc00u, kNegInf = 0x03ffu;
  static constexpr uint32_t kBase = 0u, kSlots = 22u << 10, kMantissa = 10;
  static constexpr bool kOneRow = true;
  static ACCERL_DEVINL float value(uint32_t bits) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  }
  static ACCERL_DEVINL uint32_t bits(float v) { return __half_as_ushort(__float2half_rn(v)); }
  static ACCERL_DEVINL uint32_t max2(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  static ACCERL_DEVINL void count_equal(const uint4 (&v)[8], uint32_t want, uint32_t& n) {
    const __half2 k = *reinterpret_cast<__half2*>(&want);
    __half2 sum = __float2half2_rn(0.f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) sum = __hadd2(sum, __heq2(*reinterpret_cast<const __half2*>(&w[i]), k));
    }
    n += static_cast<uint32_t>(__low2float(sum) + __high2float(sum));
  }
  static ACCERL_DEVINL uint32_t min2(uint32_t a, uint32_t b) {
    const __half2 m = __hmin2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  static ACCERL_DEVINL uint32_t below(uint32_t t) { return ~(t - 0x00010001u); }
  static ACCERL_DEVINL uint32_t outside(uint32_t w, uint32_t t) {
    return (~(t - 0x00010001u) | ((w & 0x7fff7fffu) + (0x8000u - kSlots) * 0x00010001u)) & 0x80008000u;
  }
};
// 0xffff in each half whose top bit is set
ACCERL_DEVINL uint32_t half_masks(uint32_t v) {
  uint32_t r;
  asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(r) : "r"(v));
  return r;
}
ACCERL_DEVINL uint32_t key_bits(uint32_t key) { return (key & 0x8000u) ? key ^ 0x8000u : key ^ 0xffffu; }
ACCERL_DEVINL uint32_t bits_key(uint32_t bits) { return (bits & 0x8000u) ? bits ^ 0xffffu : bits ^ 0x8000u; }
template <typename T>
ACCERL_DEVINL uint32_t bin_key(uint32_t b) {
  constexpr uint32_t S = Key16<T>::kSlots, base = Key16<T>::kBase;
  if (b < 64u) return 0x8000u;
  return b >= 64u + S ? 0x8000u + base + (b - 64u - S) : 0x7fffu - base - (63u + S - b);
}
template <typename T>
ACCERL_DEVINL uint32_t key_bin(uint32_t key) {
  constexpr uint32_t S = Key16<T>::kSlots, base = Key16<T>::kBase;
  if (key == 0x8000u) return 0u;
  return key > 0x8000u ? key - 0x8000u - base + 64u + S : key + base + 64u + S - 0x8000u;
}
// Group p (bins 64 p ..) of the window in descending order of its values: positive, zero, negative; and back.
template <typename T>
ACCERL_DEVINL int window_order(int p) {
  constexpr int half = static_cast<int>(Key16<T>::kSlots / 64);
  return p == 0 ? half : (p > half ? 2 * half - p : 2 * half + 1 - p);
}
template <typename T>
ACCERL_DEVINL int window_group(int g) {
  constexpr int half = static_cast<int>(Key16<T>::kSlots / 64);
  return g == half ? 0 : (g < half ? 2 * half - g : 2 * half + 1 - g);
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
ACCERL_DEVINL void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
ACCERL_DEVINL void cluster_wait_all() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <typename V>
ACCERL_DEVINL V* peer(V* p, int rank) {  // the same shared variable in CTA `rank` of the cluster
  return static_cast<V*>(__cluster_map_shared_rank(p, rank));
}

struct CountShared {
  // leader: tokens and mass per group (0 holds the largest values), then both up to the group's end
  uint32_t cnt[kCntGroups];
  double own[kCntGroups];
  double mass[kCntGroups];
  double lse[kCntMaxCluster * 32];  // leader: the warps' partial sums of exp(x - max)
  uint32_t warp_u[3][32];
  double warp_d[32];
  double exp2_table[64];            // 2^(j / 64)
  double ratio[2][65];              // of neighbouring values' masses by binade of the window (and the padding): at T, at 1
  // of every CTA's slice: the largest key, whether a value lies below the window, whether one escapes it otherwise
  uint32_t max_key[kCntMaxCluster], any_low[kCntMaxCluster], escape[kCntMaxCluster];
  uint32_t group_cnt[64];                     // slow path: tokens of a group's values
  int found[3];                               // the searches' groups (top-k, top-p, draw)
  double log_sum;                             // leader: log of the sum of exp(x - max)
  uint32_t key, nth;                          // its value and rank among the value's tokens; before: of the last candidate
  double cum;                                 // mass up to and with that token
  int nth_here;                               // rank of the drawn token within this CTA's slice, or -1
  float logprob;
  float set_t, set_u, set_p, set_min;         // the row's settings
  int set_k;
  uint32_t left_out;                          // counts nothing of use
};

// a count as a 64-bit float without the slow conversion
ACCERL_DEVINL double count_f64(uint32_t n) { return __hiloint2double(0x43300000, static_cast<int>(n)) - 0x1p52; }

// 2^(y / 64) for y <= 0: n = round(y), the table for n mod 64, and the Taylor series of the rest, |r| <= ln 2 / 128,
// whose sixth term is below 2^-54. The argument's rounding costs at most a relative |y| 2^-59, so a weight is
// within 2^-52 of the largest one's unit. Below 2^-1020: 0.
ACCERL_DEVINL double exp2_64th(double y, const double* table) {
  const double t = y + 0x1.8p52;
  const int n = __double2loint(t);
  const double r = (y - (t - 0x1.8p52)) * (0.693147180559945309417 / 64);
  // (1 + r) + r^2 ((1/2 + r/6) + r^2 (1/24 + r/120)): the dependent operations are what this costs
  const double r2 = r * r;
  const double hi = __fma_rn(r2, __fma_rn(r, 1.0 / 120, 1.0 / 24), __fma_rn(r, 1.0 / 6, 0.5));
  const double q = __fma_rn(r2, hi, 1.0 + r) * table[n & 63];
  const double v = __hiloint2double(__double2hiint(q) + (n >> 6) * 0x100000, __double2loint(q));
  return y < -64.0 * 1020 ? 0.0 : v;
}
constexpr double kLog2e64 = 64 * 1.44269504088896340736;

// The row's settings and how a value turns into a weight.
template <typename T>
struct RowWeights {
  double scale;  // 64 log2(e) / T
  float max;     // the row's largest logit
  uint32_t max_key, keep_key;  // its key, and that of the smallest value that min_p keeps
  const double* table;
  ACCERL_DEVINL double gap(uint32_t key) const {
    return static_cast<double>(Key16<T>::value(key_bits(key))) - static_cast<double>(max);
  }
  ACCERL_DEVINL double mass(uint32_t key, double sc) const {
    // an infinite maximum leaves nothing to the others (whose gap is -inf); at an infinite temperature (sc = 0)
    // every finite gap weighs 1
    const double y = gap(key) * sc;
    const double w = exp2_64th(y > -64.0 * 1021 ? y : -64.0 * 1021, table);  // NaN (inf * 0): the limit
    return key == max_key ? 1.0 : (isinf(max) ? 0.0 : w);
  }
  ACCERL_DEVINL double weight(uint32_t key) const { return mass(key, scale); }
  ACCERL_DEVINL double plain(uint32_t key) const { return mass(key, kLog2e64); }  // exp(x - max)
  // masses of four neighbouring keys, ascending; `even`: equally spaced, each is the one above it times the ratio r,
  // from the largest that is not above the row's maximum on
  ACCERL_DEVINL void mass4(const uint32_t (&key)[4], bool even, double r, double sc, double (&w)[4]) const {
    if (even) {
      // `above` of the keys lie above the maximum and hold nothing
      const uint32_t above = key[3] > max_key ? min(key[3] - max_key, 4u) : 0u;
      const double m0 = mass(key[3] - above, sc), r2 = r * r;
      w[3] = m0;
      w[2] = m0 * r;
      w[1] = m0 * r2;
      w[0] = w[2] * r2;
      for (uint32_t i = 0; i < above; ++i) {  // only where the maximum is
        w[0] = w[1];
        w[1] = w[2];
        w[2] = w[3];
        w[3] = 0.0;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = key[j] > max_key ? 0.0 : mass(key[j], sc);
    }
  }
  ACCERL_DEVINL bool kept(uint32_t key) const { return key >= keep_key; }
  // The smallest key whose weight is at least min_p, by the whole warp: found once, so that every later question is one
  // of whole numbers and has one answer. `lo` is not kept, `hi` is; all lanes but 0 try a key between them. The first
  // try is around max + T log(min_p), which all but always holds the border; then the range shrinks by 32 a turn.
  ACCERL_DEVINL uint32_t smallest_kept(float min_p, float t, int lane) const {
    int lo = static_cast<int>(Key16<T>::kNegInf), hi = static_cast<int>(max_key), step = 1;
    const float near = max + t * logf(fminf(min_p, 1.f));
    const uint32_t near_bits = Key16<T>::bits(near);
    int top = (near_bits & 0x7fffu) > Key16<T>::kInf ? hi : min(hi, static_cast<int>(bits_key(near_bits)) + 16);
    while (hi - lo > 1) {
      const int key = top - lane * step;
      const uint32_t yes =
          __ballot_sync(0xffffffffu, key >= hi || (key > lo && weight(static_cast<uint32_t>(key)) >= static_cast<double>(min_p)));
      const int n = yes == 0xffffffffu ? 32 : __ffs(~yes) - 1;  // so many from the top are kept
      if (n > 0) hi = min(hi, top - (n - 1) * step);
      if (n < 32) lo = ::max(lo, top - n * step);
      step = (hi - lo + 31) / 32;
      top = hi;
    }
    return static_cast<uint32_t>(hi);
  }
};

// One row per cluster of CTAs, each counting a slice of it. Two passes over the row, the second for half of it on
// average and from L2; between them nothing depends on V. Measured (bf16, V = 151936): 256 rows 53 us, of which the
// reads need 12: shared memory adds up 32 counters at random banks in 3 to 4 clocks, so two rows on an SM, counted one
// behind the other, take 27 us, the sums over the groups and the searches 16, the token's place 5. 1 row in 16 us, nearly
// all of it latency (barriers of the cluster, sums of 64-bit floats, dependent searches; min-p's border is 0.4 of it). fp16's wider range of
// values in use means 350 pairs of groups: 100 rows of 32003 take 26 us, 11 of them there. An SM's 1024 threads have 64
// registers each, a few too few: 20 bytes a thread spill (fp16: 4).
template <typename T, int kCntThreads>
__global__ void __launch_bounds__(kCntThreads, 1024 / kCntThreads)
    sample_counts_kernel(const T* __restrict__ logits, long long ld, int V, const float* __restrict__ u,
                         const float* __restrict__ temperature, const int* __restrict__ top_k,
                         const float* __restrict__ top_p, const float* __restrict__ min_p,
                         long long* __restrict__ out_tokens, float* __restrict__ out_logprobs, int csize) {
  constexpr uint32_t S = Key16<T>::kSlots, kBins = 64 + 2 * S;
  constexpr int kCntWarps = kCntThreads / 32, kCntPer = kCntGroups / kCntThreads;
  extern __shared__ uint4 dyn[];
  uint32_t* hist = reinterpret_cast<uint32_t*>(dyn);  // kBins counters and 64 more that stay zero
  __shared__ CountShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const long long row = blockIdx.x / csize;
  const unsigned short* x = reinterpret_cast<const unsigned short*>(logits) + row * ld;
  // positions are counted from the 16-byte boundary at or before the row, in chunks of 8
  const int head = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) >> 1);
  const int chunks = (head + V + 7) / 8;
  const int per = (chunks + csize - 1) / csize;
  const int ch0 = min(chunks, rank * per), ch1 = min(chunks, ch0 + per);
  // chunk ch of the row; elements outside it read as NaN, which nothing counts
  auto load2 = [&](int ch, int j) -> uint32_t {  // two elements of it
    const int a = ch * 8 - head + 2 * j, b = a + 1;
    const uint32_t lo = (a >= 0 && a < V) ? x[a] : 0xffffu, hi = (b >= 0 && b < V) ? x[b] : 0xffffu;
    return lo | (hi << 16);
  };
  auto load8 = [&](int ch) -> uint4 {
    const int i0 = ch * 8 - head;
    if (i0 >= 0 && i0 + 8 <= V) return *reinterpret_cast<const uint4*>(x + i0);
    return make_uint4(load2(ch, 0), load2(ch, 1), load2(ch, 2), load2(ch, 3));
  };
  // chunks [whole0, whole1) lie inside the row
  const int whole0 = head ? 1 : 0, whole1 = (head + V) / 8;
  constexpr int kAhead = 2;
  const uint4* src = reinterpret_cast<const uint4*>(x - head);
  // this thread's kAhead whole chunks from c on; behind `end` NaN, which nothing counts
  auto load_batch = [&](uint4 (&v)[kAhead], int c, int end) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int ch = c + j * kCntThreads;
      v[j] = ch < end ? __ldg(src + ch) : make_uint4(~0u, ~0u, ~0u, ~0u);
    }
  };
  auto load_first = [&](uint4 (&v)[kAhead], int a, int b) { load_batch(v, max(a, whole0) + tid, min(b, whole1)); };
  // f(word) for every two elements of the chunks [a, b), the next batch on its way while one is worked on; `v`
  // holds the first. The row's ends, which are not whole chunks, come after the loop: it has no other tests.
  auto for_each = [&](uint4 (&v)[kAhead], int a, int b, auto f) {
    const int end = min(b, whole1);
#pragma unroll 1
    for (int c = max(a, whole0) + tid; c < end; c += kAhead * kCntThreads) {
      uint4 next[kAhead];
      load_batch(next, c + kAhead * kCntThreads, end);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        f(v[j].x);
        f(v[j].y);
        f(v[j].z);
        f(v[j].w);
        v[j] = next[j];
      }
    }
    if (tid < 8) {  // a word each
      const int ch = tid < 4 ? 0 : whole1;  // the same one where the row ends in its first chunk
      if (ch >= a && ch < b && (tid < 4 ? whole0 == 1 : whole1 < chunks && whole1 >= whole0)) f(load2(ch, tid & 3));
    }
  };
  auto valid_key = [](uint32_t w) -> int {  // -1: -inf or NaN
    const uint32_t bits = w & 0xffffu, key = bits_key(bits == 0x8000u ? 0u : bits);
    return key > Key16<T>::kNegInf && key <= Key16<T>::kPosInf ? static_cast<int>(key) : -1;
  };
  auto clear = [&]() {
    for (int i = tid; i < static_cast<int>((kBins + 64) / 4); i += kCntThreads) dyn[i] = make_uint4(0, 0, 0, 0);
  };
  auto add = [&](uint32_t bin) { atomicAdd(&hist[bin], 1u); };
  // the same with a select, not a branch: what is left out goes to one word, which the hardware adds up per warp
  const uint32_t hist_smem = smem_u32(hist), left_out = smem_u32(&sh.left_out);
  auto add_unless = [&](uint32_t skip, uint32_t bin) {
    const uint32_t at = skip ? left_out : hist_smem + bin * 4u;
    asm volatile("red.shared::cta.add.u32 [%0], 1;" ::"r"(at) : "memory");
  };

  // the first loads travel while the counters are cleared
  uint4 batch[kAhead];
  load_first(batch, ch0, ch1);
  __syncwarp();
  cluster_arrive_relaxed();
  clear();
  if (tid < 3) sh.found[tid] = kCntGroups;
  if (tid == 0) {
    sh.nth_here = -1;
    sh.key = 0u;  // no cut
    sh.nth = ~0u;
  }
  if (tid == 192) {  // the row's settings, out of the registers while the slice is counted
    sh.set_t = temperature[row];
    sh.set_u = u[row];
    sh.set_p = top_p ? top_p[row] : 1.f;
    sh.set_min = min_p ? min_p[row] : 0.f;
    sh.set_k = top_k ? top_k[row] : 0;
  }
  if (tid < 64) sh.exp2_table[tid] = exp2(tid / 64.0);
  if (tid >= 64 && tid < 192 && ((tid - 64) & 63) < static_cast<int>(S >> Key16<T>::kMantissa)) {
    const uint32_t first = Key16<T>::kBase + (((tid - 64) & 63) << Key16<T>::kMantissa);
    const double step = static_cast<double>(Key16<T>::value(first + 1) - Key16<T>::value(first));
    const float t = tid < 128 ? temperature[row] : 1.f;
    sh.ratio[(tid - 64) >> 6][(tid - 64) & 63] = exp(-step / (t > 0.f ? static_cast<double>(t) : 1.0));
  }
  __syncthreads();

  // ---- count the slice ----
  uint32_t max2 = 0xffffffffu, min2 = 0xffffffffu, low2 = 0;  // NaN: loses to everything
  for_each(batch, ch0, ch1, [&](uint32_t w) {
    // Both halves at once, with plain 32-bit operations and no branch (instructions are what bounds this loop): no sum
    // of a half carries or borrows. With slot = magnitude - kBase, t = 0x8000 + slot, its complement for a negative
    // value is 0x7fff - slot, and v - (0x8000 - 64 - kSlots) is the bin of either sign.
    constexpr uint32_t kOff = 0x8000u - 64u - S;
    const uint32_t t = (w | 0x80008000u) - Key16<T>::kBase * 0x00010001u, v = t ^ half_masks(w);
    const uint32_t out = Key16<T>::outside(w, t);
    add_unless(out & 0xffffu, (v & 0xffffu) - kOff);
    add_unless(out & 0xffff0000u, (v >> 16) - kOff);
    max2 = Key16<T>::max2(max2, w);
    min2 = Key16<T>::min2(min2, w);
    low2 |= Key16<T>::below(t);
  });
  uint32_t escape = 0;
  if (low2 & 0x80008000u) {  // zeros, or magnitudes below the window, among the elements this thread has seen
    load_first(batch, ch0, ch1);
    for_each(batch, ch0, ch1, [&](uint32_t w) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t mag = (w >> (16 * h)) & 0x7fffu;
        if (mag == 0u) add(0u);
        else if (static_cast<int>(mag) < static_cast<int>(Key16<T>::kBase)) escape = 1u;
      }
    });
  }
  // the largest and the smallest of both halves as keys (0: there is nothing but NaN)
  auto one_key = [](uint32_t bits) -> uint32_t {
    bits &= 0xffffu;
    return (bits & 0x7fffu) > Key16<T>::kInf ? 0u : bits_key((bits & 0x7fffu) ? bits : 0u);
  };
  uint32_t max_key = one_key(Key16<T>::max2(max2, max2 >> 16));
  if (max_key <= Key16<T>::kNegInf) max_key = 0u;
  if (max_key >= 0x8000u + Key16<T>::kBase + S) escape = 1u;  // above the window
  // whether anything (-inf at least) lies below the window
  const uint32_t min_key = one_key(Key16<T>::min2(min2, min2 >> 16));
  uint32_t any_low = min_key != 0u && min_key <= 0x7fffu - Key16<T>::kBase - S ? 1u : 0u;
  max_key = __reduce_max_sync(0xffffffffu, max_key);
  any_low = __reduce_max_sync(0xffffffffu, any_low);
  escape = __reduce_max_sync(0xffffffffu, escape);
  if (lane == 0) {
    sh.warp_u[0][warp] = max_key;
    sh.warp_u[1][warp] = any_low;
    sh.warp_u[2][warp] = escape;
  }
  __syncthreads();
  cluster_wait_all();  // everybody has started
  if (warp == 0) {
    const bool has = lane < kCntWarps;
    max_key = __reduce_max_sync(0xffffffffu, has ? sh.warp_u[0][lane] : 0u);
    any_low = __reduce_max_sync(0xffffffffu, has ? sh.warp_u[1][lane] : 0u);
    escape = __reduce_max_sync(0xffffffffu, has ? sh.warp_u[2][lane] : 0u);
    if (lane < csize) {  // to every CTA of the cluster
      CountShared* o = peer(&sh, lane);
      o->max_key[rank] = max_key;
      o->any_low[rank] = any_low;
      o->escape[rank] = escape;
    }
  }
  __syncthreads();
  cluster_sync();

  // ---- the row's largest value, and whether the window holds all that matters ----
  max_key = any_low = escape = 0;
  for (int c = 0; c < csize; ++c) {
    max_key = max(max_key, sh.max_key[c]);
    any_low |= sh.any_low[c];
    escape |= sh.escape[c];
  }
  const float t = sh.set_t, row_min = sh.set_min;
  const bool greedy = !(t > 0.f);
  const double td = greedy ? 1.0 : static_cast<double>(t);
  RowWeights<T> rw;
  rw.scale = kLog2e64 / td;
  rw.table = sh.exp2_table;
  rw.max_key = max_key;
  rw.keep_key = 0u;  // min_p off
  rw.max = Key16<T>::value(key_bits(max_key));
  // what lies below the window is at most its lower edge
  const float edge = -Key16<T>::value(Key16<T>::kBase + S);
  const bool low_matters =
      !(static_cast<double>(rw.max) - static_cast<double>(edge) > kCntNegligible * fmax(td, 1.0));
  const bool slow = max_key != 0u && (escape != 0u || (any_low != 0u && low_matters));
  const bool empty = rw.max_key == 0u;
  if (row_min > 0.f && !empty) rw.keep_key = rw.smallest_kept(row_min, static_cast<float>(td), lane);

  // Keys of the four bins from b0 on, a multiple of 4, whose lowest is key0, and their weights at T and as exp(x - max).
  // The sums over the groups and the searches inside one take a value's weight from here: a group that has mass for the
  // one has it for the other.
  auto quad_keys = [&](uint32_t b0, uint32_t key0, uint32_t (&key)[4]) -> bool {
    // four neighbours, but in the group of zero, which has one value; the slow path's keys lie anywhere: no table
    const uint32_t step = slow || b0 >= 64u ? 1u : 0u;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) key[j] = key0 + j * step;
    return !slow && step != 0u;
  };
  auto quad_weights = [&](const uint32_t (&key)[4], bool even, int plain, double (&w)[4]) {
    const uint32_t binade = even ? ((key_bits(key[3]) & 0x7fffu) - Key16<T>::kBase) >> Key16<T>::kMantissa : 0u;
    rw.mass4(key, even, sh.ratio[plain][binade], plain ? kLog2e64 : rw.scale, w);
  };
  // Tokens and mass of the n groups of 64 bins in the counters, group i into the leader's arrays at order(i): four
  // bins a lane, half a warp a group, the groups spread over the cluster.
  double lse = 0.0;
  auto sum_groups = [&](int n, auto order, auto key_of) {
    // neighbouring pairs of groups, which are either all populated or all empty, to different CTAs
    for (int i2 = warp * csize + rank; i2 * 2 < n; i2 += csize * kCntWarps) {
      const uint32_t b0 = static_cast<uint32_t>(i2) * 128 + lane * 4;
      const uint4 own = *reinterpret_cast<const uint4*>(hist + b0);
      uint32_t c[4] = {own.x, own.y, own.z, own.w};
      if (csize > 1) {
#pragma unroll
        for (int r = 1; r < kCntMaxCluster; ++r)
          if (r < csize) {  // csize is a power of two
            const uint4 v = *reinterpret_cast<const uint4*>(peer(hist, rank ^ r) + b0);
            c[0] += v.x;
            c[1] += v.y;
            c[2] += v.z;
            c[3] += v.w;
          }
      }
      uint32_t num = 0;
      double m = 0.0;
      if (__any_sync(0xffffffffu, (c[0] | c[1] | c[2] | c[3]) != 0u)) {
        // the leader's counters of these bins, which nobody else reads, take the whole cluster's counts
        if (csize > 1) *reinterpret_cast<uint4*>(peer(hist, 0) + b0) = make_uint4(c[0], c[1], c[2], c[3]);
        double w[4];
        uint32_t key[4];
        const bool even = quad_keys(b0, key_of(b0), key);
        auto take = [&](const double (&at_t)[4], const double (&at_1)[4]) {
          double mk[4], ml[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t k = rw.kept(key[j]) ? c[j] : 0u;
            num += k;
            mk[j] = count_f64(k) * at_t[j];  // a weight is finite
            ml[j] = count_f64(c[j]) * at_1[j];
          }
          m = (mk[0] + mk[1]) + (mk[2] + mk[3]);
          lse += (ml[0] + ml[1]) + (ml[2] + ml[3]);
        };
        quad_weights(key, even, 0, w);
        if (t == 1.f) {
          take(w, w);
        } else {  // the two chains of operations overlap
          double w1[4];
          quad_weights(key, even, 1, w1);
          take(w, w1);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
          num += __shfl_xor_sync(0xffffffffu, num, o);
          m += __shfl_xor_sync(0xffffffffu, m, o);
        }
      }
      const int i = i2 * 2 + (lane >> 4);
      if ((lane & 15) == 0 && i < n) {
        CountShared* l = peer(&sh, 0);
        l->cnt[order(i)] = num;
        l->own[order(i)] = m;
      }
    }
  };
  int groups = kBins / 64;
  if (!slow) {
    if (!empty) sum_groups(groups, [](int i) { return window_order<T>(i); }, [](uint32_t b) { return bin_key<T>(b); });
  } else {
    // all 65,536 keys, kBins at a time from the top
    groups = kCntGroups;
    for (int hi = 65536, done = 0; hi > 0; hi -= kBins) {
      const int lo = max(0, hi - static_cast<int>(kBins));
      __syncthreads();
      cluster_sync();  // the window before has been read
      clear();
      __syncthreads();
      load_first(batch, ch0, ch1);
      for_each(batch, ch0, ch1, [&](uint32_t w) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = valid_key(w >> (16 * h));
          if (key >= lo && key < hi) add(key - lo);
        }
      });
      __syncthreads();
      cluster_sync();
      const int n = (hi - lo) / 64;
      sum_groups(n, [&](int i) { return done + n - 1 - i; }, [&](uint32_t b) { return b + lo; });
      done += n;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) lse += __shfl_xor_sync(0xffffffffu, lse, o);
  if (lane == 0) peer(&sh, 0)->lse[rank * kCntWarps + warp] = lse;
  __syncthreads();
  cluster_sync();

  // Position `nth` (from 0) of the row's tokens with `key`, searched in the chunks [a, b) by the whole CTA.
  auto write_token = [&](int a, int b, uint32_t key, uint32_t nth, float lp) {
    const uint32_t want = key_bits(key), mask = key == 0x8000u ? 0x7fffu : 0xffffu;
    auto matches = [&](uint4 v) -> uint32_t {  // bit i: element i of the chunk is one of them
      const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
      uint32_t bits = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bits |= ((vw[j] & mask) == want ? 1u : 0u) << (2 * j);
        bits |= (((vw[j] >> 16) & mask) == want ? 1u : 0u) << (2 * j + 1);
      }
      return bits;
    };
    // The CTA counts strip after strip until one holds the token, each warp a contiguous part; the warp that has it
    // goes through its part again. (256 rows of 151936: half of the row on average, 5 us for 13.)
    constexpr int kBatch = 8;
    const int wper = min(32 * kBatch, (b - a + kCntWarps - 1) / kCntWarps);
    uint32_t base = 0;
    int parity = 0;
#pragma unroll 1
    for (int s0 = a; s0 < b; s0 += wper * kCntWarps, parity ^= 1) {
      const int w0 = min(b, s0 + warp * wper), w1 = min(b, w0 + wper);
      uint32_t n = 0;
      uint4 v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int ch = w0 + lane + 32 * j;
        v[j] = make_uint4(~0u, ~0u, ~0u, ~0u);  // NaN is no candidate's pattern
        if (ch < w1 && ch >= whole0 && ch < whole1) v[j] = __ldg(src + ch);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int ch = w0 + lane + 32 * j;
        if (ch < w1 && (ch < whole0 || ch >= whole1)) v[j] = load8(ch);
      }
      Key16<T>::count_equal(v, want * 0x00010001u, n);
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) sh.warp_u[parity][warp] = n;
      __syncthreads();
      const uint32_t count = lane < kCntWarps ? sh.warp_u[parity][lane] : 0u;
      const uint32_t total = __reduce_add_sync(0xffffffffu, count);
      if (nth >= base + total) {
        base += total;
        continue;
      }
      uint32_t at = base + __reduce_add_sync(0xffffffffu, lane < warp ? count : 0u);
      if (nth < at || nth >= at + n) return;
      for (int c0 = w0; c0 < w1; c0 += 32) {
        const uint32_t bits = c0 + lane < w1 ? matches(load8(c0 + lane)) : 0u;
        const uint32_t mine = __popc(bits);
        const uint32_t incl = warp_scan_u32(mine, lane);
        const uint32_t excl = at + incl - mine;
        if (nth >= excl && nth < excl + mine) {
          uint32_t left = bits;
          for (uint32_t i = excl; i < nth; ++i) left &= left - 1;
          out_tokens[row] = static_cast<long long>(c0 + lane) * 8 - head + __ffs(left) - 1;
          out_logprobs[row] = lp;
        }
        at += __shfl_sync(0xffffffffu, incl, 31);
        if (nth < at) break;
      }
      return;
    }
  };

  if (rank == 0 && !empty) {
    // ---- prefix sums over the groups, kCntPer neighbours a thread ----
    uint32_t c[kCntPer];
    double m[kCntPer];
    uint32_t cs = 0;
    double ms = 0.0;
#pragma unroll
    for (int j = 0; j < kCntPer; ++j) {
      const int g = tid * kCntPer + j;
      cs += g < groups ? sh.cnt[g] : 0u;
      ms += g < groups ? sh.own[g] : 0.0;
      c[j] = cs;
      m[j] = ms;
    }
    const uint32_t ci = warp_scan_u32(cs, lane);
    const double mi = warp_scan_f64(ms, lane);
    if (lane == 31) {
      sh.warp_u[0][warp] = ci;
      sh.warp_d[warp] = mi;
    }
    uint32_t cb = __shfl_up_sync(0xffffffffu, ci, 1);
    double mb = __shfl_up_sync(0xffffffffu, mi, 1);
    if (lane == 0) {
      cb = 0;
      mb = 0.0;
    }
    __syncthreads();
    for (int w = 0; w < warp; ++w) {
      cb += sh.warp_u[0][w];
      mb += sh.warp_d[w];
    }
#pragma unroll
    for (int j = 0; j < kCntPer; ++j) {
      const int g = tid * kCntPer + j;
      c[j] += cb;
      m[j] += mb;
      if (g < groups) {
        sh.cnt[g] = c[j];
        sh.mass[g] = m[j];
      }
    }
    __syncthreads();
    const uint32_t n_all = sh.cnt[groups - 1];
    if (warp == kCntWarps - 1) {
      double sum = 0.0;
      for (int i = lane; i < csize * kCntWarps; i += 32) sum += sh.lse[i];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) sh.log_sum = log(sum);
    }

    // Counts of group g's values, two a lane of warp 0 in descending order, and their weights (kept ones only).
    auto load_group = [&](int g, uint32_t (&key)[2], uint32_t (&n)[2], double (&w)[2]) {
      // the lower of the lane's two bins (slow: keys)
      const uint32_t b = static_cast<uint32_t>(slow ? groups - 1 - g : window_group<T>(g)) * 64 + 62 - 2 * lane;
      n[0] = n[1] = 0;
      if (!slow) {
        const uint2 v = *reinterpret_cast<const uint2*>(hist + b);
        n[0] = v.y;
        n[1] = v.x;
      } else {
        n[0] = sh.group_cnt[63 - 2 * lane];
        n[1] = sh.group_cnt[62 - 2 * lane];
      }
      const uint32_t b0 = b & ~3u;
      uint32_t k4[4];
      double w4[4];
      const bool even = quad_keys(b0, slow ? b0 : bin_key<T>(b0), k4);
      quad_weights(k4, even, 0, w4);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        key[i] = b & 2u ? k4[3 - i] : k4[1 - i];
        w[i] = b & 2u ? w4[3 - i] : w4[1 - i];
        if (!rw.kept(key[i])) n[i] = 0;
        if (n[i] == 0) w[i] = 0.0;
      }
    };
    // the slow path has no counters left for the group: the whole CTA counts its values again
    auto recount = [&](int g) {
      if (!slow) return;
      if (tid < 64) sh.group_cnt[tid] = 0;
      __syncthreads();
      const uint32_t lo = static_cast<uint32_t>(groups - 1 - g) * 64;
      load_first(batch, 0, chunks);
      for_each(batch, 0, chunks, [&](uint32_t w) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t i = static_cast<uint32_t>(valid_key(w >> (16 * h))) - lo;
          if (i < 64u) atomicAdd(&sh.group_cnt[i], 1u);
        }
      });
      __syncthreads();
    };
    // The first position whose cumulative mass reaches (strict: exceeds) `limit`, but none behind the last candidate of
    // the cut before, whose mass was added up in another order -> sh.key, sh.nth, sh.cum.
    auto find_mass = [&](int* found, double limit, bool strict) {
      int mine = kCntGroups, last = -1;
#pragma unroll
      for (int j = kCntPer - 1; j >= 0; --j) {
        const int g = tid * kCntPer + j;
        if (g < groups && sh.own[g] > 0.0) {
          last = max(last, g);
          if (strict ? m[j] > limit : m[j] >= limit) mine = g;
        }
      }
      if (mine < kCntGroups) atomicMin(found, mine);
      __syncthreads();
      if (*found == kCntGroups) {  // rounding at the very end: the last group that has mass
        __syncthreads();
        if (tid == 0) *found = -1;
        __syncthreads();
        if (last >= 0) atomicMax(found, last);
        __syncthreads();
      }
      const int g = min(max(*found, 0), groups - 1);
      recount(g);
      if (warp == 0) {
        uint32_t key[2], n[2];
        double w[2];
        load_group(g, key, n, w);
        const double m0 = n[0] * w[0], m1 = n[1] * w[1];
        const double incl = warp_scan_f64(m0 + m1, lane);
        double at = __shfl_up_sync(0xffffffffu, incl, 1);
        at = (g ? sh.mass[g - 1] : 0.0) + (lane ? at : 0.0);
        const bool first = m0 > 0.0 && (strict ? at + m0 > limit : at + m0 >= limit);
        const bool second = m1 > 0.0 && (strict ? at + m0 + m1 > limit : at + m0 + m1 >= limit);
        const uint32_t hit = __ballot_sync(0xffffffffu, first || second);
        const uint32_t any = __ballot_sync(0xffffffffu, m0 > 0.0 || m1 > 0.0);
        // no hit: rounding inside the group, its last value that has mass (there is one: the group's sum is not 0)
        if (lane == (hit ? __ffs(hit) - 1 : 31 - __clz(any | 1u))) {
          const bool use0 = hit ? first : !(m1 > 0.0);
          const uint32_t cc = use0 ? n[0] : n[1];
          const double ww = use0 ? w[0] : w[1], a = use0 ? at : at + m0;
          const double q = (limit - a) / ww;
          double j = strict ? floor(q) : ceil(q) - 1.0;  // position among the equal tokens
          j = fmax(hit ? fmin(j, cc - 1.0) : cc - 1.0, 0.0);
          const uint32_t kk = use0 ? key[0] : key[1], jj = static_cast<uint32_t>(j);
          if (kk > sh.key || (kk == sh.key && jj < sh.nth)) {
            sh.key = kk;
            sh.nth = jj;
          }
          sh.cum = a + (j + 1.0) * ww;
        }
      }
      __syncthreads();
    };

    double kept = sh.mass[groups - 1];
    const int k = greedy || row_min > 1.f ? 1 : sh.set_k;  // the first candidate stays whatever min_p asks
    if (k > 0 && static_cast<uint32_t>(k) < n_all) {
      const uint32_t uk = static_cast<uint32_t>(k);
#pragma unroll
      for (int j = 0; j < kCntPer; ++j) {
        const int g = tid * kCntPer + j;
        if (g < groups && c[j] >= uk && (g == 0 || (j ? c[j - 1] : cb) < uk)) sh.found[0] = g;
      }
      __syncthreads();
      const int g = min(sh.found[0], groups - 1);
      recount(g);
      if (warp == 0) {
        uint32_t key[2], n[2];
        double w[2];
        load_group(g, key, n, w);
        const uint32_t mine = n[0] + n[1];
        const uint32_t before = (g ? sh.cnt[g - 1] : 0u) + warp_scan_u32(mine, lane) - mine;
        // of this lane's tokens the first `take` are among the k
        const uint32_t take = before >= uk ? 0u : min(mine, uk - before);
        const uint32_t take0 = min(take, n[0]);
        double s = take0 * w[0] + (take - take0) * w[1];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) sh.cum = (g ? sh.mass[g - 1] : 0.0) + s;
        if (take > 0u && before + mine >= uk) {  // the k-th
          sh.key = take > take0 ? key[1] : key[0];
          sh.nth = (take > take0 ? take - take0 : take0) - 1u;
        }
      }
      __syncthreads();
      kept = sh.cum;
      __syncthreads();
    }
    const double p = sh.set_p;
    const double uu = fmin(fmax(static_cast<double>(sh.set_u), 0.0), 1.0 - 0x1p-53);  // NaN: 0
    // the cut by top-p, then the draw (a loop: one copy of the search's code)
#pragma unroll 1
    for (int stage = p < 1.0 && !greedy ? 1 : 2; stage <= 2; ++stage) {
      find_mass(&sh.found[stage], stage == 1 ? fmax(p, 0.0) * kept : (greedy ? 0.0 : uu * kept), stage == 2);
      if (stage == 1) {
        kept = fmin(sh.cum, kept);
        __syncthreads();
      }
    }
    const uint32_t key = sh.key, nth = sh.nth;
    const float lp = static_cast<float>((key == rw.max_key ? 0.0 : rw.gap(key)) - sh.log_sum);
    if (slow) {
      if (tid == 0) {  // the leader goes through the whole row
        sh.nth_here = static_cast<int>(nth);
        sh.logprob = lp;
      }
    } else if (warp == 0) {
      // the CTA whose slice holds the nth of them: lane r asks CTA r
      const uint32_t b = min(key_bin<T>(key), kBins - 1u);
      uint32_t n = lane < csize ? peer(hist, lane)[b] : 0u;
      // the leader's holds everybody's
      const uint32_t others = __reduce_add_sync(0xffffffffu, lane ? n : 0u);
      if (lane == 0 && csize > 1) n -= others;
      const uint32_t before = warp_scan_u32(n, lane) - n;
      if (nth >= before && nth < before + n) {
        CountShared* o = peer(&sh, lane);
        o->key = key;
        o->nth_here = static_cast<int>(nth - before);
        o->logprob = lp;
      }
    }
  }
  if (empty && rank == 0 && tid == 0) {  // nothing to choose from
    out_tokens[row] = 0;
    out_logprobs[row] = -INFINITY;
  }
  __syncthreads();
  cluster_sync();  // the draw is known, and nobody reads another's memory any more
  if (sh.nth_here >= 0)
    write_token(slow ? 0 : ch0, slow ? chunks : ch1, sh.key, static_cast<uint32_t>(sh.nth_here), sh.logprob);
}

namespace {
template <typename T, int THREADS>
int launch_sample_counts(const void* logits, long long ld, int rows, int V, const float* u, const float* temperature,
                         const int* top_k, const float* top_p, const float* min_p, long long* tokens, float* logprobs,
                         int csize, cudaStream_t s) {
  constexpr int smem = static_cast<int>((2 * Key16<T>::kSlots + 128) * 4);
  auto kern = sample_counts_kernel<T, THREADS>;
  cudaError_t e = smem_attr_once<sample_counts_kernel<T, THREADS>>(smem);
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = csize;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * csize, 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, reinterpret_cast<const T*>(logits), ld, V, u, temperature,
                                             top_k, top_p, min_p, tokens, logprobs, csize));
}

template <typename T>
int sample_counts(const void* logits, long long ld, int rows, int V, const float* u, const float* temperature,
                  const int* top_k, const float* top_p, const float* min_p, long long* tokens, float* logprobs,
                  cudaStream_t s) {
  // Few rows: spread each over more SMs while its slices stay long enough to count and the GPU has room for them all at
  // once: pairs as far as blocks fit, larger clusters on nine tenths of the SMs (they do not fill a GPC), one block
  // each. Measured by cluster size 1, 2, 4, 8 in us: bf16, V = 151936: 1 row 28, 21, 17, 15; 30 rows 36, 26, 21, 22;
  // 60 rows 35, 26, 26, 40; 130 rows 38, 35, 47, 79; 200 rows 56, 53, 68, 116; 256 rows 57, 64, 85, 146. V = 32000:
  // 30 rows 19, 15, 14, 19; 74 rows 19, 16, 27, 46; 150 rows 24, 31, 43, 80. fp16, V = 151936: 18 rows 43, 32, 26, 44;
  // 74 rows 45, 34, 69, 110. Blocks of 1024 threads, one an SM, are what fp16's counters leave room for.
  constexpr int threads = Key16<T>::kOneRow ? 1024 : 512;
  const long long sms = device_sm_count();
  int csize = 1;
  for (int c = 2; c <= kCntMaxCluster && V / (c / 2) > 4096; c *= 2)
    if (static_cast<long long>(rows) * c <= (c == 2 ? sms * (1024 / threads) : sms * 9 / 10)) csize = c;
  if (static_cast<long long>(rows) * csize > 0x7fffffffll) return -3;
  return launch_sample_counts<T, threads>(logits, ld, rows, V, u, temperature, top_k, top_p, min_p, tokens, logprobs, csize, s);
}
}  // namespace
}  // namespace accerl

// One token per row of logits [rows, V] (half: 0 bf16, 1 fp16; row stride ld) from u [rows]. top_k, top_p and
// min_p may be null (off).
extern "C" int accerl_sample_counts(const void* logits, long long ld, int half, int rows, int V, const float* u,
                                    const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                                    long long* tokens, float* logprobs, cudaStream_t s) {
  using namespace accerl;
  if (rows <= 0) return 0;
  if (V <= 0 || V > 0x7ffffff0) return -1;
  if (half) return sample_counts<__half>(logits, ld, rows, V, u, temperature, top_k, top_p, min_p, tokens, logprobs, s);
  return sample_counts<__nv_bfloat16>(logits, ld, rows, V, u, temperature, top_k, top_p, min_p, tokens, logprobs, s);
}
