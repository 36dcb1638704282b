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
// exponential per value that occurs, and only integer atomics, so a result does not depend on their order.
//
// Counters for all values would fill 128 KB and leave one block to an SM, whose counting then waits for its own
// searches and barriers. So the kernel counts a window of the values that logits take (bf16: zero and 2^-40 to
// 2^24; fp16: below 64, each sign) in 32 KB (84 KB). Lower values, masks of the type's lowest value among them, are
// left out where they weigh nothing; a row with any other value takes the slow path, which counts all values,
// window by window.
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"

namespace accerl {

constexpr int kCntGroups = 1024;              // at most: groups of 64 neighbouring values
constexpr int kCntMaxSlice = 65528;           // elements a CTA may count without overflowing 16 bits
constexpr int kCntMaxCluster = 8;
// tokens further below the largest logit than this many temperatures weigh nothing: all of a row's together
// hold less than 1e-20 of its mass, far below what a 64-bit sum resolves
constexpr double kCntNegligible = 60.0;

// Order-preserving 16-bit keys of the finite values and +inf: (kNegInf, kPosInf]. The window holds kP
// magnitudes of each sign from the pattern kLo on; the slot of kLo itself is that of zero.
template <typename T>
struct Key16;
template <>
struct Key16<__nv_bfloat16> {
  static constexpr uint32_t kInf = 0x7f80u, kPosInf = 0xff80u, kNegInf = 0x007fu;
  static constexpr uint32_t kLo = ((127u - 40u) << 7) - 1u, kP = 64u << 7;
  static constexpr int kBlocksPerSm = 4;
  static ACCERL_DEVINL float value(uint32_t bits) { return __uint_as_float(bits << 16); }
};
template <>
struct Key16<__half> {
  static constexpr uint32_t kInf = 0x7c00u, kPosInf = 0xfc00u, kNegInf = 0x03ffu;
  static constexpr uint32_t kLo = 0u, kP = 21u << 10;
  static constexpr int kBlocksPerSm = 2;
  static ACCERL_DEVINL float value(uint32_t bits) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  }
};
ACCERL_DEVINL uint32_t key_bits(uint32_t key) { return (key & 0x8000u) ? key ^ 0x8000u : key ^ 0xffffu; }
ACCERL_DEVINL uint32_t bits_key(uint32_t bits) { return (bits & 0x8000u) ? bits ^ 0xffffu : bits ^ 0x8000u; }
// window bin (ascending with the value) <-> key
template <typename T>
ACCERL_DEVINL uint32_t bin_key(uint32_t b) {
  constexpr uint32_t P = Key16<T>::kP, lo = Key16<T>::kLo;
  if (b == P) return 0x8000u;
  return b > P ? 0x8000u + lo + (b - P) : 0x7fffu - lo - (P - 1 - b);
}
template <typename T>
ACCERL_DEVINL uint32_t key_bin(uint32_t key) {
  constexpr uint32_t P = Key16<T>::kP, lo = Key16<T>::kLo;
  if (key == 0x8000u) return P;
  return key > 0x8000u ? key - 0x8000u - lo + P : key + lo + P - 0x8000u;
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
  uint32_t max_in, max_low, max_all, escape;  // of this CTA's slice
  uint32_t group_cnt[64];                     // slow path: tokens of a group's values
  int found;                                  // a search's group
  uint32_t key, nth;                          // its value and rank among the value's tokens
  double cum;                                 // mass up to and with that token
  int nth_here;                               // rank of the drawn token within this CTA's slice, or -1
  float logprob;
};

// 2^(y / 64) for y <= 0: n = round(y), the table for n mod 64, and the Taylor series of the rest, |r| <= ln 2 / 128,
// whose sixth term is below 2^-54. The argument's rounding costs at most a relative |y| 2^-59, so a weight is
// within 2^-52 of the largest one's unit. Below 2^-1020: 0.
ACCERL_DEVINL double exp2_64th(double y, const double* table) {
  const double t = y + 0x1.8p52;
  const int n = __double2loint(t);
  const double r = (y - (t - 0x1.8p52)) * (0.693147180559945309417 / 64);
  double q = __fma_rn(r, 1.0 / 120, 1.0 / 24);
  q = __fma_rn(q, r, 1.0 / 6);
  q = __fma_rn(q, r, 0.5);
  q = __fma_rn(q, r, 1.0);
  q = __fma_rn(q, r, 1.0) * table[n & 63];
  const double v = __hiloint2double(__double2hiint(q) + (n >> 6) * 0x100000, __double2loint(q));
  return y < -64.0 * 1020 ? 0.0 : v;
}
constexpr double kLog2e64 = 64 * 1.44269504088896340736;

// The row's settings and how a value turns into a weight.
template <typename T>
struct RowWeights {
  double scale;  // 64 log2(e) / T
  double min_p;
  float max;     // the row's largest logit
  uint32_t max_key;
  const double* table;
  ACCERL_DEVINL double gap(uint32_t key) const {
    return static_cast<double>(Key16<T>::value(key_bits(key))) - static_cast<double>(max);
  }
  ACCERL_DEVINL double mass(uint32_t key, double sc) const {
    // an infinite maximum leaves nothing to the others (whose gap is -inf); at an infinite temperature (sc = 0)
    // every finite gap weighs 1
    const double w = exp2_64th(fmax(gap(key) * sc, -64.0 * 1021), table);
    return key == max_key ? 1.0 : (isinf(max) ? 0.0 : w);
  }
  ACCERL_DEVINL double weight(uint32_t key) const { return mass(key, scale); }
  ACCERL_DEVINL double plain(uint32_t key) const { return mass(key, kLog2e64); }  // exp(x - max)
  ACCERL_DEVINL bool kept(uint32_t key, double w) const { return key == max_key || !(min_p > 0.0) || w >= min_p; }
};

// One row per cluster of CTAs, each counting a slice of it.
template <typename T, int kCntThreads>
__global__ void __launch_bounds__(kCntThreads, kCntThreads == 1024 ? 1 : Key16<T>::kBlocksPerSm)
    sample_counts_kernel(const T* __restrict__ logits, long long ld, int V, const float* __restrict__ u,
                         const float* __restrict__ temperature, const int* __restrict__ top_k,
                         const float* __restrict__ top_p, const float* __restrict__ min_p,
                         long long* __restrict__ out_tokens, float* __restrict__ out_logprobs, int csize) {
  constexpr uint32_t P = Key16<T>::kP, kBins = 2 * P;
  constexpr int kCntWarps = kCntThreads / 32, kCntPer = kCntGroups / kCntThreads;
  extern __shared__ uint4 dyn[];
  uint32_t* hist = reinterpret_cast<uint32_t*>(dyn);  // kBins 16-bit counters, two to a word
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
  // f(bits) for every element of the chunks [a, b)
  auto for_each = [&](int a, int b, auto f) {
    constexpr int kAhead = 4;
    for (int c = a + tid; c < b; c += kCntThreads * kAhead) {
      uint4 v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        v[j] = c + j * kCntThreads < b ? load8(c + j * kCntThreads) : make_uint4(~0u, ~0u, ~0u, ~0u);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const uint32_t vw[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f(vw[i] & 0xffffu);
          f(vw[i] >> 16);
        }
      }
    }
  };
  auto clear = [&]() {
    for (int i = tid; i < static_cast<int>(kBins / 8); i += kCntThreads) dyn[i] = make_uint4(0, 0, 0, 0);
  };
  auto add = [&](uint32_t bin) { atomicAdd(&hist[bin >> 1], 1u << ((bin & 1u) * 16)); };

  clear();
  if (tid == 0) sh.nth_here = -1;
  if (tid < 64) sh.exp2_table[tid] = exp2(tid / 64.0);
  __syncthreads();

  // ---- count the slice ----
  uint32_t max_in = 0, max_low = 0, max_all = 0, escape = 0;
  for_each(ch0, ch1, [&](uint32_t bits) {
    const uint32_t mag = bits & 0x7fffu, slot = mag - Key16<T>::kLo;
    const uint32_t neg = (bits & 0x8000u) ? ~0u : 0u;
    if (slot - 1u < P - 1u) {
      const uint32_t bin = P + (slot ^ neg);
      max_in = max(max_in, bin + 1u);
      add(bin);
    } else if (mag == 0u) {
      max_in = max(max_in, P + 1u);
      add(P);
    } else if (mag < Key16<T>::kInf || bits == Key16<T>::kInf) {  // outside the window; -inf and NaN are nothing
      const uint32_t key = bits_key(bits);
      max_all = max(max_all, key);
      if (neg && mag >= Key16<T>::kLo + P) max_low = max(max_low, key);
      else escape = 1u;
    }
  });
  max_in = __reduce_max_sync(0xffffffffu, max_in);
  max_low = __reduce_max_sync(0xffffffffu, max_low);
  max_all = __reduce_max_sync(0xffffffffu, max_all);
  escape = __reduce_max_sync(0xffffffffu, escape);
  if (lane == 0) {
    sh.warp_u[0][warp] = max_in;
    sh.warp_u[1][warp] = max_low;
    sh.warp_u[2][warp] = (max_all << 1) | escape;
  }
  __syncthreads();
  if (warp == 0) {
    const bool has = lane < kCntWarps;
    const uint32_t all = has ? sh.warp_u[2][lane] : 0u;
    max_in = __reduce_max_sync(0xffffffffu, has ? sh.warp_u[0][lane] : 0u);
    max_low = __reduce_max_sync(0xffffffffu, has ? sh.warp_u[1][lane] : 0u);
    max_all = __reduce_max_sync(0xffffffffu, all >> 1);
    escape = __reduce_max_sync(0xffffffffu, all & 1u);
    if (lane == 0) {
      sh.max_in = max_in;
      sh.max_low = max_low;
      sh.max_all = max_all;
      sh.escape = escape;
    }
  }
  __syncthreads();
  cluster_sync();

  // ---- the row's largest value, and whether the window holds all that matters ----
  max_in = max_low = max_all = escape = 0;
#pragma unroll
  for (int c = 0; c < kCntMaxCluster; ++c)
    if (c < csize) {
      const CountShared* o = peer(&sh, c);
      max_in = max(max_in, o->max_in);
      max_low = max(max_low, o->max_low);
      max_all = max(max_all, o->max_all);
      escape |= o->escape;
    }
  RowWeights<T> rw;
  const float t = temperature[row];
  const bool greedy = !(t > 0.f);
  const double td = greedy ? 1.0 : static_cast<double>(t);
  rw.scale = kLog2e64 / td;
  rw.table = sh.exp2_table;
  rw.min_p = min_p ? static_cast<double>(min_p[row]) : 0.0;
  rw.max_key = max_in ? bin_key<T>(max_in - 1u) : 0u;
  rw.max = Key16<T>::value(key_bits(rw.max_key));
  const bool low_matters = max_low != 0u && !(max_in != 0u && -rw.gap(max_low) > kCntNegligible * fmax(td, 1.0));
  const bool slow = escape != 0u || low_matters;
  if (slow) {
    rw.max_key = max(rw.max_key, max_all);
    rw.max = Key16<T>::value(key_bits(rw.max_key));
  }
  const bool empty = rw.max_key == 0u;

  // Tokens and mass of the groups whose 64 bins each start at bin `base` + 64 i, i < n, into the leader's arrays
  // at n_before + (n - 1 - i): four bins a lane, half a warp a group, the groups spread over the cluster.
  double lse = 0.0;
  auto sum_groups = [&](int n, int n_before, auto key_of) {
    for (int i2 = rank * kCntWarps + warp; i2 * 2 < n; i2 += csize * kCntWarps) {
      const uint32_t b0 = static_cast<uint32_t>(i2) * 128 + lane * 4;
      uint32_t c[4] = {0, 0, 0, 0};
#pragma unroll
      for (int r = 0; r < kCntMaxCluster; ++r)
        if (r < csize) {
          const uint2 v = *reinterpret_cast<const uint2*>(peer(hist, r) + b0 / 2);
          c[0] += v.x & 0xffffu;
          c[1] += v.x >> 16;
          c[2] += v.y & 0xffffu;
          c[3] += v.y >> 16;
        }
      uint32_t num = 0;
      double m = 0.0;
      if (__any_sync(0xffffffffu, (c[0] | c[1] | c[2] | c[3]) != 0u)) {
        uint32_t key[4];
        double w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // all four without branches: their chains of operations overlap
          key[j] = key_of(b0 + j);
          w[j] = rw.weight(key[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t n = rw.kept(key[j], w[j]) ? c[j] : 0u;
          num += n;
          m += n ? n * w[j] : 0.0;
        }
        if (t != 1.f) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = rw.plain(key[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) lse += c[j] ? c[j] * w[j] : 0.0;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
          num += __shfl_xor_sync(0xffffffffu, num, o);
          m += __shfl_xor_sync(0xffffffffu, m, o);
        }
      }
      const int i = i2 * 2 + (lane >> 4);
      if ((lane & 15) == 0 && i < n) {
        CountShared* l = peer(&sh, 0);
        l->cnt[n_before + n - 1 - i] = num;
        l->own[n_before + n - 1 - i] = m;
      }
    }
  };
  int groups = kBins / 64;
  if (!slow) {
    if (!empty) sum_groups(groups, 0, [](uint32_t b) { return bin_key<T>(b); });
  } else {
    // all 65,536 keys, kBins at a time from the top
    groups = kCntGroups;
    for (int hi = 65536, done = 0; hi > 0; hi -= kBins) {
      const int lo = max(0, hi - static_cast<int>(kBins));
      __syncthreads();
      cluster_sync();  // the window before has been read
      clear();
      __syncthreads();
      for_each(ch0, ch1, [&](uint32_t bits) {
        if (bits == 0x8000u) bits = 0u;
        const uint32_t key = bits_key(bits);
        if (key > Key16<T>::kNegInf && key <= Key16<T>::kPosInf && static_cast<int>(key) >= lo && static_cast<int>(key) < hi)
          add(key - lo);
      });
      __syncthreads();
      cluster_sync();
      const int n = (hi - lo) / 64;
      sum_groups(n, done, [&](uint32_t b) { return b + lo; });
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
    // each warp counts a contiguous part; the one that holds the token goes through its part again
    const int wper = (b - a + kCntWarps - 1) / kCntWarps;
    const int w0 = min(b, a + warp * wper), w1 = min(b, w0 + wper);
    uint32_t n = 0;
#pragma unroll 4
    for (int c = w0 + lane; c < w1; c += 32) n += __popc(matches(load8(c)));
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) sh.warp_u[0][warp] = n;
    __syncthreads();
    uint32_t at = 0;
    for (int w = 0; w < warp; ++w) at += sh.warp_u[0][w];
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
  };

  if (rank == 0 && !empty) {
    // ---- prefix sums over the groups, four a thread ----
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

    // Counts of group g's values, two a lane of warp 0 in descending order, and their weights (kept ones only).
    auto load_group = [&](int g, uint32_t (&key)[2], uint32_t (&n)[2], double (&w)[2]) {
      const uint32_t b = static_cast<uint32_t>(groups - 1 - g) * 64 + 62 - 2 * lane;  // the lower of the two bins
      n[0] = n[1] = 0;
      if (!slow) {
#pragma unroll
        for (int r = 0; r < kCntMaxCluster; ++r)
          if (r < csize) {
            const uint32_t v = peer(hist, r)[b / 2];
            n[0] += v >> 16;
            n[1] += v & 0xffffu;
          }
      } else {
        n[0] = sh.group_cnt[63 - 2 * lane];
        n[1] = sh.group_cnt[62 - 2 * lane];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        key[i] = slow ? b + 1 - i : bin_key<T>(b + 1 - i);
        w[i] = rw.weight(key[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!rw.kept(key[i], w[i])) n[i] = 0;
        if (n[i] == 0) w[i] = 0.0;
      }
    };
    // the slow path has no counters left for the group: the whole CTA counts its values again
    auto recount = [&](int g) {
      if (!slow) return;
      if (tid < 64) sh.group_cnt[tid] = 0;
      __syncthreads();
      const uint32_t lo = static_cast<uint32_t>(groups - 1 - g) * 64;
      for_each(0, chunks, [&](uint32_t bits) {
        if (bits == 0x8000u) bits = 0u;
        const uint32_t key = bits_key(bits);
        if (key > Key16<T>::kNegInf && key <= Key16<T>::kPosInf && key - lo < 64u) atomicAdd(&sh.group_cnt[key - lo], 1u);
      });
      __syncthreads();
    };
    // The first position whose cumulative mass reaches (strict: exceeds) `limit` -> sh.key, sh.nth, sh.cum.
    auto find_mass = [&](double limit, bool strict) {
      if (tid == 0) sh.found = kCntGroups;
      __syncthreads();
      int mine = kCntGroups, last = -1;
#pragma unroll
      for (int j = kCntPer - 1; j >= 0; --j) {
        const int g = tid * kCntPer + j;
        if (g < groups && sh.own[g] > 0.0) {
          last = max(last, g);
          if (strict ? m[j] > limit : m[j] >= limit) mine = g;
        }
      }
      if (mine < kCntGroups) atomicMin(&sh.found, mine);
      __syncthreads();
      if (sh.found == kCntGroups) {  // rounding at the very end: the last group that has mass
        __syncthreads();
        if (tid == 0) sh.found = -1;
        __syncthreads();
        if (last >= 0) atomicMax(&sh.found, last);
        __syncthreads();
      }
      const int g = sh.found;
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
        // no hit: rounding inside the group, its last value that has mass
        if (lane == (hit ? __ffs(hit) - 1 : 31 - __clz(any))) {
          const bool use0 = hit ? first : !(m1 > 0.0);
          const uint32_t cc = use0 ? n[0] : n[1];
          const double ww = use0 ? w[0] : w[1], a = use0 ? at : at + m0;
          const double q = (limit - a) / ww;
          double j = strict ? floor(q) : ceil(q) - 1.0;  // position among the equal tokens
          j = hit ? fmin(fmax(j, 0.0), cc - 1.0) : cc - 1.0;
          sh.key = use0 ? key[0] : key[1];
          sh.nth = static_cast<uint32_t>(j);
          sh.cum = a + (j + 1.0) * ww;
        }
      }
      __syncthreads();
    };

    double kept = sh.mass[groups - 1];
    int k = top_k ? top_k[row] : 0;
    if (greedy || rw.min_p > 1.0) k = 1;  // the first candidate stays whatever min_p asks
    if (k > 0 && static_cast<uint32_t>(k) < n_all) {
      const uint32_t uk = static_cast<uint32_t>(k);
#pragma unroll
      for (int j = 0; j < kCntPer; ++j) {
        const int g = tid * kCntPer + j;
        if (g < groups && c[j] >= uk && (g == 0 || (j ? c[j - 1] : cb) < uk)) sh.found = g;
      }
      __syncthreads();
      const int g = sh.found;
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
      }
      __syncthreads();
      kept = sh.cum;
      __syncthreads();
    }
    const double p = top_p ? static_cast<double>(top_p[row]) : 1.0;
    if (p < 1.0 && !greedy) {
      find_mass(fmax(p, 0.0) * kept, false);
      kept = fmin(sh.cum, kept);
      __syncthreads();
    }
    const double uu = fmin(fmax(static_cast<double>(u[row]), 0.0), 1.0 - 0x1p-53);  // NaN: 0
    find_mass(greedy ? 0.0 : uu * kept, true);
    const uint32_t key = sh.key, nth = sh.nth;
    float lp = 0.f;
    if (warp == 0 || slow) {
      double s = 0.0;
      for (int i = lane; i < csize * kCntWarps; i += 32) s += sh.lse[i];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      lp = static_cast<float>((key == rw.max_key ? 0.0 : rw.gap(key)) - log(s));
    }
    if (slow) {
      write_token(0, chunks, key, nth, lp);
    } else if (warp == 0) {
      // the CTA whose slice holds the nth of them: lane r asks CTA r
      const uint32_t b = key_bin<T>(key);
      uint32_t n = 0;
      if (lane < csize) {
        const uint32_t v = peer(hist, lane)[b / 2];
        n = (b & 1u) ? v >> 16 : v & 0xffffu;
      }
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
  if (sh.nth_here >= 0) write_token(ch0, ch1, sh.key, static_cast<uint32_t>(sh.nth_here), sh.logprob);
}

namespace {
template <typename T, int THREADS>
int launch_sample_counts(const void* logits, long long ld, int rows, int V, const float* u, const float* temperature,
                         const int* top_k, const float* top_p, const float* min_p, long long* tokens, float* logprobs,
                         int csize, cudaStream_t s) {
  constexpr int smem = static_cast<int>(2 * Key16<T>::kP * 2);
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
  // a slice holds its chunks of 8 and may start 7 elements before the row
  auto slice = [&](int c) { return ((V + 14) / 8 + c - 1) / c * 8; };
  int csize = 1;
  while (csize < kCntMaxCluster && slice(csize) > kCntMaxSlice) csize *= 2;
  if (slice(csize) > kCntMaxSlice) return -2;
  if (static_cast<long long>(rows) * csize > 0x7fffffffll) return -3;
  const long long sms = device_sm_count();
  // few rows: spread each over more SMs, in blocks of 1024 threads, while its slices stay long enough to count
  const bool wide = rows * static_cast<long long>(csize) <= sms;
  const long long room = wide ? sms : sms * Key16<T>::kBlocksPerSm;
  while (csize < kCntMaxCluster && static_cast<long long>(rows) * csize * 2 <= room && slice(csize) > 4096) csize *= 2;
  if (wide)
    return launch_sample_counts<T, 1024>(logits, ld, rows, V, u, temperature, top_k, top_p, min_p, tokens, logprobs, csize, s);
  return launch_sample_counts<T, 256>(logits, ld, rows, V, u, temperature, top_k, top_p, min_p, tokens, logprobs, csize, s);
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
  if (half) return sample_counts<__half>(logits, ld, rows, V, u, temperature, top_k, top_p, min_p, tokens, logprobs, s);
  return sample_counts<__nv_bfloat16>(logits, ld, rows, V, u, temperature, top_k, top_p, min_p, tokens, logprobs, s);
}
