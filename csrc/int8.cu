// Linear layers in 8-bit integers for the rollout engine (sm_100a): rows of activations or weights to
// int8 with one scale each, and their product on the tensor cores.
//
//   rows to 8 bits: a = max_k |x|, s = a / 127, q = round_half_even(127 x / a)
//   product:        y[t, n] = sx[t] * sw[n] * sum_k qx[t, k] qw[n, k] (+ bias[n]) (+ residual[t, n])
//
// The sum runs in 32-bit integers and is exact (K <= 133144 = 2^31 / 127^2); scaling, bias and residual
// are fp32 and the result is rounded once.
#include <cuda_fp16.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "common.cuh"

namespace accerl {

// ------------------------------------------------------------------------------------------------
// rows to 8 bits
// ------------------------------------------------------------------------------------------------
// Arrival at a named barrier without waiting.
ACCERL_DEVINL void named_bar_arrive(uint32_t id, uint32_t nthreads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}

// Programmatic dependent launch: a product launched behind its quantising kernel starts while that one still
// runs, sets itself up and waits here for the whole grid before it and its memory.
ACCERL_DEVINL void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
ACCERL_DEVINL void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

enum QuantPre : int { kPreNone = 0, kPreRmsNorm = 1, kPreSwiglu = 2 };

template <typename T>
struct Half16;  // 16-bit float formats: unpacking of pairs and the bit pattern of infinity
template <>
struct Half16<__nv_bfloat16> {
  static constexpr uint32_t kInf = 0x7f80u;
  // one operation an element; the conversion intrinsic's code takes two for the upper half
  static ACCERL_DEVINL float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static ACCERL_DEVINL float one(uint32_t bits) { return __uint_as_float(bits << 16); }
};
template <>
struct Half16<__half> {
  static constexpr uint32_t kInf = 0x7c00u;
  static ACCERL_DEVINL float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  static ACCERL_DEVINL float one(uint32_t bits) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits))); }
};

// A row's largest magnitude is kept as its 16-bit pattern `amax`, whose order is that of the magnitudes, with
// infinities and NaN on top: a row that holds one gets scale NaN (its outputs are NaN) and zeros.
template <typename T>
ACCERL_DEVINL float row_scale(uint32_t amax) {
  return amax >= Half16<T>::kInf ? __uint_as_float(0x7fffffffu) : __fdiv_rn(Half16<T>::one(amax), 127.f);
}

// The factors that turn a row's elements into whole numbers.
struct RowQuant {
  float m127, a, inv;
};
template <typename T>
ACCERL_DEVINL RowQuant row_quant(uint32_t amax) {
  const float a = Half16<T>::one(amax);
  // a power of two keeps 1 / a, 127 x and the remainder below inside the normal range
  const float f = a < 0x1p-100f ? 0x1p100f : (a > 0x1p100f ? 0x1p-100f : 1.f);
  return RowQuant{127.f * f, a * f, amax == 0u ? 0.f : __frcp_rn(a * f)};
}

// round_half_even(127 x / a), decided exactly without a division per element. x and a have at most 11
// significant bits, so the quotient is either a whole number and a half or at least a relative 2^-19 away
// from every such border. p is within 2^-22 of it; the remainder 127 x - p a is exact, and the quotient
// corrected by it (Markstein, 1990) is the exact one where that is representable, which every border is. The
// last addition rounds to the nearest whole number, ties to even; the low byte of its pattern is the two's
// complement.
ACCERL_DEVINL uint32_t quant_bits(float x, const RowQuant& s) {
  const float n = __fmul_rn(x, s.m127);
  const float p = __fmul_rn(n, s.inv);
  const float e = __fmaf_rn(-p, s.a, n);
  return __float_as_uint(__fadd_rn(__fmaf_rn(e, s.inv, p), 0x1.8p23f));
}
// The same for bf16, whose 8 significant bits leave more room, with two operations instead of five: x r + 384 lies in
// [257, 511], so the first rounds the quotient to a multiple of 2^-15, within 2^-16 of it. r's rounding moves the
// quotient by at most 127 2^-24 < 2^-16: a tie is put back onto its border. Any other quotient is at least
// 0.5 / (127 255) > 2^-16 + 2^-25 from a border and stays on its side. The second rounds to the nearest whole
// number, ties to even (384 is even); the low byte is the number + 128. (Checked over all significands and
// exponents in exact arithmetic.) For 2^-100 <= a <= 2^100; r is the quotient 127 / a by an approximate reciprocal
// corrected by its exact remainder, which saves every thread of a row the division's code.
ACCERL_DEVINL bool bf16_plain(uint32_t amax) { return amax >= 0x0d80u && amax <= 0x7180u; }
ACCERL_DEVINL float bf16_ratio(uint32_t amax) {
  const float a = __uint_as_float(amax << 16);
  float i;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(i) : "f"(a));
  const float q = __fmul_rn(127.f, i);
  return __fmaf_rn(__fmaf_rn(-q, a, 127.f), i, q);
}
ACCERL_DEVINL uint32_t quant_bits_bf16(float x, float r) { return __float_as_uint(__fadd_rn(__fmaf_rn(x, r, 384.f), 0x1.8p23f)); }
ACCERL_DEVINL uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// silu(g) for |g| < 80 before its rounding to bf16, as swiglu_h gives it but without the division, which kept this
// kernel at the instruction limit: the quotient g / (1 + e^-g) from an approximate reciprocal, corrected by its exact
// remainder (Markstein, 1990). The flushing forms differ from __expf's only where e^-g vanishes against 1.
ACCERL_DEVINL float silu_small(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(g, -1.4426950408889634f)));
  const float d = 1.f + e;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  const float q = __fmul_rn(g, r);
  return __fmaf_rn(__fmaf_rn(-q, d, g), r, q);
}

// Reduction over the 2^lg threads of a row (32..blockDim); `red`, one slot per warp, is used by one reduction of the
// kernel only.
template <typename V, typename F>
ACCERL_DEVINL V row_reduce(V v, int lg, V* red, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (lg > 5) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = 1 << (lg - 5);
    v = red[((threadIdx.x >> lg) << (lg - 5)) + (threadIdx.x & (warps - 1))];
    for (int o = 1; o < warps; o <<= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  }
  return v;
}

ACCERL_DEVINL uint32_t amax_pair(uint32_t m) { return max(m & 0xffffu, m >> 16); }

// The pieces of a row that a thread holds, NC chunks of 8 elements 2^lg threads apart (packed pairs).
// All chunks but the last lie inside the row (kWhole: NC is no rounded-up count).
template <int NC>
struct RowPart {
  static constexpr bool kWhole = NC <= 5;
  static ACCERL_DEVINL bool inside(int j, int c, int end) { return (kWhole && j < NC - 1) || c < end; }
  uint4 v[NC];
  ACCERL_DEVINL uint32_t* words(int j) { return reinterpret_cast<uint32_t*>(&v[j]); }
  // gate -> silu(gate) up
  ACCERL_DEVINL void swiglu(int j, uint4 up) {
    const uint32_t uw[4] = {up.x, up.y, up.z, up.w};
    uint32_t* g = words(j);
    uint32_t m2 = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m2 = __vmaxu2(m2, g[i] & 0x7fff7fffu);
    if (amax_pair(m2) < 0x42a0u) {  // every |gate| < 80
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 fg = Half16<__nv_bfloat16>::unpack(g[i]), fu = Half16<__nv_bfloat16>::unpack(uw[i]);
        const float2 a = Half16<__nv_bfloat16>::unpack(pack_bf16x2(silu_small(fg.x), silu_small(fg.y)));
        g[i] = pack_bf16x2(a.x * fu.x, a.y * fu.y);
      }
    } else {
      for (int i = 0; i < 4; ++i) {
        const float2 fg = Half16<__nv_bfloat16>::unpack(g[i]), fu = Half16<__nv_bfloat16>::unpack(uw[i]);
        g[i] = pack_bf16x2(swiglu_h(fg.x, fu.x), swiglu_h(fg.y, fu.y));
      }
    }
  }
  ACCERL_DEVINL float sum_squares() {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Half16<__nv_bfloat16>::unpack(words(j)[i]);
        ss = __fmaf_rn(f.y, f.y, __fmaf_rn(f.x, f.x, ss));
      }
    return ss;
  }
  // x -> bf16(bf16(x r) w), the roundings of the framework's norm
  ACCERL_DEVINL void normalise(const __nv_bfloat16* __restrict__ w, float r, int in_row, int lg, int K) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = ((j << lg) + in_row) * 8;
      if (!inside(j, c, K)) continue;
      const uint4 wv = *reinterpret_cast<const uint4*>(w + c);
      const uint32_t ww[4] = {wv.x, wv.y, wv.z, wv.w};
      uint32_t* p = words(j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Half16<__nv_bfloat16>::unpack(p[i]), g = Half16<__nv_bfloat16>::unpack(ww[i]);
        const float2 n = Half16<__nv_bfloat16>::unpack(pack_bf16x2(f.x * r, f.y * r));
        p[i] = pack_bf16x2(n.x * g.x, n.y * g.y);
      }
    }
  }
  ACCERL_DEVINL uint32_t amax() {
    uint32_t m2 = 0;
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) m2 = __vmaxu2(m2, words(j)[i] & 0x7fff7fffu);
    return amax_pair(m2);
  }
  // round and store; the columns K..Kp are written as zeros
  template <typename T>
  ACCERL_DEVINL void store(int8_t* qr, uint32_t amax, int in_row, int lg, int Kp) {
    if (std::is_same<T, __nv_bfloat16>::value && bf16_plain(amax)) {
      const float r = bf16_ratio(amax);
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int c = ((j << lg) + in_row) * 8;
        if (!inside(j, c, Kp)) continue;
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = Half16<T>::unpack(words(j)[i]);
          b[2 * i] = quant_bits_bf16(f.x, r);
          b[2 * i + 1] = quant_bits_bf16(f.y, r);
        }
        *reinterpret_cast<uint2*>(qr + c) =
            make_uint2(pack4(b[0], b[1], b[2], b[3]) ^ 0x80808080u, pack4(b[4], b[5], b[6], b[7]) ^ 0x80808080u);
      }
      return;
    }
    const bool finite = amax < Half16<T>::kInf;
    const RowQuant s = row_quant<T>(amax);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = ((j << lg) + in_row) * 8;
      if (!inside(j, c, Kp)) continue;
      uint32_t b[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Half16<T>::unpack(words(j)[i]);
        b[2 * i] = quant_bits(f.x, s);
        b[2 * i + 1] = quant_bits(f.y, s);
      }
      const uint2 o = make_uint2(pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7]));
      *reinterpret_cast<uint2*>(qr + c) = finite ? o : make_uint2(0, 0);
    }
  }
};

// One row per 2^lg threads, held in registers between the maximum and the rounding so that it is read once. PRE
// turns the input row into the row to round: RMSNorm (x [rows, K], weight w) or SwiGLU (x = gate | up, [rows, 2K]),
// with the roundings of the framework's own kernels (both give rows in T). Bound by memory where there are many rows
// (bf16 [8192, 8960]: 43 us, 5.1 TB/s; RMSNorm, which reduces twice, 83 us; [2048, 4096]: 6.5 and 9.2 us, SwiGLU 11),
// by one load, one or two reductions and one store in a row where there are few ([64, 1536]: 2.0, 2.6 and 2.4 us).
template <typename T, int PRE, int NC>
__global__ void __launch_bounds__(512) quantize_rows_kernel(const T* __restrict__ x, long long ldx,
                                                            const T* __restrict__ w, float eps,
                                                            int8_t* __restrict__ q, float* __restrict__ scale,
                                                            long long rows, int K, int Kp, int lg) {
  pdl_launch_dependents();  // the product may set itself up; it waits for this grid's end before it reads
  __shared__ uint32_t red_u[16];
  __shared__ float red_f[16];
  const int in_row = threadIdx.x & ((1 << lg) - 1);
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x >> lg) + (threadIdx.x >> lg);
  const bool live = row < rows;
  const T* xr = x + (live ? row : 0) * ldx;
  // every load of the row is issued up front; chunks behind its end read its first one and are zeroed
  RowPart<NC> part;
  uint4 up[PRE == kPreSwiglu ? NC : 1];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = ((j << lg) + in_row) * 8, at = part.inside(j, c, K) ? c : 0;
    part.v[j] = *reinterpret_cast<const uint4*>(xr + at);
    if constexpr (PRE == kPreSwiglu) up[j] = *reinterpret_cast<const uint4*>(xr + K + at);
  }
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    if (!part.inside(j, ((j << lg) + in_row) * 8, K)) part.v[j] = make_uint4(0, 0, 0, 0);
    else if constexpr (PRE == kPreSwiglu) part.swiglu(j, up[j]);
  }
  if constexpr (PRE == kPreRmsNorm) {
    const float ss = row_reduce(part.sum_squares(), lg, red_f, [](float a, float b) { return a + b; });
    part.normalise(w, rsqrtf(ss / static_cast<float>(K) + eps), in_row, lg, K);
  }
  const uint32_t amax = row_reduce(part.amax(), lg, red_u, [](uint32_t a, uint32_t b) { return max(a, b); });
  if (!live) return;
  if (in_row == 0) scale[row] = row_scale<T>(amax);
  part.template store<T>(q + row * Kp, amax, in_row, lg, Kp);
}

ACCERL_DEVINL void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// SwiGLU of many rows: persistent blocks of 256 threads take 256 >> lg rows at a time out of a ring of shared memory
// that bulk copies keep full, so that memory never waits for a row's reduction. Bound by instructions more than by
// memory: [8192, 2 x 8960] takes 78 us of which its bytes need 56.
constexpr int kBulkThreads = 256;
constexpr int kBulkMaxStages = 4;
constexpr int kBulkSmem = 74 * 1024;  // three blocks an SM
template <int NC>
__global__ void __launch_bounds__(kBulkThreads) quantize_rows_bulk_kernel(const __nv_bfloat16* __restrict__ x, long long ldx,
                                                                        int8_t* __restrict__ q, float* __restrict__ scale,
                                                                        long long rows, int K, int Kp, int lg, int stages,
                                                                        int* status) {
  extern __shared__ uint4 ring[];
  __shared__ uint64_t full[kBulkMaxStages];
  __shared__ uint32_t red_u[2][8];
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = kBulkThreads >> lg;  // rows per stage
  const int in_row = threadIdx.x & ((1 << lg) - 1), slot = threadIdx.x >> lg;
  const uint32_t row_bytes = static_cast<uint32_t>(K) * 4u;
  const long long batches = (rows + per - 1) / per;
  uint8_t* base = reinterpret_cast<uint8_t*>(ring);
  auto load = [&](long long batch, int s) {  // one thread
    const int n = static_cast<int>(min(static_cast<long long>(per), rows - batch * per));
    mbar_arrive_expect_tx(&full[s], n * row_bytes);
    for (int i = 0; i < n; ++i)
      bulk_load(base + (s * per + i) * row_bytes, x + (batch * per + i) * ldx, row_bytes, &full[s]);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
    for (int s = 0; s < stages; ++s) {
      const long long b = blockIdx.x + static_cast<long long>(s) * gridDim.x;
      if (b < batches) load(b, s);
    }
  }
  __syncthreads();
  int s = 0, buf = 0;
  uint32_t phase = 0;
  for (long long b = blockIdx.x; b < batches; b += gridDim.x) {
    const bool ok = mbar_wait(&full[s], phase, status, kStatusTimeoutProducer);
    const long long row = b * per + slot;
    const bool live = row < rows;
    const uint8_t* src = base + (s * per + slot) * row_bytes;
    RowPart<NC> part;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = ((j << lg) + in_row) * 8;
      if (live && part.inside(j, c, K)) {
        part.v[j] = *reinterpret_cast<const uint4*>(src + c * 2);
        part.swiglu(j, *reinterpret_cast<const uint4*>(src + (K + c) * 2));
      } else {
        part.v[j] = make_uint4(0, 0, 0, 0);
      }
    }
    const int w0 = slot << (lg - 5);
    uint32_t amax = __reduce_max_sync(0xffffffffu, part.amax());
    if (lane == 0) red_u[buf][warp] = amax;
    // everyone has read the stage (and the wait ran out for all or for nobody)
    if (!__syncthreads_and(ok)) {
      // no copy stays in flight into a finished block
      if (threadIdx.x == 0)
        for (int k = 0; k < stages; ++k)
          if (b + static_cast<long long>(k) * gridDim.x < batches)
            mbar_wait(&full[(s + k) % stages], phase ^ (s + k >= stages ? 1u : 0u), nullptr, 0, 20000000ull);
      return;
    }
    const long long next = b + static_cast<long long>(stages) * gridDim.x;
    if (threadIdx.x == 0 && next < batches) load(next, s);
    amax = __reduce_max_sync(0xffffffffu, red_u[buf][w0 + (lane & ((1 << (lg - 5)) - 1))]);
    if (live) {
      if (in_row == 0) scale[row] = row_scale<__nv_bfloat16>(amax);
      part.template store<__nv_bfloat16>(q + row * Kp, amax, in_row, lg, Kp);
    }
    buf ^= 1;
    if (++s == stages) {
      s = 0;
      phase ^= 1u;
    }
  }
}

// Any K, stride and alignment: one block per row, the row read twice (the second time from cache) in the aligned
// chunks of 8 that cover it. For rows longer than the registers of a block hold, and for odd ones. Bound by
// instructions: [4096, 4095] takes 21 us, where [4096, 4096] above takes 10 (element by element: 45).
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(const T* __restrict__ x, long long ldx,
                                                                int8_t* __restrict__ q, float* __restrict__ scale,
                                                                int K, int Kp) {
  pdl_launch_dependents();
  __shared__ uint32_t red_u[32];
  const long long row = blockIdx.x;
  const unsigned short* xr = reinterpret_cast<const unsigned short*>(x) + row * ldx;
  // chunks of 8 elements from the 16-byte boundary at or before the row; zeros outside the row
  const int head = static_cast<int>((reinterpret_cast<uintptr_t>(xr) & 15) >> 1);
  const uint4* src = reinterpret_cast<const uint4*>(xr - head);
  auto chunk = [&](int ch) -> uint4 {
    const int i0 = ch * 8 - head;
    if (i0 >= 0 && i0 + 8 <= K) return src[ch];
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = i0 + 2 * j, o = e + 1;
      const uint32_t lo = (e >= 0 && e < K) ? xr[e] : 0u, hi = (o >= 0 && o < K) ? xr[o] : 0u;
      w[j] = lo | (hi << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  uint32_t m2 = 0;
  for (int c = threadIdx.x; c * 8 < head + K; c += blockDim.x) {
    const uint4 v = chunk(c);
    m2 = __vmaxu2(m2, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
  }
  const uint32_t amax = row_reduce(amax_pair(m2), 8, red_u, [](uint32_t a, uint32_t b) { return max(a, b); });
  const RowQuant s = row_quant<T>(amax);
  if (threadIdx.x == 0) scale[row] = row_scale<T>(amax);
  const bool finite = amax < Half16<T>::kInf;
  for (int c = threadIdx.x; c * 8 < Kp; c += blockDim.x) {
    // 8 elements of the row out of two chunks: a shift by `head` halves, the same for all of the row
    const uint4 a = chunk(c), b = head ? chunk(c + 1) : make_uint4(0, 0, 0, 0);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (head & 4)
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    if (head & 2)
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    if (head & 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Half16<T>::unpack(w[i]);
      o[2 * i] = quant_bits(f.x, s);
      o[2 * i + 1] = quant_bits(f.y, s);
    }
    *reinterpret_cast<uint2*>(q + row * Kp + c * 8) =
        finite ? make_uint2(pack4(o[0], o[1], o[2], o[3]), pack4(o[4], o[5], o[6], o[7])) : make_uint2(0, 0);
  }
}

// ------------------------------------------------------------------------------------------------
// product
// ------------------------------------------------------------------------------------------------
// Instruction descriptor for kind::i8: signed 8-bit operands, both K-major, a 32-bit integer accumulator.
__host__ __device__ constexpr uint32_t make_idesc_s8_s32(int M, int N) {
  return (2u << 4)                                 // D format: s32
         | (1u << 7)                               // A format: s8
         | (1u << 10)                              // B format: s8
         | (static_cast<uint32_t>(N >> 3) << 17)   // N / 8
         | (static_cast<uint32_t>(M >> 4) << 24);  // M / 16
}

ACCERL_DEVINL void umma_s8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

constexpr int kI8BK = 128;         // elements (= bytes) of K per stage: one 128-byte swizzled row
constexpr int kI8Rows = 128;       // weight rows per tile
constexpr int kI8MaxTokens = 128;  // per tile of the streaming kernel
constexpr int kI8Threads = 192;

enum OutType : int { kOutBf16 = 0, kOutF16 = 1, kOutF32 = 2 };

struct Int8Params {
  int M, N, K;
  const float* sx;
  const float* sw;
  const void* bias;
  const void* residual;
  long long ldr;
  void* out;
  long long ldo;
  int out_type;  // of out; bias and residual are in_type
  int in_type;
  int bt, stages;                  // few tokens: tokens per tile, ring size
  int tiles_m, tiles_n, group_m;   // many tokens: the tile grid
  int w_early;                     // weight loads need not wait for the kernel before
  int* status;
};

ACCERL_DEVINL void st_cluster_s32(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
// the two halves of cluster_sync
ACCERL_DEVINL void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
ACCERL_DEVINL void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
ACCERL_DEVINL void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
ACCERL_DEVINL uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

ACCERL_DEVINL float load_as_float(const void* p, long long i, int type) {
  if (type == kOutBf16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  if (type == kOutF16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}
ACCERL_DEVINL void store_from_float(void* p, long long i, int type, float v) {
  if (type == kOutBf16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16(v);
  else if (type == kOutF16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<float*>(p)[i] = v;
}

// acc * sx * sw + bias without leaving fp32's range on the way to a result inside it. The product of two scales may
// (1e-20 each; 1e37 each, with a sum of 0). acc * sx may not, up to sx = 2^96: below 2^127, and as the multiple of sx's
// own step that it is, without loss below the normal range. Larger scales are taken 2^64 times smaller and the result
// back. (One multiplication more than the product of the scales takes: 185 us for 183 at 8192 x 1536 x 17920.)
struct TokenScale {
  float s, back;
};
ACCERL_DEVINL TokenScale token_scale(float sx) {
  const bool large = sx > 0x1p96f;
  return TokenScale{large ? sx * 0x1p-64f : sx, large ? 0x1p64f : 1.f};
}
ACCERL_DEVINL float scaled(float acc, const TokenScale& t, float sw, float bias) {
  return __fmaf_rn(__fmul_rn(__fmul_rn(acc, t.s), sw), t.back, bias);
}

// Four neighbouring channels of a row: the residual as it is loaded, and y = acc * sx * sw + bias (+ residual).
ACCERL_DEVINL uint4 load_residual4(const Int8Params& p, long long t, int n) {
  if (!p.residual) return make_uint4(0, 0, 0, 0);
  const long long at = t * p.ldr + n;
  if (p.in_type == kOutF32) return *reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p.residual) + at);
  const uint2 r = *reinterpret_cast<const uint2*>(reinterpret_cast<const unsigned short*>(p.residual) + at);
  return make_uint4(r.x, r.y, 0, 0);
}
template <int OUT>
ACCERL_DEVINL void finish4(const Int8Params& p, long long t, int n, int4 acc, float sx, float4 sw, float4 b, uint4 r) {
  const TokenScale ts = token_scale(sx);
  float4 y = make_float4(scaled(static_cast<float>(acc.x), ts, sw.x, b.x), scaled(static_cast<float>(acc.y), ts, sw.y, b.y),
                         scaled(static_cast<float>(acc.z), ts, sw.z, b.z), scaled(static_cast<float>(acc.w), ts, sw.w, b.w));
  if (p.residual) {
    if (p.in_type == kOutF32) {
      y.x += __uint_as_float(r.x), y.y += __uint_as_float(r.y), y.z += __uint_as_float(r.z), y.w += __uint_as_float(r.w);
    } else {
      const bool bf = p.in_type == kOutBf16;
      const float2 lo = bf ? Half16<__nv_bfloat16>::unpack(r.x) : Half16<__half>::unpack(r.x);
      const float2 hi = bf ? Half16<__nv_bfloat16>::unpack(r.y) : Half16<__half>::unpack(r.y);
      y.x += lo.x, y.y += lo.y, y.z += hi.x, y.w += hi.y;
    }
  }
  const long long at = t * p.ldo + n;
  if constexpr (OUT == kOutF32)
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = y;
  else if constexpr (OUT == kOutBf16)
    *reinterpret_cast<uint2*>(reinterpret_cast<unsigned short*>(p.out) + at) =
        make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
  else
    *reinterpret_cast<uint2*>(reinterpret_cast<unsigned short*>(p.out) + at) =
        make_uint2(pack_f16x2(y.x, y.y), pack_f16x2(y.z, y.w));
}

// Few tokens: one tile of 128 output channels x bt tokens per cluster of CTAs. The weight rows are the MMA's
// 128 rows, so a decode batch of few tokens wastes no tensor rows and streams the weight once. The CTAs of a
// cluster split K (there are only N / 128 tiles to spread over 148 SMs): each sends its integer partial of a token to
// the CTA that finishes that token (every CTA a share of them), straight from TMEM into that one's shared memory.
// Integer sums have no order, so the split changes no bit. The two cluster barriers are split into arrival and wait:
// the first (everybody has started) hides behind the products, the second is the only wait for the peers.
//   warp 0: TMA producer into a ring of stages;  warp 1: TMEM and MMA issue;  warps 2-5: accumulator to
//   shared memory;  then all warps: a token row each, four neighbouring channels a lane (VEC: aligned rows) or
//   every 32nd channel.
// Bound by the latency of one CTA's chain (setup, first tile, exchange, store: about 4 us) where there are few tiles,
// by memory where there are many. Measured without the quantising kernel: 1 x 1536 x 2048 4.7 us, 64 x 1536 x 17920
// 11.9 us (2.5 TB/s), 256 x 8960 x 1536 14.6 us, 1 x 1536 x 151936 41 us (5.7 TB/s). VEC spills 4 bytes a thread.
template <int OUT, bool VEC>
__global__ void __launch_bounds__(kI8Threads) gemm_int8_stream_kernel(const __grid_constant__ CUtensorMap tmW,
                                                                      const __grid_constant__ CUtensorMap tmX,
                                                                      const Int8Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[16], empty[16], done;
  __shared__ uint32_t tmem_slot;
  __shared__ float sx_s[kI8MaxTokens];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * kI8Rows, t0 = blockIdx.y * p.bt;
  const int split = blockIdx.z, splits = gridDim.z;
  const int kbs_all = (p.K + kI8BK - 1) / kI8BK;
  const int kb_first = static_cast<int>(static_cast<long long>(kbs_all) * split / splits);
  const int kbs = static_cast<int>(static_cast<long long>(kbs_all) * (split + 1) / splits) - kb_first;
  const uint32_t stage_bytes = (kI8Rows + p.bt) * kI8BK;
  uint32_t cols = 32;
  while (cols < static_cast<uint32_t>(p.bt)) cols <<= 1;
  bool ok = true;
  int issued = 0;
  // warp 0 goes on to its loads as soon as the barriers stand; the others meet behind the TMEM allocation
  if (warp == 0) {
    if (lane == 0) {
      for (int s = 0; s < p.stages; ++s) {
        mbar_init(&full[s], 1);
        mbar_init(&empty[s], 1);
      }
      mbar_init(&done, 1);
      fence_mbar_init();
    }
    __syncwarp();
    named_bar_arrive(1, kI8Threads);
    if (lane == 0) {
      // behind a quantising kernel the first weight tiles start even before the tokens are there (p.w_early: nothing
      // that kernel writes is part of the weight)
      if (!p.w_early) pdl_wait();
      for (; issued < min(p.stages, kbs); ++issued) {
        mbar_arrive_expect_tx(&full[issued], stage_bytes);
        tma_load_2d(smem + issued * stage_bytes, &tmW, &full[issued], (kb_first + issued) * kI8BK, n0);
        if (!p.w_early)
          tma_load_2d(smem + issued * stage_bytes + kI8Rows * kI8BK, &tmX, &full[issued], (kb_first + issued) * kI8BK, t0);
      }
      if (p.w_early) {
        pdl_wait();
        for (int s = 0; s < issued; ++s)
          tma_load_2d(smem + s * stage_bytes + kI8Rows * kI8BK, &tmX, &full[s], (kb_first + s) * kI8BK, t0);
      }
    }
    __syncwarp();
  } else {
    if (warp == 1) tmem_alloc(&tmem_slot, cols);
    tc_fence_before();
    named_bar_sync(1, kI8Threads);
    tc_fence_after();
  }
  pdl_wait();
  if (splits > 1) cluster_arrive_relaxed();  // nothing to publish yet: only that this CTA has started
  const uint32_t tbase = warp == 0 ? 0u : tmem_slot;
  // the tokens this CTA finishes, and where the partials of all of the cluster's CTAs for them arrive
  const int share = p.bt / splits, share_lg = 31 - __clz(share);  // powers of two
  int* parts = reinterpret_cast<int*>(smem + (splits > 1 ? p.stages * stage_bytes : 0));
  // the lane's channel scales and bias, loaded long before they are used
  float4 sw = make_float4(0.f, 0.f, 0.f, 0.f), b = sw;
  if constexpr (VEC) {
    const int n = n0 + lane * 4;
    if (n < p.N) {
      sw = *reinterpret_cast<const float4*>(p.sw + n);
      if (p.bias)
        b = make_float4(load_as_float(p.bias, n, p.in_type), load_as_float(p.bias, n + 1, p.in_type),
                        load_as_float(p.bias, n + 2, p.in_type), load_as_float(p.bias, n + 3, p.in_type));
    }
  }

  if (warp == 0) {
    if (lane == 0) {
      for (int kb = issued; kb < kbs; ++kb) {
        const int s = kb % p.stages;
        if (!mbar_wait(&empty[s], ((kb / p.stages) & 1) ^ 1u, p.status, kStatusTimeoutProducer)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[s], stage_bytes);
        tma_load_2d(smem + s * stage_bytes, &tmW, &full[s], (kb_first + kb) * kI8BK, n0);
        tma_load_2d(smem + s * stage_bytes + kI8Rows * kI8BK, &tmX, &full[s], (kb_first + kb) * kI8BK, t0);
        ++issued;
      }
      // never leave a copy in flight into the shared memory of a finished CTA
      if (!ok)
        for (int kb = max(0, issued - p.stages); kb < issued; ++kb)
          mbar_wait(&full[kb % p.stages], (kb / p.stages) & 1, nullptr, 0, 20000000ull);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc_s8_s32(kI8Rows, p.bt);
      for (int kb = 0; kb < kbs; ++kb) {
        const int s = kb % p.stages;
        if (!mbar_wait(&full[s], (kb / p.stages) & 1, p.status, kStatusTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t w_addr = smem_u32(smem + s * stage_bytes);
        const uint32_t x_addr = w_addr + kI8Rows * kI8BK;
#pragma unroll
        for (int kk = 0; kk < kI8BK / 32; ++kk)
          umma_s8(tbase, make_sw128_desc(w_addr + kk * 32, 16, 1024), make_sw128_desc(x_addr + kk * 32, 16, 1024),
                  idesc, (kb | kk) != 0);
        umma_commit(&empty[s]);
      }
      if (ok) umma_commit(&done);
    }
  } else {
    for (int i = threadIdx.x - 64; i < p.bt; i += 128) sx_s[i] = t0 + i < p.M ? p.sx[t0 + i] : 0.f;
    ok = mbar_wait(&done, 0, p.status, kStatusTimeoutEpilogue);
    tc_fence_after();
  }
  __syncwarp();
  if (splits > 1) cluster_wait();
  if (warp >= 2 && ok) {  // a timed-out wait leaves what it finds there (the status word is set)
    const int quarter = warp & 3;  // TMEM lanes this warp may read
    const uint32_t t_row = tbase + (static_cast<uint32_t>(quarter * 32) << 16);
    const int ch = quarter * 32 + lane;
#pragma unroll 1
    for (int c0 = 0; c0 < min(p.bt, p.M - t0); c0 += 16) {
      uint32_t v[16];
      tmem_ld16(t_row + c0, v);
      tmem_wait_ld();
      if (splits == 1) {
        // every MMA of this CTA has read its stages: their memory takes the accumulator, [token][channel]
#pragma unroll
        for (int i = 0; i < 16; ++i) parts[(c0 + i) * kI8Rows + ch] = static_cast<int>(v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {  // [sender][token of the share][channel] at the token's owner
          const int c = c0 + i, owner = c >> share_lg;
          st_cluster_s32(map_shared_rank(parts + (split * share + (c & (share - 1))) * kI8Rows + ch, owner),
                         static_cast<int>(v[i]));
        }
      }
    }
  }
  if (warp >= 2) tc_fence_before();
  __syncwarp();
  if (splits > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }

  const int c_lo = split * share, c_hi = min(min(p.bt, p.M - t0), c_lo + share);
  constexpr int kWarps = kI8Threads / 32;
  if constexpr (VEC) {
    const int n = n0 + lane * 4;
    if (n < p.N) {  // N is a multiple of 4
      constexpr int kRows = 4;  // tokens at once: their residuals are loaded before any result is stored
      for (int c0 = c_lo + warp; c0 < c_hi; c0 += kWarps * kRows) {
        uint4 res[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (c0 + i * kWarps < c_hi) res[i] = load_residual4(p, t0 + c0 + i * kWarps, n);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const int c = c0 + i * kWarps;
          if (c >= c_hi) break;
          const int4* src = reinterpret_cast<const int4*>(parts + (c - c_lo) * kI8Rows) + lane;
          int4 acc = *src;
          for (int r = 1; r < splits; ++r) {
            const int4 o = src[r * share * (kI8Rows / 4)];
            acc.x += o.x, acc.y += o.y, acc.z += o.z, acc.w += o.w;
          }
          finish4<OUT>(p, t0 + c, n, acc, sx_s[c], sw, b, res[i]);
        }
      }
    }
  } else {
    float sc[4], bi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + i * 32 + lane;
      sc[i] = n < p.N ? p.sw[n] : 0.f;
      bi[i] = (n < p.N && p.bias) ? load_as_float(p.bias, n, p.in_type) : 0.f;
    }
    constexpr int kRows = 4;
    for (int c0 = c_lo + warp; c0 < c_hi; c0 += kWarps * kRows) {
      float res[kRows][4];
#pragma unroll
      for (int j = 0; j < kRows; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = c0 + j * kWarps, n = n0 + i * 32 + lane;
          res[j][i] = p.residual && c < c_hi && n < p.N
                          ? load_as_float(p.residual, static_cast<long long>(t0 + c) * p.ldr + n, p.in_type)
                          : 0.f;
        }
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int c = c0 + j * kWarps;
        if (c >= c_hi) break;
        const TokenScale ts = token_scale(sx_s[c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = n0 + i * 32 + lane;
          if (n >= p.N) continue;
          const int* src = parts + (c - c_lo) * kI8Rows + i * 32 + lane;
          int acc = *src;
          for (int r = 1; r < splits; ++r) acc += src[r * share * kI8Rows];
          store_from_float(p.out, static_cast<long long>(t0 + c) * p.ldo + n, OUT,
                           scaled(static_cast<float>(acc), ts, sc[i], bi[i]) + res[j][i]);
        }
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, cols);
  }
}

// ---- many tokens: persistent CTA pairs, 256 tokens x 256 channels per tile ----
ACCERL_DEVINL void umma_s8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

constexpr int kI8Tile = 256;    // tokens and channels per tile of a CTA pair
constexpr int kI8Stages = 5;
constexpr int kI8HalfBytes = 128 * kI8BK;          // a CTA's 128 rows of either operand
constexpr int kI8StageBytes = 2 * kI8HalfBytes;
constexpr int kI8EpiWarps = 8;                     // two per TMEM lane quarter, half of the channels each
constexpr int kI8PairThreads = 64 + 32 * kI8EpiWarps;
constexpr int kI8EpiBytes = 32 * 128;              // staging per epilogue warp: 32 rows x 32 columns of fp32
constexpr int kI8PairSmem = kI8Stages * kI8StageBytes + kI8EpiWarps * kI8EpiBytes + 2 * 2 * kI8Tile * 4 + 1024;
static_assert(kI8PairSmem + 1024 <= 232448, "shared memory per CTA");

// tile t -> (token block, channel block), in groups of `group_m` token blocks for L2 reuse of the weight
ACCERL_DEVINL void int8_tile(const Int8Params& p, int t, int& m_blk, int& n_blk) {
  const int per_group = p.group_m * p.tiles_n;
  const int group = t / per_group;
  const int first = group * p.group_m;
  const int size = min(p.tiles_m - first, p.group_m);
  const int r = t % per_group;
  m_blk = first + r % size;
  n_blk = r / size;
}

// f[0..32) += residual[row, col0..col0 + 32), columns behind N left alone. Rows are 16-byte aligned.
ACCERL_DEVINL void add_residual32(float (&f)[32], const Int8Params& p, long long row, int col0) {
  const long long at = row * p.ldr + col0;
  if (col0 + 32 > p.N) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (col0 + i < p.N) f[i] += load_as_float(p.residual, at + i, p.in_type);
  } else if (p.in_type == kOutF32) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 r = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.residual) + at + i);
      f[i] += r.x;
      f[i + 1] += r.y;
      f[i + 2] += r.z;
      f[i + 3] += r.w;
    }
  } else {
    const bool bf = p.in_type == kOutBf16;
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      const uint4 r = *reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned short*>(p.residual) + at + i);
      const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = bf ? Half16<__nv_bfloat16>::unpack(rw[j]) : Half16<__half>::unpack(rw[j]);
        f[i + 2 * j] += a.x;
        f[i + 2 * j + 1] += a.y;
      }
    }
  }
}

// The two CTAs of a pair compute one 256 x 256 tile with tcgen05.mma.cta_group::2: each stages its 128
// tokens and 128 of the channels, the even CTA issues the MMAs, each drains the 128 x 256 accumulator of its
// tokens. Accumulators are double-buffered in TMEM, so the epilogue of a tile runs under the next one's
// products. TMA_OUT: the result leaves through swizzled shared memory and TMA stores (16-byte aligned rows);
// otherwise (rows that end inside 16 bytes among them), and for residuals that are not aligned, through fp32 staging and
// coalesced element stores.
// Bound by what L2 delivers (64 KB per 128 of K and tile: 12 to 14 TB/s in all; 5 stages, 4 cost 3 % more), where K is
// short also by the result's way through it (8192 x 1536 x 17920: 152 us without an epilogue, 157 without its stores),
// and by the last wave. Measured without the quantising kernel: 8192 x 1536 x 17920 180 us (2.5 POP/s), 8192 x 8960 x
// 1536 85 us (2.7; 81 behind the kernel that made its rows), 2048 x 4096 x 24576 143 us (2.9); 8-bit dense peak 3.3.
template <int OUT, bool TMA_OUT>
__global__ void __launch_bounds__(kI8PairThreads, 1)
    gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                          const __grid_constant__ CUtensorMap tmOut, const Int8Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smEpi = smem + kI8Stages * kI8StageBytes;
  float* sm_scale = reinterpret_cast<float*>(smEpi + kI8EpiWarps * kI8EpiBytes);  // [buffer][scale, bias][channel]
  __shared__ uint64_t full[kI8Stages], empty[kI8Stages], tfull[2], tempty[2];
  __shared__ uint32_t tmem_slot;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int kbs = (p.K + kI8BK - 1) / kI8BK;
  const int first = static_cast<int>(blockIdx.x >> 1), stride = static_cast<int>(gridDim.x >> 1);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kI8Stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * 32 * kI8EpiWarps);
    }
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmX);
    prefetch_tmap(&tmW);
  }
  if (warp == 1) tmem_alloc_pair(&tmem_slot, 2 * kI8Tile);
  pdl_wait();
  tc_fence_before();
  cluster_sync();  // barriers of both CTAs initialised before any remote signal
  tc_fence_after();
  const uint32_t tbase = tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, parity = 0;
      bool ok = true;
      for (int t = first; t < p.tiles_m * p.tiles_n && ok; t += stride) {
        int m_blk, n_blk;
        int8_tile(p, t, m_blk, n_blk);
        const int m0 = m_blk * kI8Tile + static_cast<int>(rank) * 128, n0 = n_blk * kI8Tile + static_cast<int>(rank) * 128;
        for (int kb = 0; kb < kbs; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, p.status, kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          const uint32_t bar = map_shared_rank(&full[stage], 0);  // both CTAs' bytes complete the even one's
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * kI8StageBytes);
          uint8_t* dst = smem + stage * kI8StageBytes;
          tma_load_2d_pair(dst, &tmX, bar, kb * kI8BK, m0);
          tma_load_2d_pair(dst + kI8HalfBytes, &tmW, bar, kb * kI8BK, n0);
          issued |= 1u << stage;
          parity = (parity & ~(1u << stage)) | (phase << stage);
          if (++stage == kI8Stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (ok) {
        // wait until the MMAs have consumed every stage this CTA filled: no commit may arrive after it left
        for (int i = 0; i < kI8Stages; ++i) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, p.status, kStatusTimeoutProducer)) break;
          if (++stage == kI8Stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      } else if (rank == 0) {
        for (int s = 0; s < kI8Stages; ++s)  // no copy stays in flight into a finished CTA
          if (issued & (1u << s)) mbar_wait(&full[s], (parity >> s) & 1u, nullptr, 0, 20000000ull);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = make_idesc_s8_s32(kI8Tile, kI8Tile);
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = first; t < p.tiles_m * p.tiles_n && ok; t += stride, ++local) {
        const int acc = local & 1;
        if (!mbar_wait(&tempty[acc], ((local >> 1) & 1) ^ 1u, p.status, kStatusTimeoutMma)) break;
        tc_fence_after();
        for (int kb = 0; kb < kbs; ++kb) {
          if (!mbar_wait(&full[stage], phase, p.status, kStatusTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t x_addr = smem_u32(smem + stage * kI8StageBytes), w_addr = x_addr + kI8HalfBytes;
#pragma unroll
          for (int kk = 0; kk < kI8BK / 32; ++kk)
            umma_s8_pair(tbase + acc * kI8Tile, make_sw128_desc(x_addr + kk * 32, 16, 1024),
                         make_sw128_desc(w_addr + kk * 32, 16, 1024), idesc, (kb | kk) != 0);
          umma_commit_pair(&empty[stage], 0x3);
          if (++stage == kI8Stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) umma_commit_pair(&tfull[acc], 0x3);
      }
    }
  } else {
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    const uint32_t tempty_even = map_shared_rank(&tempty[0], 0);
    uint8_t* wbuf = smEpi + (warp - 2) * kI8EpiBytes;
    int local = 0, chunk = 0;
    for (int t = first; t < p.tiles_m * p.tiles_n; t += stride, ++local) {
      int m_blk, n_blk;
      int8_tile(p, t, m_blk, n_blk);
      const int acc = local & 1;
      const int n0 = n_blk * kI8Tile;
      const int y0 = m_blk * kI8Tile + static_cast<int>(rank) * 128 + quarter * 32;  // first row of this warp
      const int row = y0 + lane;
      const bool row_ok = row < p.M;
      const TokenScale sx = token_scale(row_ok ? __ldg(p.sx + row) : 0.f);
      // channel scales and bias of the tile, one buffer per accumulator
      float* scale = sm_scale + acc * 2 * kI8Tile;
      for (int i = threadIdx.x - 64; i < kI8Tile; i += 32 * kI8EpiWarps) {
        const int n = n0 + i;
        scale[i] = n < p.N ? p.sw[n] : 0.f;
        scale[kI8Tile + i] = (n < p.N && p.bias) ? load_as_float(p.bias, n, p.in_type) : 0.f;
      }
      // the epilogue warps go on, or give up, together
      if (!named_bar_and(1, 32 * kI8EpiWarps, mbar_wait(&tfull[acc], (local >> 1) & 1, p.status, kStatusTimeoutEpilogue)))
        break;
      tc_fence_after();
      const uint32_t t_row = tbase + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kI8Tile;
      const int c_end = min(half * 128 + 128, p.N - n0);
      uint32_t v[32];
      if (half * 128 < c_end) tmem_ld32(t_row + half * 128, v);
#pragma unroll 1
      for (int c0 = half * 128; c0 < c_end; c0 += 32) {
        tmem_wait_ld();
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = static_cast<float>(static_cast<int>(v[i]));
        if (c0 + 32 < c_end) tmem_ld32(t_row + c0 + 32, v);  // the next columns travel while these are finished
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 s4 = *reinterpret_cast<const float4*>(scale + c0 + i);
          const float4 b4 = *reinterpret_cast<const float4*>(scale + kI8Tile + c0 + i);
          f[i] = scaled(f[i], sx, s4.x, b4.x);
          f[i + 1] = scaled(f[i + 1], sx, s4.y, b4.y);
          f[i + 2] = scaled(f[i + 2], sx, s4.z, b4.z);
          f[i + 3] = scaled(f[i + 3], sx, s4.w, b4.w);
        }
        const int col0 = n0 + c0;
        if constexpr (TMA_OUT) {
          if (p.residual && row_ok) add_residual32(f, p, row, col0);
          // 16-bit results: two buffers of 32 rows x 64 bytes; fp32: one of 32 x 128
          constexpr int kBufs = OUT == kOutF32 ? 1 : 2;
          uint8_t* buf = wbuf + (chunk % kBufs) * (kI8EpiBytes / kBufs);
          ++chunk;
          if (lane == 0) bulk_wait_read<kBufs - 1>();  // the store issued from this buffer has read it
          __syncwarp();
          if constexpr (OUT == kOutF32) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<float4*>(buf + swz128(lane, j)) =
                  make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t o[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                o[i] = OUT == kOutBf16 ? pack_bf16x2(f[8 * j + 2 * i], f[8 * j + 2 * i + 1])
                                       : pack_f16x2(f[8 * j + 2 * i], f[8 * j + 2 * i + 1]);
              *reinterpret_cast<uint4*>(buf + swz64(lane, j)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
          }
          fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmOut, buf, col0, y0);
            bulk_commit();
          }
        } else {
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float4*>(wbuf + swz128(lane, j)) =
                make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
          __syncwarp();
          const int n = col0 + lane;
          if (n < p.N) {
            const int rows = min(32, p.M - y0);
            for (int r0 = 0; r0 < rows; r0 += 8) {
              float y[8];  // the residual of 8 rows is loaded before any of their results is stored
#pragma unroll
              for (int i = 0; i < 8; ++i)
                y[i] = p.residual && r0 + i < rows
                           ? load_as_float(p.residual, static_cast<long long>(y0 + r0 + i) * p.ldr + n, p.in_type)
                           : 0.f;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int r = r0 + i;
                if (r < rows)
                  store_from_float(p.out, static_cast<long long>(y0 + r) * p.ldo + n, OUT,
                                   y[i] + *reinterpret_cast<const float*>(wbuf + swz128(r, lane >> 2) + (lane & 3) * 4));
              }
            }
          }
        }
      }
      tc_fence_before();
      mbar_arrive_cluster(tempty_even + acc * 8);
    }
    if (TMA_OUT && lane == 0) bulk_wait<0>();
  }
  __syncthreads();
  tc_fence_before();
  cluster_sync();  // neither CTA leaves while the other may still signal into its shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tbase, 2 * kI8Tile);
  }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
namespace {

PFN_cuTensorMapEncodeTiled_v12000 int8_encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// Map of int8 rows (pitch in bytes, a multiple of 16): boxes of 128 bytes x `box_rows`, 128B swizzle.
bool make_int8_map(CUtensorMap* out, const void* ptr, uint64_t pitch, uint64_t rows, uint32_t box_rows) {
  auto fn = int8_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {pitch, rows};
  cuuint64_t strides[1] = {pitch};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(kI8BK), box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Map of the output (16-byte aligned rows) for tiles of 32 columns x 32 rows.
bool make_out_map(CUtensorMap* out, const Int8Params& p) {
  const uint64_t es = p.out_type == kOutF32 ? 4 : 2;
  auto fn = int8_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.N), static_cast<cuuint64_t>(p.M)};
  cuuint64_t strides[1] = {p.ldo * es};
  cuuint32_t box[2] = {32, 32};
  cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType dt = p.out_type == kOutF32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : p.out_type == kOutF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return fn(out, dt, 2, p.out, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            es == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaLaunchConfig_t cluster_config(dim3 grid, int threads, int smem, cudaStream_t s, cudaLaunchAttribute* attr, unsigned x,
                                  unsigned z) {
  cudaLaunchConfig_t cfg = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = x;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = z;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cfg;
}

template <int OUT, bool TMA_OUT>
int launch_pair(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mo, const Int8Params& p, cudaStream_t s) {
  auto kern = gemm_int8_pair_kernel<OUT, TMA_OUT>;
  static std::atomic<int> cache[kMaxHostDevices];  // pairs that can be resident at once, per device
  const int dev = host_current_device();
  if (dev < 0 || dev >= kMaxHostDevices) return -14;
  cudaLaunchAttribute attr[2];
  int pairs = cache[dev].load(std::memory_order_acquire);
  if (pairs == 0) {
    cudaError_t e = smem_attr_once<gemm_int8_pair_kernel<OUT, TMA_OUT>>(kI8PairSmem);
    if (e != cudaSuccess) return static_cast<int>(e);
    cudaLaunchConfig_t cfg = cluster_config(dim3(2 * (device_sm_count() / 2)), kI8PairThreads, kI8PairSmem, s, attr, 2, 1);
    cfg.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&pairs, kern, &cfg);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (pairs < 1) return -13;
    cache[dev].store(pairs, std::memory_order_release);
  }
  const int grid = 2 * std::min(pairs, p.tiles_m * p.tiles_n);
  cudaLaunchConfig_t cfg = cluster_config(dim3(grid), kI8PairThreads, kI8PairSmem, s, attr, 2, 1);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, mx, mw, mo, p));
}

template <int OUT, bool VEC>
int launch_stream(const CUtensorMap& mw, const CUtensorMap& mx, const Int8Params& p, dim3 grid, int smem, cudaStream_t s) {
  cudaError_t e = smem_attr_once<gemm_int8_stream_kernel<OUT, VEC>>(201 * 1024);
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = cluster_config(grid, kI8Threads, smem, s, attr, 1, grid.z);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, gemm_int8_stream_kernel<OUT, VEC>, mw, mx, p));
}

// SMs that clusters of `splits` CTAs can use at once, one CTA each: larger ones do not fill a GPC.
int int8_room(int splits, int sms) { return splits >= 4 ? sms * 9 / 10 : sms; }

// Which kernel runs a product: bt = 0 the persistent pairs, else the streaming kernel with bt tokens per tile and
// `splits` CTAs per tile. The candidate with the least estimated cost wins. An estimate has a fixed part, a part per
// 128 elements of K and one per token of the tile, times the share of an SM that a CTA gets (pairs: the waves); its
// constants are fitted to the times of all candidates over M 1..4096 and fourteen (K, N) from (300, 700) to (1536,
// 151936) so that the choice is right (they are no times): the chosen candidate took 1.4 % longer than the best on
// average, 18 % at most. `store_ok`: TMA can store the result; `vec`: the streaming kernel can store four channels at
// once. What element stores cost either is fitted to eight more (K, N) with such N (512 x 17913 to 8000 x 1537): 3 %
// longer on average, 31 % at most (without: 5 % and 113 %).
struct Int8Plan {
  int bt, splits;
};
Int8Plan plan_int8(int M, int N, int K, bool store_ok, bool vec, int sms) {
  const int kbs = (K + kI8BK - 1) / kI8BK;
  const double pair_tiles = static_cast<double>((M + kI8Tile - 1) / kI8Tile) * ((N + kI8Tile - 1) / kI8Tile);
  const double waves = std::ceil(pair_tiles / (sms / 2));
  double best = 8.5 + waves * kbs * 0.326 + (waves - 1) * 2.06 + (store_ok ? 0.0 : 6.0 + waves * 10.0);
  Int8Plan plan{0, 1};
  for (int bt = 16; bt <= kI8MaxTokens && (bt == 16 || bt < 2 * M); bt *= 2) {
    if ((M + bt - 1) / bt > 65535) continue;  // a grid's second dimension
    const double tiles = static_cast<double>((M + bt - 1) / bt) * ((N + kI8Rows - 1) / kI8Rows);
    for (int sp = 1; sp <= 8 && sp <= kbs; sp *= 2) {
      const double ctas = tiles * sp;
      if (sp > 1 && ctas > 4 * sms) break;
      const double room = int8_room(sp, sms);
      const double t = 6.47 + (sp > 1 ? 0.33 : 0.0) +
                       (ctas <= room ? 1.0 : (ctas > 2 * room && sp == 1 ? 0.758 : 1.24) * ctas / room) *
                           (((kbs + sp - 1) / sp) * (0.252 + 0.00177 * bt) +
                            ((sp > 1 ? 0.0197 : 0.0139) + (vec ? 0.0 : 0.02)) * bt);
      if (t < best) {
        best = t;
        plan = Int8Plan{bt, sp};
      }
    }
  }
  return plan;
}

template <int NC>
int launch_quantize_bulk(const __nv_bfloat16* x, long long ldx, int8_t* q, float* scale, long long rows, int K, int Kp, int lg,
                       int stages, int smem, int* status, cudaStream_t s) {
  const cudaError_t e = smem_attr_once<quantize_rows_bulk_kernel<NC>>(kBulkSmem);
  if (e != cudaSuccess) return static_cast<int>(e);
  const long long batches = (rows + (kBulkThreads >> lg) - 1) / (kBulkThreads >> lg);
  const int resident = device_sm_count() * std::min(4, (224 * 1024) / (smem + 2048));
  const unsigned grid = static_cast<unsigned>(std::min<long long>(batches, resident));
  quantize_rows_bulk_kernel<NC><<<grid, kBulkThreads, smem, s>>>(x, ldx, q, scale, rows, K, Kp, lg, stages, status);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int PRE>
int launch_quantize(const T* x, long long ldx, const T* w, float eps, int8_t* q, float* scale, long long rows, int K,
                    int Kp, int* status, cudaStream_t s) {
  const bool vec = K % 8 == 0 && ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  const int chunks = (Kp + 7) / 8;
  if (!vec || chunks > 8 * 512) {
    if constexpr (PRE == kPreNone) {
      quantize_rows_any_kernel<T><<<static_cast<unsigned>(rows), 256, 0, s>>>(x, ldx, q, scale, K, Kp);
      return static_cast<int>(cudaGetLastError());
    } else {
      return -2;
    }
  }
  // the fewest threads a row that hold it in 4 chunks each, 256 at most
  int lg = 5;
  while (lg < 8 && chunks > (4 << lg)) ++lg;
  int nc = (chunks + (1 << lg) - 1) >> lg;
  if constexpr (PRE == kPreSwiglu) {
    // The ring pays where an SM sees many rows: SwiGLU of 8960 columns took 78 us against 91 at 8192 rows, 37 against
    // 33 at 2048. A ring for plain rows and RMSNorm was never faster (8192 x 8960: 42 us either way; 16384 x 4096
    // RMSNorm: 60 against 49), and they have none.
    const int per = kBulkThreads >> lg;
    const int stage = per * K * 4;
    const int stages = std::min(kBulkMaxStages, kBulkSmem / stage);
    if (rows > 24ll * per * device_sm_count() && stages >= 2) {  // two rows of K fit: K <= 9472, at most 5 chunks
      auto launch = [&](auto n) {
        return launch_quantize_bulk<decltype(n)::value>(x, ldx, q, scale, rows, K, Kp, lg, stages, stages * stage, status, s);
      };
      if (nc <= 1) return launch(std::integral_constant<int, 1>());
      if (nc <= 2) return launch(std::integral_constant<int, 2>());
      if (nc <= 3) return launch(std::integral_constant<int, 3>());
      if (nc <= 4) return launch(std::integral_constant<int, 4>());
      return launch(std::integral_constant<int, 5>());
    }
  }
  if (nc > 4) {
    lg = 9;
    nc = (chunks + 511) / 512;
  }
  const int block = std::max(1 << lg, 128);
  const unsigned grid = static_cast<unsigned>((rows + (block >> lg) - 1) / (block >> lg));
  auto launch = [&](auto kern) { kern<<<grid, block, 0, s>>>(x, ldx, w, eps, q, scale, rows, K, Kp, lg); };
  if (nc <= 1) launch(quantize_rows_kernel<T, PRE, 1>);
  else if (nc <= 2) launch(quantize_rows_kernel<T, PRE, 2>);
  else if (nc <= 3) launch(quantize_rows_kernel<T, PRE, 3>);
  else if (nc <= 4) launch(quantize_rows_kernel<T, PRE, 4>);
  else launch(quantize_rows_kernel<T, PRE, 8>);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace
}  // namespace accerl

// x [rows, K] (pre 2: [rows, 2K]) of 16-bit floats (half: 0 bf16, 1 fp16; pre 1 and 2 are bf16) -> q
// [rows, Kp] with Kp = K rounded up to 16 (zeros behind K) and scale [rows]. -2: a norm or SwiGLU row
// whose size, stride or alignment does not fit 16-byte accesses.
extern "C" int accerl_quantize_rows(const void* x, long long ldx, int half, int pre, const void* w, float eps, void* q,
                                    float* scale, long long rows, int K, int* status, cudaStream_t s) {
  using namespace accerl;
  if (rows <= 0) return 0;
  if (K <= 0 || rows > 0x7fffffffll) return -1;
  const int Kp = (K + 15) / 16 * 16;
  int8_t* qp = reinterpret_cast<int8_t*>(q);
  if (half) {
    if (pre != kPreNone) return -3;
    return launch_quantize<__half, kPreNone>(reinterpret_cast<const __half*>(x), ldx, nullptr, eps, qp, scale, rows, K,
                                             Kp, status, s);
  }
  const auto* xb = reinterpret_cast<const __nv_bfloat16*>(x);
  const auto* wb = reinterpret_cast<const __nv_bfloat16*>(w);
  if (pre == kPreRmsNorm) return launch_quantize<__nv_bfloat16, kPreRmsNorm>(xb, ldx, wb, eps, qp, scale, rows, K, Kp, status, s);
  if (pre == kPreSwiglu) return launch_quantize<__nv_bfloat16, kPreSwiglu>(xb, ldx, nullptr, eps, qp, scale, rows, K, Kp, status, s);
  return launch_quantize<__nv_bfloat16, kPreNone>(xb, ldx, nullptr, eps, qp, scale, rows, K, Kp, status, s);
}

// The kernel that accerl_gemm_int8 takes on the current device: tokens per tile of the streaming kernel and its CTAs per
// tile, or 0 and 1 for the persistent pairs. `store_ok`, `vec`: as for plan_int8.
extern "C" int accerl_int8_plan(int M, int N, int K, int store_ok, int vec, int* splits) {
  const accerl::Int8Plan plan = accerl::plan_int8(M, N, K, store_ok != 0, vec != 0, accerl::device_sm_count());
  *splits = plan.splits;
  return plan.bt;
}

// out [M, N] (out_type) = sx sw (qx qw^T) (+ bias [N]) (+ residual [M, N]), bias and residual of in_type
// (types: 0 bf16, 1 fp16, 2 fp32). qx [M, Kp] and qw [N, Kp], Kp = K rounded up to 16. `w_early`: the kernel
// before this one on the stream writes nothing of the weight, so its loads need not wait for that kernel.
extern "C" int accerl_gemm_int8(const void* qx, const float* sx, const void* qw, const float* sw, int M, int N, int K,
                                const void* bias, const void* residual, long long ldr, int in_type, void* out,
                                long long ldo, int out_type, int w_early, int* status, cudaStream_t stream) {
  using namespace accerl;
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K > 133144) return -1;
  if ((reinterpret_cast<uintptr_t>(qx) | reinterpret_cast<uintptr_t>(qw)) & 15) return -3;
  const uint64_t Kp = (static_cast<uint64_t>(K) + 15) / 16 * 16;
  Int8Params p;
  p.M = M;
  p.N = N;
  p.K = K;
  p.sx = sx;
  p.sw = sw;
  p.bias = bias;
  p.residual = residual;
  p.ldr = ldr;
  p.out = out;
  p.ldo = ldo;
  p.out_type = out_type;
  p.in_type = in_type;
  p.status = status;
  p.w_early = w_early;
  const int es = out_type == kOutF32 ? 4 : 2, rs = in_type == kOutF32 ? 4 : 2;
  // A TMA store cuts a row off at a multiple of 16 bytes: one that ends inside would write up to 14 bytes behind it.
  const bool store_ok = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && ldo * es % 16 == 0 && ldo >= N &&
                        static_cast<long long>(N) * es % 16 == 0 &&
                        (!residual || ((reinterpret_cast<uintptr_t>(residual) & 15) == 0 && ldr * rs % 16 == 0));
  const bool vec = N % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0 && ldo % 4 == 0 &&
                   (reinterpret_cast<uintptr_t>(sw) & 15) == 0 &&
                   (!residual || ((reinterpret_cast<uintptr_t>(residual) & 15) == 0 && ldr % 4 == 0));
  const Int8Plan plan = plan_int8(M, N, K, store_ok, vec, device_sm_count());
  CUtensorMap mx, mw, mo;
  if (plan.bt == 0) {
    p.tiles_m = (M + kI8Tile - 1) / kI8Tile;
    p.tiles_n = (N + kI8Tile - 1) / kI8Tile;
    p.group_m = 8;
    if (static_cast<long long>(p.tiles_m) * p.tiles_n > 0x3fffffff) return -4;
    if (!make_int8_map(&mx, qx, Kp, static_cast<uint64_t>(M), 128)) return -7;
    if (!make_int8_map(&mw, qw, Kp, static_cast<uint64_t>(N), 128)) return -8;
    if (store_ok) {
      if (!make_out_map(&mo, p)) return -9;
      if (out_type == kOutBf16) return launch_pair<kOutBf16, true>(mx, mw, mo, p, stream);
      if (out_type == kOutF16) return launch_pair<kOutF16, true>(mx, mw, mo, p, stream);
      return launch_pair<kOutF32, true>(mx, mw, mo, p, stream);
    }
    mo = mx;
    if (out_type == kOutBf16) return launch_pair<kOutBf16, false>(mx, mw, mo, p, stream);
    if (out_type == kOutF16) return launch_pair<kOutF16, false>(mx, mw, mo, p, stream);
    return launch_pair<kOutF32, false>(mx, mw, mo, p, stream);
  }
  p.bt = plan.bt;
  const dim3 grid((N + kI8Rows - 1) / kI8Rows, (M + p.bt - 1) / p.bt, plan.splits);
  const int kbs = (K + kI8BK - 1) / kI8BK;
  const int stage_bytes = (kI8Rows + p.bt) * kI8BK;
  // the accumulator: behind the stages where peers write it, else where the stages were
  const int acc_bytes = p.bt * kI8Rows * 4;
  // One CTA on an SM gets all of its shared memory, two half each. Of more, three an SM: while one finishes its tile the
  // others load (the LM head, 1 x 1536 x 151936: 46 us with two an SM, 41 with three, 43 with four).
  const long long ctas = static_cast<long long>(grid.x) * grid.y * grid.z, sms = int8_room(plan.splits, device_sm_count());
  const int room = (ctas <= sms ? 200 : (ctas > 2 * sms && plan.splits == 1 ? 72 : 100)) * 1024 -
                   (plan.splits > 1 ? acc_bytes : 0);
  p.stages = std::max(2, std::min({16, (kbs + plan.splits - 1) / plan.splits, room / stage_bytes}));
  const int smem_bytes =
      (plan.splits > 1 ? p.stages * stage_bytes + acc_bytes : std::max(p.stages * stage_bytes, acc_bytes)) + 1024;
  if (!make_int8_map(&mw, qw, Kp, static_cast<uint64_t>(N), kI8Rows)) return -7;
  if (!make_int8_map(&mx, qx, Kp, static_cast<uint64_t>(M), static_cast<uint32_t>(p.bt))) return -8;
  auto launch = [&](auto type) {
    constexpr int OUT = decltype(type)::value;
    return vec ? launch_stream<OUT, true>(mw, mx, p, grid, smem_bytes, stream)
               : launch_stream<OUT, false>(mw, mx, p, grid, smem_bytes, stream);
  };
  if (out_type == kOutBf16) return launch(std::integral_constant<int, kOutBf16>());
  if (out_type == kOutF16) return launch(std::integral_constant<int, kOutF16>());
  return launch(std::integral_constant<int, kOutF32>());
}
