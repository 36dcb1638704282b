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
#include <mutex>

#include "common.cuh"

namespace accerl {

// ------------------------------------------------------------------------------------------------
// rows to 8 bits
// ------------------------------------------------------------------------------------------------
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
  static ACCERL_DEVINL float2 unpack(uint32_t v) { return unpack_bf16x2(v); }
  static ACCERL_DEVINL float one(uint32_t bits) { return __uint_as_float(bits << 16); }
};
template <>
struct Half16<__half> {
  static constexpr uint32_t kInf = 0x7c00u;
  static ACCERL_DEVINL float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  static ACCERL_DEVINL float one(uint32_t bits) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits))); }
};

// Scale of a row and the factors that turn its elements into whole numbers. `amax` is the largest
// magnitude as a 16-bit pattern, whose order is that of the magnitudes, with infinities and NaN on top:
// a row that holds one gets scale NaN (its outputs are NaN) and zeros.
struct RowQuant {
  float scale, m127, a, inv;
};
template <typename T>
ACCERL_DEVINL RowQuant row_quant(uint32_t amax) {
  RowQuant o{0.f, 0.f, 0.f, 0.f};
  if (amax >= Half16<T>::kInf) {
    o.scale = __uint_as_float(0x7fffffffu);
  } else if (amax != 0u) {
    const float a = Half16<T>::one(amax);
    // a power of two keeps 1 / a, 127 x and the remainder below inside the normal range
    const float f = a < 0x1p-100f ? 0x1p100f : (a > 0x1p100f ? 0x1p-100f : 1.f);
    o.scale = __fdiv_rn(a, 127.f);
    o.a = a * f;
    o.m127 = 127.f * f;
    o.inv = __frcp_rn(o.a);
  }
  return o;
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
ACCERL_DEVINL uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// silu(g) u with the activation rounded to bf16, as swiglu_h gives it, without its division, which kept this
// kernel at the instruction limit: the quotient g / (1 + e^-g) from an approximate reciprocal, corrected by its
// exact remainder (Markstein, 1990). Gates beyond 80, where remainder or reciprocal could leave the normal
// range, take swiglu_h itself.
ACCERL_DEVINL float swiglu_row(float g, float u) {
  if (!(fabsf(g) < 80.f)) return swiglu_h(g, u);
  const float d = 1.f + __expf(-g);
  const float r = __fdividef(1.f, d);
  const float q = __fmul_rn(g, r);
  return bf16_round(__fmaf_rn(__fmaf_rn(-q, d, g), r, q)) * u;
}

// Reduction over the `tpr` threads of a row (a power of two, 32..blockDim); `red`, one slot per warp, is used
// by one reduction of the kernel only.
template <typename V, typename F>
ACCERL_DEVINL V row_reduce(V v, int tpr, V* red, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int w0 = (threadIdx.x / tpr) * (tpr >> 5);
    v = red[w0];
    for (int w = 1; w < (tpr >> 5); ++w) v = f(v, red[w0 + w]);
  }
  return v;
}

ACCERL_DEVINL uint32_t amax_pair(uint32_t m) { return max(m & 0xffffu, m >> 16); }

// One row per `tpr` threads, 8 elements a thread and chunk, the row held in registers between the maximum
// and the rounding so that it is read once. PRE turns the input row into the row to round: RMSNorm
// (x [rows, K], weight w) or SwiGLU (x = gate | up, [rows, 2K]), with the roundings of the framework's
// own kernels (both give rows in T).
template <typename T, int PRE, int NC>
__global__ void __launch_bounds__(512) quantize_rows_kernel(const T* __restrict__ x, long long ldx,
                                                            const T* __restrict__ w, float eps,
                                                            int8_t* __restrict__ q, float* __restrict__ scale,
                                                            long long rows, int K, int Kp, int tpr) {
  pdl_launch_dependents();  // the product may set itself up; it waits for this grid's end before it reads
  __shared__ uint32_t red_u[16];
  __shared__ float red_f[16];
  const int in_row = threadIdx.x % tpr;
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x / tpr) + threadIdx.x / tpr;
  const bool live = row < rows;
  const T* xr = x + (live ? row : 0) * ldx;
  // every load of the row is issued up front; chunks behind its end read its first one and are zeroed
  uint4 v[NC], up[PRE == kPreSwiglu ? NC : 1];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = (j * tpr + in_row) * 8;
    v[j] = *reinterpret_cast<const uint4*>(xr + (c < K ? c : 0));
    if constexpr (PRE == kPreSwiglu) up[j] = *reinterpret_cast<const uint4*>(xr + K + (c < K ? c : 0));
  }
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    if ((j * tpr + in_row) * 8 >= K) {
      v[j] = make_uint4(0, 0, 0, 0);
    } else if constexpr (PRE == kPreSwiglu) {
      uint32_t* g = reinterpret_cast<uint32_t*>(&v[j]);
      const uint32_t uw[4] = {up[j].x, up[j].y, up[j].z, up[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 fg = unpack_bf16x2(g[i]), fu = unpack_bf16x2(uw[i]);
        g[i] = pack_bf16x2(swiglu_row(fg.x, fu.x), swiglu_row(fg.y, fu.y));
      }
    }
  }
  if constexpr (PRE == kPreRmsNorm) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(&v[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_bf16x2(p[i]);
        ss += f.x * f.x + f.y * f.y;
      }
    }
    ss = row_reduce(ss, tpr, red_f, [](float a, float b) { return a + b; });
    const float r = rsqrtf(ss / static_cast<float>(K) + eps);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = (j * tpr + in_row) * 8;
      if (c >= K) continue;
      const uint4 wv = *reinterpret_cast<const uint4*>(w + c);
      const uint32_t ww[4] = {wv.x, wv.y, wv.z, wv.w};
      uint32_t* p = reinterpret_cast<uint32_t*>(&v[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_bf16x2(p[i]), g = unpack_bf16x2(ww[i]);
        const float2 n = unpack_bf16x2(pack_bf16x2(f.x * r, f.y * r));
        p[i] = pack_bf16x2(n.x * g.x, n.y * g.y);
      }
    }
  }
  uint32_t m2 = 0;
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(&v[j]);
#pragma unroll
    for (int i = 0; i < 4; ++i) m2 = __vmaxu2(m2, p[i] & 0x7fff7fffu);
  }
  const uint32_t amax = row_reduce(amax_pair(m2), tpr, red_u, [](uint32_t a, uint32_t b) { return max(a, b); });
  const RowQuant s = row_quant<T>(amax);
  if (!live) return;
  if (in_row == 0) scale[row] = s.scale;
  const bool finite = amax < Half16<T>::kInf;
  int8_t* qr = q + row * Kp;
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = (j * tpr + in_row) * 8;
    if (c >= Kp) continue;  // the columns K..Kp are written as zeros
    const uint32_t* p = reinterpret_cast<const uint32_t*>(&v[j]);
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Half16<T>::unpack(p[i]);
      b[2 * i] = finite ? quant_bits(f.x, s) : 0u;
      b[2 * i + 1] = finite ? quant_bits(f.y, s) : 0u;
    }
    *reinterpret_cast<uint2*>(qr + c) = make_uint2(pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7]));
  }
}

// Any K, stride and alignment: one block per row, element by element, the row read twice (the second time
// from cache). For rows longer than the registers of a block hold, and for odd ones.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(const T* __restrict__ x, long long ldx,
                                                                int8_t* __restrict__ q, float* __restrict__ scale,
                                                                int K, int Kp) {
  pdl_launch_dependents();
  __shared__ uint32_t red_u[32];
  const long long row = blockIdx.x;
  const unsigned short* xr = reinterpret_cast<const unsigned short*>(x) + row * ldx;
  uint32_t m = 0;
  for (int c = threadIdx.x; c < K; c += blockDim.x) m = max(m, xr[c] & 0x7fffu);
  const uint32_t amax = row_reduce(m, blockDim.x, red_u, [](uint32_t a, uint32_t b) { return max(a, b); });
  const RowQuant s = row_quant<T>(amax);
  if (threadIdx.x == 0) scale[row] = s.scale;
  const bool finite = amax < Half16<T>::kInf;
  for (int c = threadIdx.x; c < Kp; c += blockDim.x)
    q[row * Kp + c] = static_cast<int8_t>(
        (c < K && finite) ? static_cast<int>(quant_bits(Half16<T>::one(xr[c]), s) & 0xffu) : 0);
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

ACCERL_DEVINL int ld_cluster_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
ACCERL_DEVINL int4 ld_cluster_s32x4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
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

// Four neighbouring channels of a row: y = acc * sx * sw + bias (+ residual).
template <int OUT>
ACCERL_DEVINL void finish4(const Int8Params& p, long long t, int n, int4 acc, float sx, float4 sw, float4 b) {
  float4 y = make_float4(__fmaf_rn(static_cast<float>(acc.x), sx * sw.x, b.x),
                         __fmaf_rn(static_cast<float>(acc.y), sx * sw.y, b.y),
                         __fmaf_rn(static_cast<float>(acc.z), sx * sw.z, b.z),
                         __fmaf_rn(static_cast<float>(acc.w), sx * sw.w, b.w));
  if (p.residual) {
    const long long at = t * p.ldr + n;
    if (p.in_type == kOutF32) {
      const float4 r = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.residual) + at);
      y.x += r.x, y.y += r.y, y.z += r.z, y.w += r.w;
    } else {
      const uint2 r = *reinterpret_cast<const uint2*>(reinterpret_cast<const unsigned short*>(p.residual) + at);
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
// cluster split K (there are only N / 128 tiles to spread over 148 SMs): each leaves its integer partial in its
// shared memory, and each sums and finishes its share of the tokens over the cluster. Integer sums have no
// order, so the split changes no bit.
//   warp 0: TMA producer into a ring of stages;  warp 1: TMEM and MMA issue;  warps 2-5: accumulator to
//   shared memory;  then all warps: a token row each, four neighbouring channels a lane (VEC: 16-byte rows) or
//   every 32nd channel.
template <int OUT, bool VEC>
__global__ void __launch_bounds__(kI8Threads) gemm_int8_stream_kernel(const __grid_constant__ CUtensorMap tmW,
                                                                      const __grid_constant__ CUtensorMap tmX,
                                                                      const Int8Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[16], empty[16], done;
  __shared__ uint32_t tmem_slot;
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
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    fence_mbar_init();
    // the first weight tiles start at once, behind a quantising kernel even before the tokens are there
    // (p.w_early: nothing that kernel writes is part of the weight)
    if (!p.w_early) pdl_wait();
    for (; issued < min(p.stages, kbs); ++issued) {
      mbar_arrive_expect_tx(&full[issued], stage_bytes);
      tma_load_2d(smem + issued * stage_bytes, &tmW, &full[issued], (kb_first + issued) * kI8BK, n0);
    }
    pdl_wait();
    for (int s = 0; s < issued; ++s)
      tma_load_2d(smem + s * stage_bytes + kI8Rows * kI8BK, &tmX, &full[s], (kb_first + s) * kI8BK, t0);
  }
  __syncwarp();
  if (warp == 1) tmem_alloc(&tmem_slot, cols);
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = tmem_slot;

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
    const int quarter = warp & 3;  // TMEM lanes this warp may read
    if (mbar_wait(&done, 0, p.status, kStatusTimeoutEpilogue)) {
      tc_fence_after();
      const uint32_t t_row = tbase + (static_cast<uint32_t>(quarter * 32) << 16);
      // every MMA of this CTA has read its stages: their memory takes the accumulator, [token][channel]
      int* part = reinterpret_cast<int*>(smem) + quarter * 32 + lane;
#pragma unroll 1
      for (int c0 = 0; c0 < min(p.bt, p.M - t0); c0 += 16) {
        uint32_t v[16];
        tmem_ld16(t_row + c0, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(c0 + i) * kI8Rows] = static_cast<int>(v[i]);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (splits > 1) cluster_sync();

  // this CTA's share of the tokens; a timed-out wait leaves what it finds there (the status word is set)
  const int share = (p.bt + splits - 1) / splits;
  const int c_lo = split * share, c_hi = min(min(p.bt, p.M - t0), c_lo + share);
  constexpr int kWarps = kI8Threads / 32;
  if constexpr (VEC) {
    const int n = n0 + lane * 4;
    if (n < p.N) {  // N is a multiple of 4
      const float4 sw = *reinterpret_cast<const float4*>(p.sw + n);
      float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p.bias)
        b = make_float4(load_as_float(p.bias, n, p.in_type), load_as_float(p.bias, n + 1, p.in_type),
                        load_as_float(p.bias, n + 2, p.in_type), load_as_float(p.bias, n + 3, p.in_type));
#pragma unroll 2
      for (int c = c_lo + warp; c < c_hi; c += kWarps) {
        const uint32_t off = (c * kI8Rows + lane * 4) * 4;
        int4 acc = *reinterpret_cast<const int4*>(smem + off);
        for (int r = 1; r < splits; ++r) {
          const int4 o = ld_cluster_s32x4(map_shared_rank(smem, (split + r) % splits) + off);
          acc.x += o.x, acc.y += o.y, acc.z += o.z, acc.w += o.w;
        }
        finish4<OUT>(p, t0 + c, n, acc, __ldg(p.sx + t0 + c), sw, b);
      }
    }
  } else {
    float sw[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + i * 32 + lane;
      sw[i] = n < p.N ? p.sw[n] : 0.f;
      b[i] = (n < p.N && p.bias) ? load_as_float(p.bias, n, p.in_type) : 0.f;
    }
    for (int c = c_lo + warp; c < c_hi; c += kWarps) {
      const long long t = t0 + c;
      const float sx = __ldg(p.sx + t);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = n0 + i * 32 + lane;
        if (n >= p.N) continue;
        const uint32_t off = (c * kI8Rows + i * 32 + lane) * 4;
        int acc = *reinterpret_cast<const int*>(smem + off);
        for (int r = 1; r < splits; ++r) acc += ld_cluster_s32(map_shared_rank(smem, (split + r) % splits) + off);
        float y = __fmaf_rn(static_cast<float>(acc), sx * sw[i], b[i]);
        if (p.residual) y += load_as_float(p.residual, t * p.ldr + n, p.in_type);
        store_from_float(p.out, t * p.ldo + n, OUT, y);
      }
    }
  }
  __syncthreads();
  if (splits > 1) cluster_sync();  // nobody leaves while its partial may still be read
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
// otherwise, and for residuals that are not aligned, through fp32 staging and coalesced element stores.
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
      const float sx = row_ok ? __ldg(p.sx + row) : 0.f;
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
          f[i] = __fmaf_rn(f[i], sx * s4.x, b4.x);
          f[i + 1] = __fmaf_rn(f[i + 1], sx * s4.y, b4.y);
          f[i + 2] = __fmaf_rn(f[i + 2], sx * s4.z, b4.z);
          f[i + 3] = __fmaf_rn(f[i + 3], sx * s4.w, b4.w);
        }
        const int col0 = n0 + c0;
        if constexpr (TMA_OUT) {
          if (p.residual && row_ok) add_residual32(f, p, row, col0);
          // 16-bit results: two buffers of 32 rows x 64 bytes; fp32: one of 32 x 128
          uint8_t* buf = wbuf + (OUT == kOutF32 ? 0 : (chunk & 1) * (kI8EpiBytes / 2));
          ++chunk;
          if (lane == 0) {  // the store issued from this buffer has read it
            if constexpr (OUT == kOutF32) bulk_wait_read<0>();
            else bulk_wait_read<1>();
          }
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
#pragma unroll 8
            for (int r = 0; r < rows; ++r) {
              float y = *reinterpret_cast<const float*>(wbuf + swz128(r, lane >> 2) + (lane & 3) * 4);
              const long long at = y0 + r;
              if (p.residual) y += load_as_float(p.residual, at * p.ldr + n, p.in_type);
              store_from_float(p.out, at * p.ldo + n, OUT, y);
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

// Map of the output for tiles of 32 columns x 32 rows. False when TMA cannot store it (alignment).
bool make_out_map(CUtensorMap* out, const Int8Params& p) {
  const uint64_t es = p.out_type == kOutF32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(p.out) & 15) || (p.ldo * es) % 16 || p.ldo < p.N) return false;
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

template <typename T, int PRE>
int launch_quantize(const T* x, long long ldx, const T* w, float eps, int8_t* q, float* scale, long long rows, int K,
                    int Kp, cudaStream_t s) {
  const bool vec = K % 8 == 0 && ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  const int chunks = (Kp + 7) / 8;
  if (!vec || chunks > 4 * 1024) {
    if constexpr (PRE == kPreNone) {
      quantize_rows_any_kernel<T><<<static_cast<unsigned>(rows), 256, 0, s>>>(x, ldx, q, scale, K, Kp);
      return static_cast<int>(cudaGetLastError());
    } else {
      return -2;
    }
  }
  // the fewest threads a row that hold it in 4 chunks each (SwiGLU: of both halves), 512 at most
  int tpr = 32;
  while (tpr < 512 && chunks > 4 * tpr) tpr *= 2;
  const int block = std::max(tpr, 128);
  const int nc = (chunks + tpr - 1) / tpr;
  const unsigned grid = static_cast<unsigned>((rows + block / tpr - 1) / (block / tpr));
  auto launch = [&](auto kern) { kern<<<grid, block, 0, s>>>(x, ldx, w, eps, q, scale, rows, K, Kp, tpr); };
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
                                    float* scale, long long rows, int K, cudaStream_t s) {
  using namespace accerl;
  if (rows <= 0) return 0;
  if (K <= 0 || rows > 0x7fffffffll) return -1;
  const int Kp = (K + 15) / 16 * 16;
  int8_t* qp = reinterpret_cast<int8_t*>(q);
  if (half) {
    if (pre != kPreNone) return -3;
    return launch_quantize<__half, kPreNone>(reinterpret_cast<const __half*>(x), ldx, nullptr, eps, qp, scale, rows, K,
                                             Kp, s);
  }
  const auto* xb = reinterpret_cast<const __nv_bfloat16*>(x);
  const auto* wb = reinterpret_cast<const __nv_bfloat16*>(w);
  if (pre == kPreRmsNorm) return launch_quantize<__nv_bfloat16, kPreRmsNorm>(xb, ldx, wb, eps, qp, scale, rows, K, Kp, s);
  if (pre == kPreSwiglu) return launch_quantize<__nv_bfloat16, kPreSwiglu>(xb, ldx, nullptr, eps, qp, scale, rows, K, Kp, s);
  return launch_quantize<__nv_bfloat16, kPreNone>(xb, ldx, nullptr, eps, qp, scale, rows, K, Kp, s);
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
  p.tiles_m = (M + kI8Tile - 1) / kI8Tile;
  p.tiles_n = (N + kI8Tile - 1) / kI8Tile;
  p.group_m = 8;
  if (M > 256) {
    CUtensorMap mx, mw, mo;
    if (!make_int8_map(&mx, qx, Kp, static_cast<uint64_t>(M), 128)) return -7;
    if (!make_int8_map(&mw, qw, Kp, static_cast<uint64_t>(N), 128)) return -8;
    const int rs = in_type == kOutF32 ? 4 : 2;
    const bool res_ok = !residual || ((reinterpret_cast<uintptr_t>(residual) & 15) == 0 && (ldr * rs) % 16 == 0);
    if (static_cast<long long>(p.tiles_m) * p.tiles_n > 0x3fffffff) return -4;
    if (res_ok && make_out_map(&mo, p)) {
      if (out_type == kOutBf16) return launch_pair<kOutBf16, true>(mx, mw, mo, p, stream);
      if (out_type == kOutF16) return launch_pair<kOutF16, true>(mx, mw, mo, p, stream);
      return launch_pair<kOutF32, true>(mx, mw, mo, p, stream);
    }
    mo = mx;
    if (out_type == kOutBf16) return launch_pair<kOutBf16, false>(mx, mw, mo, p, stream);
    if (out_type == kOutF16) return launch_pair<kOutF16, false>(mx, mw, mo, p, stream);
    return launch_pair<kOutF32, false>(mx, mw, mo, p, stream);
  }
  p.bt = 16;
  while (p.bt < M) p.bt *= 2;
  const int kbs = (K + kI8BK - 1) / kI8BK;
  const int tiles = (N + kI8Rows - 1) / kI8Rows;
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= device_sm_count() && splits * 2 <= kbs) splits *= 2;
  const int stage_bytes = (kI8Rows + p.bt) * kI8BK;
  const int budget = tiles * splits > device_sm_count() ? 100 * 1024 : 200 * 1024;
  p.stages = std::max(2, std::min({16, (kbs + splits - 1) / splits, budget / stage_bytes}));
  // the accumulator in the end lies where the stages were
  const int smem_bytes = std::max(p.stages * stage_bytes, p.bt * kI8Rows * 4) + 1024;
  CUtensorMap mw, mx;
  if (!make_int8_map(&mw, qw, Kp, static_cast<uint64_t>(N), kI8Rows)) return -7;
  if (!make_int8_map(&mx, qx, Kp, static_cast<uint64_t>(M), static_cast<uint32_t>(p.bt))) return -8;
  const int es = out_type == kOutF32 ? 4 : 2, rs = in_type == kOutF32 ? 4 : 2;
  const bool vec = N % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0 && (ldo * es) % (4 * es) == 0 &&
                   (reinterpret_cast<uintptr_t>(sw) & 15) == 0 &&
                   (!residual || ((reinterpret_cast<uintptr_t>(residual) & 15) == 0 && (ldr * rs) % (4 * rs) == 0));
  const dim3 grid(tiles, 1, splits);
  if (out_type == kOutBf16) return vec ? launch_stream<kOutBf16, true>(mw, mx, p, grid, smem_bytes, stream) : launch_stream<kOutBf16, false>(mw, mx, p, grid, smem_bytes, stream);
  if (out_type == kOutF16) return vec ? launch_stream<kOutF16, true>(mw, mx, p, grid, smem_bytes, stream) : launch_stream<kOutF16, false>(mw, mx, p, grid, smem_bytes, stream);
  return vec ? launch_stream<kOutF32, true>(mw, mx, p, grid, smem_bytes, stream) : launch_stream<kOutF32, false>(mw, mx, p, grid, smem_bytes, stream);
}
