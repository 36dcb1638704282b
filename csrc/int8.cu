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
// from every such border. p is within 2^-23 of it; the remainder 127 x - p a is exact, and the corrected
// quotient is the exact one where that is representable, which every border is. The last addition rounds to
// the nearest whole number, ties to even; the low byte of its pattern is the two's complement.
ACCERL_DEVINL uint32_t quant_bits(float x, const RowQuant& s) {
  const float n = __fmul_rn(x, s.m127);
  const float p = __fmul_rn(n, s.inv);
  const float e = __fmaf_rn(-p, s.a, n);
  return __float_as_uint(__fadd_rn(__fmaf_rn(e, s.inv, p), 0x1.8p23f));
}
ACCERL_DEVINL uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Reduction over the `tpr` threads of a row (a power of two, 32..blockDim); `red` has one slot per warp.
template <typename V, typename F>
ACCERL_DEVINL V row_reduce(V v, int tpr, V* red, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    const int w0 = (threadIdx.x / tpr) * (tpr >> 5);
    v = red[w0];
    for (int w = 1; w < (tpr >> 5); ++w) v = f(v, red[w0 + w]);
    __syncthreads();
  }
  return v;
}

ACCERL_DEVINL uint32_t amax_pair(uint32_t m) { return max(m & 0xffffu, m >> 16); }

// One row per `tpr` threads, 8 elements a thread and chunk, the row held in registers between the maximum
// and the rounding so that it is read once. PRE turns the input row into the row to round: RMSNorm
// (x [rows, K], weight w) or SwiGLU (x = gate | up, [rows, 2K]), with the roundings of the framework's
// own kernels (both give rows in T).
template <typename T, int PRE, int NC>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const T* __restrict__ x, long long ldx,
                                                             const T* __restrict__ w, float eps,
                                                             int8_t* __restrict__ q, float* __restrict__ scale,
                                                             long long rows, int K, int Kp, int tpr) {
  __shared__ uint32_t red_u[32];
  __shared__ float red_f[32];
  const int in_row = threadIdx.x % tpr;
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x / tpr) + threadIdx.x / tpr;
  const bool live = row < rows;
  const T* xr = x + (live ? row : 0) * ldx;
  uint4 v[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = (j * tpr + in_row) * 8;
    v[j] = make_uint4(0, 0, 0, 0);
    if (live && c < K) {
      v[j] = *reinterpret_cast<const uint4*>(xr + c);
      if constexpr (PRE == kPreSwiglu) {
        const uint4 u = *reinterpret_cast<const uint4*>(xr + K + c);
        uint32_t* g = reinterpret_cast<uint32_t*>(&v[j]);
        const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 fg = unpack_bf16x2(g[i]), fu = unpack_bf16x2(uw[i]);
          g[i] = pack_bf16x2(swiglu_h(fg.x, fu.x), swiglu_h(fg.y, fu.y));
        }
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
constexpr int kI8MaxTokens = 256;  // tokens per tile
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
  int bt;      // tokens per tile
  int stages;
  int* status;
};

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

// One tile of 128 output channels x bt tokens per CTA: the weight rows are the MMA's 128 rows, so a decode
// batch of few tokens wastes no tensor rows and streams the weight once.
//   warp 0: TMA producer into a ring of stages;  warp 1: TMEM and MMA issue;  warps 2-5: epilogue (one
//   TMEM lane = one output channel per thread; the 32 lanes of a warp store 32 neighbouring channels).
__global__ void __launch_bounds__(kI8Threads) gemm_int8_kernel(const __grid_constant__ CUtensorMap tmW,
                                                               const __grid_constant__ CUtensorMap tmX,
                                                               const Int8Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[16], empty[16], done;
  __shared__ uint32_t tmem_slot;
  __shared__ float sx_s[kI8MaxTokens];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * kI8Rows, t0 = blockIdx.y * p.bt;
  const int kbs = (p.K + kI8BK - 1) / kI8BK;
  const uint32_t stage_bytes = (kI8Rows + p.bt) * kI8BK;
  uint32_t cols = 32;
  while (cols < static_cast<uint32_t>(p.bt)) cols <<= 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmW);
    prefetch_tmap(&tmX);
  }
  if (warp == 1) tmem_alloc(&tmem_slot, cols);
  if (warp >= 2)
    for (int i = threadIdx.x - 64; i < p.bt; i += 128) sx_s[i] = t0 + i < p.M ? p.sx[t0 + i] : 0.f;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int issued = 0;
      for (int kb = 0; kb < kbs; ++kb) {
        const int s = kb % p.stages;
        if (!mbar_wait(&empty[s], ((kb / p.stages) & 1) ^ 1u, p.status, kStatusTimeoutProducer)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[s], stage_bytes);
        tma_load_2d(smem + s * stage_bytes, &tmW, &full[s], kb * kI8BK, n0);
        tma_load_2d(smem + s * stage_bytes + kI8Rows * kI8BK, &tmX, &full[s], kb * kI8BK, t0);
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
      bool ok = true;
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
    const int n = n0 + quarter * 32 + lane;
    if (mbar_wait(&done, 0, p.status, kStatusTimeoutEpilogue)) {
      tc_fence_after();
      const bool n_ok = n < p.N;
      const float sw = n_ok ? p.sw[n] : 0.f;
      const float b = (n_ok && p.bias) ? load_as_float(p.bias, n, p.in_type) : 0.f;
#pragma unroll 1
      for (int c0 = 0; c0 < p.bt && t0 + c0 < p.M; c0 += 16) {
        uint32_t v[16];
        tmem_ld16(tbase + (static_cast<uint32_t>(quarter * 32) << 16) + c0, v);
        tmem_wait_ld();
        if (n_ok) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const long long t = t0 + c0 + i;
            if (t < p.M) {
              float y = static_cast<float>(static_cast<int>(v[i])) * (sx_s[c0 + i] * sw) + b;
              if (p.residual) y += load_as_float(p.residual, t * p.ldr + n, p.in_type);
              store_from_float(p.out, t * p.ldo + n, p.out_type, y);
            }
          }
        }
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, cols);
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
  int tpr = 32;
  while (tpr < 1024 && chunks > 4 * tpr) tpr *= 2;
  const int block = std::max(tpr, 128);
  const int nc = (chunks + tpr - 1) / tpr;
  const unsigned grid = static_cast<unsigned>((rows + block / tpr - 1) / (block / tpr));
  if (nc <= 1) quantize_rows_kernel<T, PRE, 1><<<grid, block, 0, s>>>(x, ldx, w, eps, q, scale, rows, K, Kp, tpr);
  else if (nc <= 2) quantize_rows_kernel<T, PRE, 2><<<grid, block, 0, s>>>(x, ldx, w, eps, q, scale, rows, K, Kp, tpr);
  else quantize_rows_kernel<T, PRE, 4><<<grid, block, 0, s>>>(x, ldx, w, eps, q, scale, rows, K, Kp, tpr);
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
// (types: 0 bf16, 1 fp16, 2 fp32). qx [M, Kp] and qw [N, Kp], Kp = K rounded up to 16.
extern "C" int accerl_gemm_int8(const void* qx, const float* sx, const void* qw, const float* sw, int M, int N, int K,
                                const void* bias, const void* residual, long long ldr, int in_type, void* out,
                                long long ldo, int out_type, int* status, cudaStream_t stream) {
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
  p.bt = 16;
  while (p.bt < M && p.bt < kI8MaxTokens) p.bt *= 2;
  const int kbs = (K + kI8BK - 1) / kI8BK;
  const int stage_bytes = (kI8Rows + p.bt) * kI8BK;
  p.stages = std::max(2, std::min({16, kbs, 200 * 1024 / stage_bytes}));
  const int smem_bytes = p.stages * stage_bytes + 1024;
  CUtensorMap mw, mx;
  if (!make_int8_map(&mw, qw, Kp, static_cast<uint64_t>(N), kI8Rows)) return -7;
  if (!make_int8_map(&mx, qx, Kp, static_cast<uint64_t>(M), static_cast<uint32_t>(p.bt))) return -8;
  cudaError_t e = smem_attr_once<gemm_int8_kernel>(16 * 1024 + 200 * 1024);
  if (e != cudaSuccess) return static_cast<int>(e);
  const long long tiles_t = (static_cast<long long>(M) + p.bt - 1) / p.bt;
  if (tiles_t > 65535) return -4;
  const dim3 grid((N + kI8Rows - 1) / kI8Rows, static_cast<unsigned>(tiles_t));
  gemm_int8_kernel<<<grid, kI8Threads, smem_bytes, stream>>>(mw, mx, p);
  return static_cast<int>(cudaGetLastError());
}
