// Microscaled 4-bit floating point (OCP MX, MXFP4): rows as blocks of 32 values along K, each block one
// scale 2^(s - 127) (a byte s, E8M0) and 32 E2M1 codes (sign, magnitudes 0 0.5 1 1.5 2 3 4 6).
//
//   quantise   s = clamp(floor(log2 max|x|) - 2 + 127, 0, 254), code = x 2^(127 - s) to the nearest code,
//              ties to the even one, above 6 to 6; a block of zeros: s = 0; a block with inf or NaN: s = 255,
//              which stands for NaN
//   product    C[m][n] = sum over blocks b of 2^(sa + sw - 254) sum over the block of a w, then
//              * ra[m] col_scale * rw[n] (cosine scores) and + bias[n]
//
// Layout: codes (rows, KB 16) bytes, the even element in the low half of a byte; scales (rows, KB) bytes; KB =
// ceil(K / 32), values past K are zero. Both contiguous. That is 4.25 bits a value: a 1M x 768 catalog is
// 408 MB instead of 1.5 GB in 16 bits, and the matrix cores multiply it at four times the 16-bit rate
// (v_mfma_scale_f32_16x16x128_f8f6f4: a lane holds one block of a row and that block's scale). Products of
// codes are exact; sums are fp32.
#include "rf_common.h"

#include <algorithm>

namespace rf {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// ---- quantise --------------------------------------------------------------------------------
// neighbours of a quad of lanes: 0xB1 = [1 0 3 2], 0x4E = [2 3 0 1]
template <int CTRL>
__device__ __forceinline__ float quad(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}

template <typename T>
__device__ __forceinline__ void load8(const T* x, int c, int K, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= K) {
    T e[8];
    __builtin_memcpy(e, __builtin_assume_aligned(x + c, 16), sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? to_f32(x[c + i]) : 0.f;
  }
}

// A row is taken by 2^sh lanes, eight values a lane at a time, four lanes a block. HBM bound (read the
// row, write 17 bytes a block).
template <typename T>
__global__ void __launch_bounds__(256) k_mxfp4_quantize(int64_t M, int K, int KB, const T* __restrict__ x, int64_t ldx,
                                                        int sh, bool vec, float eps, uint8_t* __restrict__ codes,
                                                        uint8_t* __restrict__ scales, float* __restrict__ rnorm) {
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = gid >> sh;
  const int L = 1 << sh, sub = (int)(gid & (L - 1));
  if (row >= M) return;  // whole rows of lanes
  const T* xr = x + row * ldx;
  float sq = 0.f;
  for (int c = 8 * sub; c < KB * 32; c += 8 * L) {
    float v[8];
    load8(xr, c, K, vec, v);
    float top = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = fabsf(v[i]);
      top = fmaxf(top, a);
      bad |= !(a < __builtin_inff());
      sq = fmaf(v[i], v[i], sq);
    }
    if (bad) top = __builtin_inff();  // (fmaxf drops a NaN)
    top = fmaxf(top, quad<0xB1>(top));
    top = fmaxf(top, quad<0x4E>(top));
    const int e = (int)(__float_as_uint(top) >> 23);  // biased exponent; 0: zero or subnormal
    const int s = e == 255 ? 255 : max(e - 2, 0);
    const float inv = __uint_as_float((uint32_t)(254 - min(s, 254)) << 23);  // 2^(127 - s), exact
    uint32_t w = 0;
    if (s != 255) {
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0] * inv, v[1] * inv, 1.0f, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2] * inv, v[3] * inv, 1.0f, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4] * inv, v[5] * inv, 1.0f, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6] * inv, v[7] * inv, 1.0f, 3);
    }
    *reinterpret_cast<uint32_t*>(codes + row * KB * 16 + (c >> 1)) = w;
    if ((sub & 3) == 0) scales[row * KB + (c >> 5)] = (uint8_t)s;
  }
  if (rnorm) {
    for (int o = L >> 1; o > 0; o >>= 1) sq += __shfl_xor(sq, o, 64);
    if (sub == 0) rnorm[row] = 1.0f / fmaxf(sqrtf(sq), eps);
  }
}

// ---- back to values --------------------------------------------------------------------------
__device__ __forceinline__ float scale_value(int s) {  // 2^(s - 127); 255: NaN
  return __uint_as_float(s == 255 ? 0x7FC00000u : s == 0 ? 0x00400000u : (uint32_t)s << 23);
}

template <typename T>
__global__ void __launch_bounds__(256) k_mxfp4_dequantize(int64_t M, int K, int KB, const uint8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                          int64_t ldo, int sh, bool vec) {
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = gid >> sh;
  const int L = 1 << sh, sub = (int)(gid & (L - 1));
  if (row >= M) return;
  T* o = out + row * ldo;
  for (int c = 8 * sub; c < K; c += 8 * L) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + row * KB * 16 + (c >> 1));
    const float f = scale_value(scales[row * KB + (c >> 5)]);
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t q = w >> (4 * i);
      // magnitude code m: 0 0.5 | 1 1.5 | 2 3 | 4 6 = (1 + (m & 1) / 2) 2^((m >> 1) - 1), and m / 2 below 2
      const uint32_t m = q & 7;
      const float a = m < 2 ? 0.5f * (float)m : __uint_as_float((126 + (m >> 1)) << 23 | (m & 1) << 22);
      e[i] = from_f32<T>((q & 8 ? -a : a) * f);
    }
    if (vec && c + 8 <= K) {
      __builtin_memcpy(__builtin_assume_aligned(o + c, 16), e, sizeof(e));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < K) o[c + i] = e[i];
    }
  }
}

// ---- product ---------------------------------------------------------------------------------
struct MxArgs {
  int64_t M, N;
  int KB;
  const uint8_t *ac, *as, *wc, *ws;
  const float *bias, *ra, *rw;
  float col_scale;
  void* c;
  int64_t ldc;
  int nTm, nTn, gm;
};

// a and b: fp4 (format 4) in the lower 16 bytes; the scales' byte is picked by an immediate
template <int OA, int OB>
__device__ __forceinline__ f32x4 mfma_mx(u32x4 a, u32x4 b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, OA, (int)sa, OB, (int)sb);
}

// four consecutive columns [n, n + 4) of row m
template <typename T>
__device__ __forceinline__ void store4(const MxArgs& a, int64_t m, int64_t n, f32x4 v, float ra) {
  if (a.ra) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= ra * a.rw[min(n + i, a.N - 1)];
  }
  if (a.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += a.bias[min(n + i, a.N - 1)];
  }
  T* o = (T*)a.c + m * a.ldc + n;
  T e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(v[i]);
  if (n + 4 <= a.N) {
    __builtin_memcpy(__builtin_assume_aligned(o, 4 * sizeof(T)), e, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) o[i] = e[i];
  }
}

// 128 x 128 tiles, four waves of 64 x 64, K in steps of 128 (four blocks a row) through two LDS stages.
// W is the matrix instruction's first operand, so that a lane's four results are neighbours in a row of C.
// Rows of a stage are 64 bytes; their 16-byte slots are permuted by (row / 4) % 4, so that the 16 rows a
// fragment read touches at once fall into different banks.
constexpr int MX_T = 128;
constexpr int MX_STAGE = 2 * MX_T * 64;  // bytes: W rows, then A rows

template <typename T>
__global__ void __launch_bounds__(256, 4) k_mxfp4_gemm(MxArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t code[2][MX_STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t scl[2][2 * MX_T * 4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int r = lane & 15, g = lane >> 4;
  // columns of tiles in groups of gm row tiles: the group's A rows stay in an XCD's L2 while W streams by
  const int v = xcd_remap(blockIdx.x, gridDim.x);
  const int grp = v / (a.gm * a.nTn), in = v - grp * a.gm * a.nTn;
  const int gm = min(a.gm, a.nTm - grp * a.gm);
  const int64_t m0 = (int64_t)(grp * a.gm + in % gm) * MX_T, n0 = (int64_t)(in / gm) * MX_T;
  const int KB = a.KB, nk = (KB + 3) >> 2;
  // staging: a wave instruction fills 16 rows; lane l writes slot l % 4 of row l / 4
  const int srow = lane >> 2, sch = (lane & 3) ^ ((srow >> 2) & 3);
  const uint8_t* src[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (wave * 4 + i) * 16 + srow;  // 0..127: W rows, 128..255: A rows
    src[i] = row < MX_T ? a.wc + min(n0 + row, a.N - 1) * KB * 16 : a.ac + min(m0 + row - MX_T, a.M - 1) * KB * 16;
  }
  const uint8_t* ssrc = t < MX_T ? a.ws + min(n0 + t, a.N - 1) * KB : a.as + min(m0 + t - MX_T, a.M - 1) * KB;
  const bool sdw = (KB & 3) == 0 && ((reinterpret_cast<uintptr_t>(a.ws) | reinterpret_cast<uintptr_t>(a.as)) & 3) == 0;
  auto stage = [&](int kt, int b) {
    const int ch = min(4 * kt + sch, KB - 1);  // past the last block: a block of the row, multiplied by 0 below
#pragma unroll
    for (int i = 0; i < 4; ++i) glds16(src[i] + ch * 16, &code[b][(wave * 4 + i) * 1024]);
  };
  auto load_scales = [&](int kt) -> uint32_t {
    if (sdw) return *reinterpret_cast<const uint32_t*>(ssrc + 4 * kt);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (uint32_t)(4 * kt + i < KB ? ssrc[4 * kt + i] : 127) << (8 * i);
    return w;
  };
  // scales in LDS as the fragments read them: for 64 rows (four 16-row tiles j), byte j of word [block][row % 16]
  auto put_scales = [&](int b, uint32_t w) {
    uint8_t* d = &scl[b][(t >> 6) * 256 + (t & 15) * 4 + ((t >> 4) & 3)];
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i * 64] = (uint8_t)(w >> (8 * i));
  };
  const int wn = (wave & 1) * 64, wm = (wave >> 1) * 64;
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  stage(0, 0);
  put_scales(0, load_scales(0));
  for (int kt = 0; kt < nk; ++kt) {
    const int b = kt & 1;
    wait_vmcnt0();
    __syncthreads();  // stage kt is in LDS; everyone is done with stage kt - 1
    u32x4 fw[4], fa[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rw = wn + i * 16 + r, rm = MX_T + wm + i * 16 + r, slot = (g ^ ((r >> 2) & 3)) * 16;
      fw[i] = *reinterpret_cast<const u32x4*>(&code[b][rw * 64 + slot]);
      fa[i] = *reinterpret_cast<const u32x4*>(&code[b][rm * 64 + slot]);
    }
    const uint32_t sw = *reinterpret_cast<const uint32_t*>(&scl[b][(wn >> 6) * 256 + (g * 16 + r) * 4]);
    const uint32_t sa = *reinterpret_cast<const uint32_t*>(&scl[b][(2 + (wm >> 6)) * 256 + (g * 16 + r) * 4]);
    uint32_t next = 0;
    if (kt + 1 < nk) {
      stage(kt + 1, b ^ 1);
      next = load_scales(kt + 1);
    }
    if (4 * kt + g >= KB) {
#pragma unroll
      for (int i = 0; i < 4; ++i) fa[i] = u32x4{0, 0, 0, 0};
    }
#define MX_COL(i, j) acc[i][j] = mfma_mx<i, j>(fw[i], fa[j], acc[i][j], sw, sa)
#define MX_ROW(i) MX_COL(i, 0); MX_COL(i, 1); MX_COL(i, 2); MX_COL(i, 3)
    MX_ROW(0); MX_ROW(1); MX_ROW(2); MX_ROW(3);
#undef MX_ROW
#undef MX_COL
    if (kt + 1 < nk) put_scales(b ^ 1, next);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t m = m0 + wm + j * 16 + r;
    if (m < a.M) {
      const float ra = a.ra ? a.ra[m] * a.col_scale : 1.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t n = n0 + wn + i * 16 + 4 * g;
        if (n < a.N) store4<T>(a, m, n, acc[i][j], ra);
      }
    }
  }
}

// Up to 16 MT rows of A: W is read once from memory straight into the fragments, a wave per 16 of its rows,
// U steps of K at a time in flight; the A rows come from the caches. Bound by the read of W.
template <typename T, int MT>
__global__ void __launch_bounds__(256) k_mxfp4_skinny(MxArgs a) {
  constexpr int U = MT == 1 ? 6 : MT == 2 ? 4 : 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int64_t n0 = ((int64_t)blockIdx.x * 4 + wave) * 16;
  if (n0 >= a.N) return;
  const int KB = a.KB, nk = (KB + 3) >> 2;
  const int64_t wr = min(n0 + r, a.N - 1);
  const uint8_t *wc = a.wc + wr * KB * 16, *ws = a.ws + wr * KB;
  f32x4 acc[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < nk; k0 += U) {
    u32x4 fw[U];
    uint32_t sw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = min(4 * (k0 + u) + g, KB - 1);
      fw[u] = *reinterpret_cast<const u32x4*>(wc + b * 16);
      sw[u] = ws[b];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = 4 * (k0 + u) + g;
      const bool in = b < KB;
      const uint32_t sb = in ? sw[u] : 127;
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int64_t m = min((int64_t)j * 16 + r, a.M - 1);
        u32x4 fa = *reinterpret_cast<const u32x4*>(a.ac + m * KB * 16 + min(b, KB - 1) * 16);
        uint32_t sa = a.as[m * KB + min(b, KB - 1)];
        if (!in) {
          fa = u32x4{0, 0, 0, 0};
          sa = 127;
        }
        acc[j] = mfma_mx<0, 0>(fw[u], fa, acc[j], sb, sa);
      }
    }
  }
  const int64_t n = n0 + 4 * g;
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int64_t m = (int64_t)j * 16 + r;
    if (m < a.M && n < a.N) store4<T>(a, m, n, acc[j], a.ra ? a.ra[m] * a.col_scale : 1.f);
  }
}

// ---- host --------------------------------------------------------------------------------------
static int lane_shift(int K) {  // lanes a row: enough for its eights, at least a block's four
  int sh = 2;
  while (sh < 6 && (8 << sh) < K) ++sh;
  return sh;
}

template <typename T>
static void launch_gemm(const MxArgs& a, hipStream_t st) {
  if (a.M <= 64) {
    const unsigned grid = (unsigned)((a.N + 63) / 64);
    if (a.M <= 16) k_mxfp4_skinny<T, 1><<<grid, 256, 0, st>>>(a);
    else if (a.M <= 32) k_mxfp4_skinny<T, 2><<<grid, 256, 0, st>>>(a);
    else k_mxfp4_skinny<T, 4><<<grid, 256, 0, st>>>(a);
  } else {
    k_mxfp4_gemm<T><<<(unsigned)((int64_t)a.nTm * a.nTn), 256, 0, st>>>(a);
  }
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace rf

using namespace rf;

extern "C" int rf_mxfp4_quantize(int dtype, int M, int K, const void* x, int64_t ldx, float eps, uint8_t* codes,
                                 uint8_t* scales, float* rnorm, rf_stream_t stream) {
  RF_REQUIRE(dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16, "rf_mxfp4_quantize: bad dtype %d", dtype);
  RF_REQUIRE(M >= 0 && K > 0 && K <= (1 << 30) && ldx >= K, "rf_mxfp4_quantize: bad shape M=%d K=%d", M, K);
  if (M == 0) return RF_OK;
  RF_REQUIRE(x && codes && scales, "rf_mxfp4_quantize: null pointer");
  const int es = dtype == RF_F32 ? 4 : 2;
  RF_REQUIRE((reinterpret_cast<uintptr_t>(x) & (es - 1)) == 0 && aligned16(codes),
             "rf_mxfp4_quantize: misaligned rows or codes");
  const int KB = (K + 31) / 32, sh = lane_shift(K);
  const bool vec = aligned16(x) && ldx * es % 16 == 0;
  const int64_t blocks = (((int64_t)M << sh) + 255) / 256;
  RF_REQUIRE(blocks < 0x7FFFFFFF, "rf_mxfp4_quantize: too many rows");
  hipStream_t st = as_stream(stream);
#define MXQ(T)                                                                                                      \
  k_mxfp4_quantize<T><<<(unsigned)blocks, 256, 0, st>>>(M, K, KB, (const T*)x, ldx, sh, vec, eps, codes, scales, rnorm)
  if (dtype == RF_F32) MXQ(float);
  else if (dtype == RF_BF16) MXQ(bf16);
  else MXQ(f16);
#undef MXQ
  RF_LAUNCH_CHECK("rf_mxfp4_quantize");
}

extern "C" int rf_mxfp4_dequantize(int dtype, int M, int K, const uint8_t* codes, const uint8_t* scales, void* out,
                                   int64_t ldo, rf_stream_t stream) {
  RF_REQUIRE(dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16, "rf_mxfp4_dequantize: bad dtype %d", dtype);
  RF_REQUIRE(M >= 0 && K > 0 && K <= (1 << 30) && ldo >= K, "rf_mxfp4_dequantize: bad shape M=%d K=%d", M, K);
  if (M == 0) return RF_OK;
  RF_REQUIRE(out && codes && scales, "rf_mxfp4_dequantize: null pointer");
  const int es = dtype == RF_F32 ? 4 : 2;
  RF_REQUIRE((reinterpret_cast<uintptr_t>(out) & (es - 1)) == 0 && aligned16(codes),
             "rf_mxfp4_dequantize: misaligned rows or codes");
  const int KB = (K + 31) / 32, sh = lane_shift(K);
  const bool vec = aligned16(out) && ldo * es % 16 == 0;
  const int64_t blocks = (((int64_t)M << sh) + 255) / 256;
  RF_REQUIRE(blocks < 0x7FFFFFFF, "rf_mxfp4_dequantize: too many rows");
  hipStream_t st = as_stream(stream);
#define MXD(T) k_mxfp4_dequantize<T><<<(unsigned)blocks, 256, 0, st>>>(M, K, KB, codes, scales, (T*)out, ldo, sh, vec)
  if (dtype == RF_F32) MXD(float);
  else if (dtype == RF_BF16) MXD(bf16);
  else MXD(f16);
#undef MXD
  RF_LAUNCH_CHECK("rf_mxfp4_dequantize");
}

extern "C" int rf_mxfp4_gemm(int out_dtype, int M, int N, int K, const uint8_t* a_codes, const uint8_t* a_scales,
                             const uint8_t* w_codes, const uint8_t* w_scales, const float* bias, const float* ra,
                             const float* rw, float col_scale, void* C, int64_t ldc, rf_stream_t stream) {
  RF_REQUIRE(out_dtype == RF_F32 || out_dtype == RF_BF16 || out_dtype == RF_F16, "rf_mxfp4_gemm: bad dtype %d",
             out_dtype);
  RF_REQUIRE(M >= 0 && N >= 0 && K > 0 && K <= (1 << 30) && ldc >= N, "rf_mxfp4_gemm: bad shape M=%d N=%d K=%d", M, N,
             K);
  if (M == 0 || N == 0) return RF_OK;
  RF_REQUIRE(a_codes && a_scales && w_codes && w_scales && C, "rf_mxfp4_gemm: null pointer");
  RF_REQUIRE(!ra == !rw, "rf_mxfp4_gemm: ra and rw go together");
  const int es = out_dtype == RF_F32 ? 4 : 2;
  RF_REQUIRE(aligned16(a_codes) && aligned16(w_codes), "rf_mxfp4_gemm: codes must be 16-byte aligned");
  RF_REQUIRE((reinterpret_cast<uintptr_t>(C) & (4 * es - 1)) == 0 && ldc % 4 == 0,
             "rf_mxfp4_gemm: the result's rows must be aligned to four elements");
  MxArgs a{};
  a.M = M; a.N = N; a.KB = (K + 31) / 32;
  a.ac = a_codes; a.as = a_scales; a.wc = w_codes; a.ws = w_scales;
  a.bias = bias; a.ra = ra; a.rw = rw; a.col_scale = col_scale; a.c = C; a.ldc = ldc;
  a.nTm = (M + MX_T - 1) / MX_T;
  a.nTn = (N + MX_T - 1) / MX_T;
  // row tiles whose codes fill half of an XCD's 4 MB of L2
  a.gm = (int)std::max<int64_t>(1, std::min<int64_t>(a.nTm, (2 << 20) / ((int64_t)MX_T * a.KB * 16)));
  RF_REQUIRE((int64_t)a.nTm * a.nTn < 0x7FFFFFFF, "rf_mxfp4_gemm: too many tiles");
  hipStream_t st = as_stream(stream);
  if (out_dtype == RF_F32) launch_gemm<float>(a, st);
  else if (out_dtype == RF_BF16) launch_gemm<bf16>(a, st);
  else launch_gemm<f16>(a, st);
  RF_LAUNCH_CHECK("rf_mxfp4_gemm");
}
