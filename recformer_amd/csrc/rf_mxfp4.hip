// Microscaled 4-bit floating point (OCP MX, MXFP4): rows as blocks of 32 values along K, each block one
// scale 2^(s - 127) (a byte s, E8M0) and 32 E2M1 codes (sign, magnitudes 0 0.5 1 1.5 2 3 4 6).
//
//   quantise   s = clamp(floor(log2 max|x|) - 2 + 127, 0, 254), code = x 2^(127 - s) to the nearest code,
//              ties to the even one, above 6 to 6; a block of zeros: s = 0; a block with inf or NaN: s = 255,
//              which stands for NaN
//   product    C[m][n] = sum over blocks b of 2^(sa + sw - 254) sum over the block of a w, then
//              * ra[m] col_scale * rw[n] (cosine scores; ra = rw = 1 without them) and + bias[n]
//
// Layout: codes (rows, KB 16) bytes, the even element in the low half of a byte; scales (rows, KB) bytes; KB =
// ceil(K / 32), values past K are zero. Both contiguous. That is 4.25 bits a value: a 1M x 768 catalog is
// 408 MB instead of 1.5 GB in 16 bits, and the matrix cores multiply it at four times the 16-bit rate
// (v_mfma_scale_f32_16x16x128_f8f6f4: a lane holds one block of a row and that block's scale). Products of
// codes are exact; sums are fp32.
#include "rf_common.h"

#include <algorithm>
#include <type_traits>

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
__device__ __forceinline__ void load8(const T* x, int c, int K, float (&v)[8]) {
  if (c + 8 <= K) {
    T e[8];
    // 16 bytes at any alignment (element by element 100000 x 770 bf16 took 90 us instead of 39)
    __builtin_memcpy(e, x + c, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? to_f32(x[c + i]) : 0.f;
  }
}

// A row is taken by 2^sh lanes, eight values a lane at a time, four lanes a block. HBM bound (read the
// row, write 17 bytes a block): 1M x 768 bf16 361 us, 5.4 TB/s, with the norms 426.
template <typename T>
__global__ void __launch_bounds__(256) k_mxfp4_quantize(int64_t M, int K, int KB, const T* __restrict__ x, int64_t ldx,
                                                        int sh, float eps, uint8_t* __restrict__ codes,
                                                        uint8_t* __restrict__ scales, float* __restrict__ rnorm) {
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = gid >> sh;
  const int L = 1 << sh, sub = (int)(gid & (L - 1));
  if (row >= M) return;  // whole rows of lanes
  const T* xr = x + row * ldx;
  float sq = 0.f;
  for (int c = 8 * sub; c < KB * 32; c += 8 * L) {
    float v[8];
    load8(xr, c, K, v);
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

// Eights of values, flat over the rows (G = ceil(K / 8) a row), two a thread 64 apart so that a wave's loads and
// stores are contiguous. HBM bound; the stores are non-temporal (1M x 768 to bf16: 307 us, 6.3 TB/s; 538 us
// through the caches). Rows of other alignments take unaligned stores (100000 x 770 bf16: 32 us; element by element
// 100).
template <typename T>
__global__ void __launch_bounds__(256) k_mxfp4_dequantize(int64_t total, int G, int K, int KB,
                                                          const uint8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                          int64_t ldo, bool vec) {
  const int64_t first = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 128 + (threadIdx.x & 63);
  int64_t row[2];
  int c[2];
  uint32_t w[2];
  int sc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t at = min(first + 64 * i, total - 1);
    row[i] = total <= 0xFFFFFFFFll ? (int64_t)((uint32_t)at / (uint32_t)G) : at / G;
    c[i] = (int)(at - row[i] * G) * 8;
    w[i] = *reinterpret_cast<const uint32_t*>(codes + row[i] * KB * 16 + (c[i] >> 1));
    sc[i] = scales[row[i] * KB + (c[i] >> 5)];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (first + 64 * i >= total) break;
    const float f = scale_value(sc[i]);
    typedef float v2 __attribute__((ext_vector_type(2)));
    const v2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 0),
                     __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 1),
                     __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 2),
                     __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.0f, 3)};
    T e[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) e[x] = from_f32<T>(p[x >> 1][x & 1] * f);
    T* o = out + row[i] * ldo + c[i];
    if (!vec && c[i] + 8 <= K) {
      __builtin_memcpy(o, e, sizeof(e));
    } else if (vec && c[i] + 8 <= K) {
      u32x4 q[sizeof(e) / 16];
      __builtin_memcpy(q, e, sizeof(e));
#pragma unroll
      for (int x = 0; x < (int)(sizeof(e) / 16); ++x) __builtin_nontemporal_store(q[x], reinterpret_cast<u32x4*>(o) + x);
    } else {
#pragma unroll
      for (int x = 0; x < 8; ++x)
        if (c[i] + x < K) o[x] = e[x];
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
  int nTm, nTn, gm, gn;
  bool vec;  // rows of C are 16-byte aligned
};

// a and b: fp4 (format 4) in the lower 16 bytes, the scales in the lowest byte
__device__ __forceinline__ f32x4 mfma_mx(u32x4 a, u32x4 b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

// what the epilogue takes for four consecutive columns [n, n + 4)
struct Cols {
  f32x4 rw, bias;
};
template <bool EDGE>
__device__ __forceinline__ f32x4 load_cols(const float* __restrict__ p, int64_t n, int64_t N, float none) {
  if (!p) return f32x4{none, none, none, none};
  if (!EDGE || n + 4 <= N) return *reinterpret_cast<const f32x4*>(p + n);
  f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = p[min(n + i, N - 1)];
  return v;
}
__device__ __forceinline__ Cols cols_of(const MxArgs& a, int64_t n) {
  return {load_cols<true>(a.rw, n, a.N, 1.f), load_cols<true>(a.bias, n, a.N, 0.f)};
}

// four consecutive columns of row m: (v * ra * rw) + bias, rounded once; ra: the row's factor times col_scale
template <typename T>
__device__ __forceinline__ void store4(const MxArgs& a, int64_t m, int64_t n, f32x4 v, float ra, const Cols& c) {
  T* o = (T*)a.c + m * a.ldc + n;
  T e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(fmaf(v[i] * ra, c.rw[i], c.bias[i]));
  if (n + 4 <= a.N) {
    __builtin_memcpy(__builtin_assume_aligned(o, 4 * sizeof(T)), e, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) o[i] = e[i];
  }
}

__device__ __forceinline__ void put_one(float v, __amdgpu_buffer_rsrc_t rc, int o) {
  __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), rc, o, 0, 0);
}
template <typename T>
__device__ __forceinline__ void put_one(T v, __amdgpu_buffer_rsrc_t rc, int o) {
  __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v), rc, o, 0, 0);
}

// up to 64 floats from p[at] on; past p[n - 1] reads as 0
__device__ __forceinline__ __amdgpu_buffer_rsrc_t part_of(const float* p, int64_t at, int64_t n) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)(p + at), (short)0, (int)max(min(n - at, (int64_t)64), (int64_t)0) * 4,
                                           0x00020000);
}

// row and column factors of a wave's 64 x 64 results, loaded before they are needed
template <typename T>
struct MxVec {
  static constexpr int NV = 16 / sizeof(T);  // neighbours a lane holds: 16 bytes
  static constexpr int NQ = 16 / NV;         // such pieces, 64 bytes apart: piece q holds columns q 4 NV + NV g
  float ra[4];
  f32x4 rw[4], bias[4];  // [q (NV / 4) + h]
  __device__ __forceinline__ void load(const MxArgs& a, int64_t mw, int64_t nw, int r, int g) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ra[i] = 1.f;
      rw[i] = f32x4{1.f, 1.f, 1.f, 1.f};
      bias[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (a.ra) {
      const __amdgpu_buffer_rsrc_t rr = part_of(a.ra, mw, a.M), rc = part_of(a.rw, nw, a.N);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ra[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rr, r * 4 + i * 64, 0, 0));
        rw[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rc, col(g, i) * 4, 0, 0));
      }
    }
    if (a.bias) {
      const __amdgpu_buffer_rsrc_t rc = part_of(a.bias, nw, a.N);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        bias[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rc, col(g, i) * 4, 0, 0));
    }
  }
  static __device__ __forceinline__ int col(int g, int i) {
    return (i / (NV / 4)) * 4 * NV + NV * g + 4 * (i % (NV / 4));
  }
};

// A wave's 64 x 64 results to rows mw.., columns nw..: acc[i][j] holds columns MxMap::wrow(i, 4 g ..) of row
// j 16 + r. A lane holds 16 bytes of a row at a time, and the same 64 bytes further on: lanes of rows r and r + 1
// (r even) trade, so that the even lane holds the first piece of both rows and the odd lane the second, and a
// store writes whole 128-byte lines (non-temporal 64-byte halves took 1625 instead of 1229 us at 4096 x 125000 fp32 with
// rows off the lines; with rows on lines it takes 515).
// EDGE: element by element, those outside of C at an offset that the buffer store drops.
template <typename T, bool EDGE>
__device__ __forceinline__ void mx_epilogue(const MxArgs& a, int64_t mw, int64_t nw, int r, int g,
                                            const f32x4 (&acc)[4][4], const MxVec<T>& vec) {
  constexpr int NV = MxVec<T>::NV, NQ = MxVec<T>::NQ;
  const bool odd = r & 1;
  const int row = (int)a.ldc * (int)sizeof(T);
  const int at = (r & ~1) * row + (NV * g + (odd ? 4 * NV : 0)) * (int)sizeof(T);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc(
        (T*)a.c + (mw + j * 16) * a.ldc + nw, (short)0, 0x7FFFFFFF, 0x00020000);
    const float ra = vec.ra[j] * a.col_scale;
#pragma unroll
    for (int q = 0; q < NQ; q += 2) {
      u32x4 w[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        T e[NV];
#pragma unroll
        for (int x = 0; x < NV; ++x) {
          const int i = (q + p) * (NV / 4) + x / 4;
          e[x] = from_f32<T>(fmaf(acc[i][j][x & 3] * ra, vec.rw[i][x & 3], vec.bias[i][x & 3]));
        }
        __builtin_memcpy(&w[p], e, 16);
      }
      u32x4 even_row, odd_row;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t n0 = (uint32_t)__builtin_amdgcn_mov_dpp((int)w[0][x], 0xB1, 0xF, 0xF, true);
        const uint32_t n1 = (uint32_t)__builtin_amdgcn_mov_dpp((int)w[1][x], 0xB1, 0xF, 0xF, true);
        even_row[x] = odd ? n1 : w[0][x];
        odd_row[x] = odd ? w[1][x] : n0;
      }
      // non-temporal: the tables stay in L2 (512 x 100000 x 768 fp32: 48 us, 83 without; what a reader that finds the
      // result in no cache loses is less or about as much: with the top 10 of each row behind it 129 and 122, 4096 x
      // 125000 905 and 1032)
      if (!EDGE) {
        __builtin_amdgcn_raw_buffer_store_b128(even_row, rc, at + q * 64, 0, 2);
        __builtin_amdgcn_raw_buffer_store_b128(odd_row, rc, at + row + q * 64, 0, 2);
      } else {
        const int64_t m = mw + j * 16 + (r & ~1), n = nw + NV * g + (q + (odd ? 1 : 0)) * (4 * NV);
        T e0[NV], e1[NV];
        __builtin_memcpy(e0, &even_row, 16);
        __builtin_memcpy(e1, &odd_row, 16);
#pragma unroll
        for (int x = 0; x < NV; ++x) {
          const int o = at + q * 64 + x * (int)sizeof(T);
          put_one(e0[x], rc, m < a.M && n + x < a.N ? o : -4);
          put_one(e1[x], rc, m + 1 < a.M && n + x < a.N ? o + row : -4);
        }
      }
    }
  }
}

// 128 x 128 tiles, four waves of 64 x 64. K goes in steps of 256 (eight blocks, a 128-byte line of a row)
// through two LDS stages filled by LDS-DMA: while one is multiplied, the next is on its way, across the end
// of a tile too (a workgroup takes tile after tile, so the next tile's first stage loads during the
// epilogue); two workgroups a CU. W is the matrix instruction's first operand, so that a lane's results are
// neighbours in a row of C; with 16-bit results the W rows of a pair of instructions are interleaved by fours,
// so that a lane holds eight neighbours.
// For short K the stores bound it (4096 x 125000 x 768 fp32: 416 us, 4.9 TB/s of results; 4915 x 50265 x 768 bf16 167 us,
// where stores alone take 108); for long K the fragments' and the LDS-DMA's way through LDS beside the matrix
// instructions (8192^3: 376 us, 2.9 PFLOP/s). Loads two steps ahead, with a second barrier a step, took 5% longer.
// Rows of a stage are 128 bytes; their 16-byte slots are permuted by three bits of the row, so that eight
// neighbouring lanes of a fragment read cover all banks.
constexpr int MX_T = 128;
constexpr int MX_CODES = 2 * MX_T * 128;   // bytes of a stage: W rows, then A rows
constexpr int MX_STAGE = MX_CODES + 2 * MX_T * 8;  // their scales: [word of four][64 rows: x 4 + i]
constexpr int MX_WGS = 2 * 256;            // workgroups that fit the card

template <typename T>
struct MxMap {
  static constexpr bool H = sizeof(T) == 2;
  // row of the wave's 64 that instruction i's row x stands for, and the permutation of a row's slots
  static __device__ __forceinline__ int wrow(int i, int x) {
    return H ? (i >> 1) * 32 + (x >> 2) * 8 + (i & 1) * 4 + (x & 3) : i * 16 + x;
  }
  static __device__ __forceinline__ int wkey(int row) { return H ? (row & 3) | ((row >> 3) & 1) << 2 : row & 7; }
  static __device__ __forceinline__ int akey(int row) { return row & 7; }
};

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// blocks of gm x gn tiles, columns first within: the block's A and W rows stay in an XCD's L2, and
// neighbouring pieces of C's rows are written at about the same time
__device__ __forceinline__ void tile_of(const MxArgs& a, int v, int64_t& m0, int64_t& n0) {
  v = xcd_remap(v, a.nTm * a.nTn);
  const int band = v / (a.gm * a.nTn), inb = v - band * a.gm * a.nTn;
  const int gm = min(a.gm, a.nTm - band * a.gm);
  const int cg = inb / (gm * a.gn), inc = inb - cg * gm * a.gn;
  const int gn = min(a.gn, a.nTn - cg * a.gn);
  m0 = (int64_t)(band * a.gm + inc / gn) * MX_T;
  n0 = (int64_t)(cg * a.gn + inc % gn) * MX_T;
}

// Four scales from p on of a matrix's n at base, at any alignment; in the place of bytes past the end, anything.
__device__ __forceinline__ uint32_t word_at(const uint8_t* p, const uint8_t* base, int64_t n) {
  uint32_t w = 0;
  if (n >= 4) {
    const uint8_t* last = base + n - 4;
    const uint8_t* q = p < last ? p : last;
    __builtin_memcpy(&w, q, 4);
    return w >> (8 * (int)(p - q));
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (p + i < base + n) w |= (uint32_t)p[i] << (8 * i);
  return w;
}

// DW: KB is a multiple of 4 and the scales are 4-byte aligned, so a row's scales come by LDS-DMA in words; without,
// a thread a row loads them as unaligned words and writes them to LDS (8192 x 8192 x 4064: 260 us, in bytes 485; with
// aligned rows 8192 x 8192 x 4096 takes 204)
template <typename T, bool DW>
__global__ void __launch_bounds__(256, 2) k_mxfp4_gemm(MxArgs a) {
  typedef MxMap<T> Map;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];  // (with a static array hipcc would drain every
                                                                  //  LDS-DMA in flight before an LDS read)
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int KB = a.KB, nk = (KB + 7) >> 3, tiles = a.nTm * a.nTn;
  const int wn = (wave & 1) * 64, wm = (wave >> 1) * 64;
  // staging: waves 0 and 1 take the W rows, 2 and 3 the A rows; an instruction fills 8 rows, lane l writes slot
  // l % 8 of row l / 8. The buffers end with the matrices: what lies behind reads as 0.
  const bool isw = wave < 2;
  int vo[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = (wave & 1) * 64 + i * 8 + (lane >> 3);
    vo[i] = row * KB * 16 + ((lane & 7) ^ (isw ? Map::wkey(row) : Map::akey(row))) * 16;
  }
  // a lane of the fragments reads the words of its four rows i at once
  const int srow = (wave & 1) * 64 + (isw ? Map::wrow(lane & 3, lane >> 2) : (lane & 3) * 16 + (lane >> 2));
  // (the second word's 4 bytes are part of the lane's offset: with the scalar offset past the end of an empty
  //  buffer the range check would be on a number below 0)
  const int so[2] = {srow * KB, srow * KB + 4};
  const uint8_t* sbase = nullptr;
  int rows = 0;
  __amdgpu_buffer_rsrc_t rc, rs;
  auto aim = [&](int64_t m0, int64_t n0, bool any) {
    rows = any ? (int)min((int64_t)MX_T, isw ? a.N - n0 : a.M - m0) : 0;
    sbase = isw ? a.ws + n0 * KB : a.as + m0 * KB;
    rc = __builtin_amdgcn_make_buffer_rsrc((void*)(isw ? a.wc + n0 * KB * 16 : a.ac + m0 * KB * 16), (short)0,
                                           rows * KB * 16, 0x00020000);
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)sbase, (short)0, rows * KB, 0x00020000);
  };
  // piece p of a stage: eight of codes, two of scales
  auto piece = [&](int kt, int b, int p) {
    uint8_t* dst = smem + b * MX_STAGE;
    if (p < 8)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rc, (__attribute__((address_space(3))) void*)(dst + (wave * 8 + p) * 1024), 16, vo[p], kt * 128, 0, 0);
    else if (DW)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(dst + MX_CODES + (p - 8) * 1024 + wave * 256), 4, so[(p - 8) & 1],
          8 * kt, 0, 0);
  };
  uint32_t pend[2] = {0, 0};  // !DW: this thread's row's scales of the stage on its way
  auto scale_words = [&](int kt) {
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const int at = 8 * kt + 4 * d;
      pend[d] = 0x7F7F7F7Fu;
      if (srow < rows && at < KB) pend[d] = word_at(sbase + so[0] + at, isw ? a.ws : a.as, (isw ? a.N : a.M) * KB);
    }
  };
  // fragment reads: the permutation does not depend on i, and block 4 h + g is slot (g ^ key) ^ 4 h
  const int ow = (wn + Map::wrow(0, r)) * 128 + (g ^ Map::wkey(Map::wrow(0, r))) * 16;
  const int oa = (MX_T + wm + r) * 128 + (g ^ Map::akey(r)) * 16;
  const int osw = MX_CODES + (wn + r * 4) * 4, osa = MX_CODES + (MX_T + wm + r * 4) * 4;
  int v = blockIdx.x, b = 0, relax = 0;
  int64_t m0, n0;
  tile_of(a, v, m0, n0);
  aim(m0, n0, true);
#pragma unroll
  for (int p = 0; p < 10; ++p) piece(0, 0, p);
  if (!DW) scale_words(0);
  while (true) {
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int nv = v + (int)gridDim.x;
    int64_t m1 = m0, n1 = n0;
    const bool inside = m0 + MX_T <= a.M && n0 + MX_T <= a.N && a.vec;
    MxVec<T> vec;
    for (int kt = 0; kt < nk; ++kt) {
      uint8_t* cur = smem + b * MX_STAGE;
      if (!DW) {
        *reinterpret_cast<uint32_t*>(cur + MX_CODES + t * 4) = pend[0];
        *reinterpret_cast<uint32_t*>(cur + MX_CODES + 1024 + t * 4) = pend[1];
      }
      // the previous tile's stores, younger than this stage's loads, may stay in flight
      if (DW && kt == 0 && relax) wait_vm<sizeof(T) == 4 ? 16 : 8>();
      else wait_vm<0>();
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
      __builtin_amdgcn_s_barrier();        // the stage is in LDS; everyone is done with the other one
      asm volatile("" ::: "memory");
      u32x4 fw[2][4], fa[2][4], sw[2], sa[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          fw[h][i] = *reinterpret_cast<const u32x4*>(cur + (ow ^ h * 64) + Map::wrow(i, 0) * 128);
          fa[h][i] = *reinterpret_cast<const u32x4*>(cur + (oa ^ h * 64) + i * 2048);
        }
        sw[h] = *reinterpret_cast<const u32x4*>(cur + osw + h * 1024);
        sa[h] = *reinterpret_cast<const u32x4*>(cur + osa + h * 1024);
      }
      // the next stage: of this tile, of the next one, or (an empty buffer, zeros) of none
      int next = kt + 1;
      if (next == nk) {
        next = 0;
        vec.load(a, m0 + wm, n0 + wn, r, g);
        if (nv < tiles) tile_of(a, nv, m1, n1);
        aim(m1, n1, nv < tiles);
      }
      if (!DW) scale_words(next);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sw[h][i] >>= 8 * g;
          sa[h][i] >>= 8 * g;
        }
      }
      if (8 * kt + 8 > KB) {  // past the last block: 0 * 1
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool in = 8 * kt + 4 * h + g < KB;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sw[h][i] = in ? sw[h][i] : 127;
            sa[h][i] = in ? sa[h][i] : 127;
#pragma unroll
            for (int x = 0; x < 4; ++x) fa[h][i][x] = in ? fa[h][i][x] : 0;
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // issuing a piece takes some sixty cycles: between matrix instructions they pass unnoticed
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          piece(next, b ^ 1, h * 5 + i);
          if (i == 3) piece(next, b ^ 1, h * 5 + 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = mfma_mx(fw[h][i], fa[h][j], acc[i][j], sw[h][i], sa[h][j]);
        }
#pragma unroll
        for (int x = 0; x < 5; ++x) {
          __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // one load
          __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);  // three matrix instructions
        }
      }
      b ^= 1;
    }
    int er = r, eg = g;
    asm volatile("" : "+v"(er), "+v"(eg));  // the epilogue's addresses are not kept through the K loop
    if (inside) mx_epilogue<T, false>(a, m0 + wm, n0 + wn, er, eg, acc, vec);
    else mx_epilogue<T, true>(a, m0 + wm, n0 + wn, er, eg, acc, vec);
    relax = inside;
    if (nv >= tiles) break;
    v = nv;
    m0 = m1;
    n0 = n1;
  }
  wait_vm<0>();  // the last stage's (empty) loads land before the LDS is given away
}

// Up to 16 MT rows of A: W is read once from memory straight into the fragments, a wave per 16 NT of its rows,
// U steps of K in flight; the A rows come from the caches. Bound by the read of W for few rows (two tables in turn:
// 1 x 1M x 768 79 us, 5.2 TB/s; 1 x 100000 x 4096 48 us, 4.5 TB/s), by the A fragments' way through the caches for
// many (16 x 1M x 768 110 us, 4.3 TB/s with the result, 64 x 1M x 768 210 us, 3.2 TB/s). DW: a row's four scales of
// a step are an aligned word; the four lanes of a row load the words of four steps and trade them (a byte a lane and
// step took 66 instead of 41 us at 1 x 100000 x 4096). Without, a lane loads its bytes (unaligned words took 100
// instead of 92 us at 1 x 1M x 736).
template <typename T, int MT, int NT, bool DW>
__global__ void __launch_bounds__(256) k_mxfp4_skinny(MxArgs a) {
  constexpr int U = NT == 4 ? (MT == 4 ? 1 : 2) : MT == 4 ? 2 : 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int64_t n0 = ((int64_t)blockIdx.x * 4 + wave) * (16 * NT);
  if (n0 >= a.N) return;
  const int KB = a.KB, nk = (KB + 3) >> 2;
  const uint8_t *wc[NT], *ws[NT], *ac[MT], *as[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int64_t row = min(n0 + i * 16 + r, a.N - 1);
    wc[i] = a.wc + row * KB * 16;
    ws[i] = a.ws + row * KB;
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int64_t row = min((int64_t)j * 16 + r, a.M - 1);
    ac[j] = a.ac + row * KB * 16;
    as[j] = a.as + row * KB;
  }
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto words = [&](const uint8_t* p, int k4) -> uint32_t {  // of step k4 + g
    return *reinterpret_cast<const uint32_t*>(p + 4 * min(k4 + g, nk - 1));
  };
  for (int k4 = 0; k4 < nk; k4 += 4) {
    uint32_t w4[NT], a4[MT];
    if (DW) {
#pragma unroll
      for (int i = 0; i < NT; ++i) w4[i] = words(ws[i], k4);
#pragma unroll
      for (int j = 0; j < MT; ++j) a4[j] = words(as[j], k4);
    }
#pragma unroll
    for (int k0 = 0; k0 < 4; k0 += U) {
      if (k4 + k0 >= nk) break;
      u32x4 fw[U][NT], fa[U][MT];
      uint32_t sw[U][NT], sa[U][MT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int b = min(4 * (k4 + k0 + u) + g, KB - 1);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          fw[u][i] = *reinterpret_cast<const u32x4*>(wc[i] + b * 16);
          if (!DW) sw[u][i] = ws[i][b];
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          fa[u][j] = *reinterpret_cast<const u32x4*>(ac[j] + b * 16);
          if (!DW) sa[u][j] = as[j][b];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (DW) {
#pragma unroll
          for (int i = 0; i < NT; ++i) sw[u][i] = (uint32_t)__shfl((int)w4[i], r + 16 * (k0 + u), 64) >> (8 * g);
#pragma unroll
          for (int j = 0; j < MT; ++j) sa[u][j] = (uint32_t)__shfl((int)a4[j], r + 16 * (k0 + u), 64) >> (8 * g);
        }
        if (4 * (k4 + k0 + u) + 4 > KB) {  // past the last block: 0 * 1
          const bool in = 4 * (k4 + k0 + u) + g < KB;
#pragma unroll
          for (int i = 0; i < NT; ++i) sw[u][i] = in ? sw[u][i] : 127;
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            sa[u][j] = in ? sa[u][j] : 127;
#pragma unroll
            for (int x = 0; x < 4; ++x) fa[u][j][x] = in ? fa[u][j][x] : 0;
          }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < MT; ++j) acc[i][j] = mfma_mx(fw[u][i], fa[u][j], acc[i][j], sw[u][i], sa[u][j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int64_t n = n0 + i * 16 + 4 * g;
    if (n >= a.N) continue;
    const Cols c = cols_of(a, n);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int64_t m = (int64_t)j * 16 + r;
      if (m < a.M) store4<T>(a, m, n, acc[i][j], (a.ra ? a.ra[m] : 1.f) * a.col_scale, c);
    }
  }
}

// ---- host --------------------------------------------------------------------------------------
static int lane_shift(int K) {  // lanes a row: enough for its eights, at least a block's four
  int sh = 2;
  while (sh < 6 && (8 << sh) < K) ++sh;
  return sh;
}

template <typename T, int NT, bool DW>
static void launch_skinny(const MxArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)((a.N + 64 * NT - 1) / (64 * NT));
  if (a.M <= 16) k_mxfp4_skinny<T, 1, NT, DW><<<grid, 256, 0, st>>>(a);
  else if (a.M <= 32) k_mxfp4_skinny<T, 2, NT, DW><<<grid, 256, 0, st>>>(a);
  else k_mxfp4_skinny<T, 4, NT, DW><<<grid, 256, 0, st>>>(a);
}

// Up to 64 rows a wave streams one tile of W's rows, or four that share the A fragments; the tile kernel shares W's
// lines through LDS as well and hides a long K better. Four: for more columns than two workgroups of one tile a CU,
// while K is short. One: for fewer (for 17 to 64 rows while its workgroups are one a CU), and for up to 4 rows,
// whose fragments cost little.
// us for one tile / four / tile kernel, fp32 results, the table read again and again:
//   K = 512:   1 x 400k 18.6 20.4 29.4; 16 x 400k 30.8 27.2 39.7; 64 x 50k 15.7 13.1 14.8; 64 x 16k 6.1 11.3 8.4
//   K = 1024:  1 x 400k 35.9 39.4 41.9; 32 x 400k 88.8 65.4 66.7; 64 x 400k 164 105 105;   64 x 16k 9.0 16.1 9.9
//   K = 1536: 16 x 400k 90.9 84.9 85.0; 32 x 400k 130 107 102;    64 x 400k 228 144 135;   64 x 16k 11.0 19.3 11.2
//   K = 4096:  1 x 400k 158 192 181;    16 x 400k 255 225 208;    32 x 16k 16.3 31.5 20.9; 64 x 16k 25.6 42.5 23.1
// From HBM, 1 x 1M x 768: 93.6 and 87.5 us (4.7 TB/s) for one and four.
template <typename T, bool DW>
static void launch_gemm(const MxArgs& a, hipStream_t st) {
  constexpr int cols = 64 * 256;  // of one workgroup a CU, a tile a wave
  const bool four = a.N > 2 * cols && a.KB <= (a.M <= 16 ? 48 : 32);
  const bool one = a.M <= 4 || (a.N <= (a.M <= 16 ? 2 : 1) * cols && (a.M <= 32 || a.KB <= 48));
  if (a.M <= 64 && four) return launch_skinny<T, 4, DW>(a, st);
  if (a.M <= 64 && one) return launch_skinny<T, 1, DW>(a, st);
  constexpr int lds = 2 * MX_STAGE;
  (void)hipFuncSetAttribute((const void*)k_mxfp4_gemm<T, DW>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  k_mxfp4_gemm<T, DW><<<(unsigned)std::min(a.nTm * a.nTn, MX_WGS), 256, lds, st>>>(a);
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace rf

using namespace rf;

extern "C" int rf_mxfp4_quantize(int dtype, int M, int K, const void* x, int64_t ldx, float eps, uint8_t* codes,
                                 uint8_t* scales, float* rnorm, rf_stream_t stream) {
  RF_REQUIRE(dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16, "rf_mxfp4_quantize: bad dtype %d", dtype);
  RF_REQUIRE(M >= 0 && K > 0 && K <= (1 << 24) && ldx >= K, "rf_mxfp4_quantize: bad shape M=%d K=%d", M, K);
  if (M == 0) return RF_OK;
  RF_REQUIRE(x && codes && scales, "rf_mxfp4_quantize: null pointer");
  const int es = dtype == RF_F32 ? 4 : 2;
  RF_REQUIRE((reinterpret_cast<uintptr_t>(x) & (es - 1)) == 0 && aligned16(codes),
             "rf_mxfp4_quantize: misaligned rows or codes");
  const int KB = (K + 31) / 32, sh = lane_shift(K);
  const int64_t blocks = (((int64_t)M << sh) + 255) / 256;
  RF_REQUIRE(blocks * 256 <= 0xFFFFFFFFll, "rf_mxfp4_quantize: %d rows are too many for a launch", M);
  hipStream_t st = as_stream(stream);
#define MXQ(T)                                                                                                      \
  k_mxfp4_quantize<T><<<(unsigned)blocks, 256, 0, st>>>(M, K, KB, (const T*)x, ldx, sh, eps, codes, scales, rnorm)
  if (dtype == RF_F32) MXQ(float);
  else if (dtype == RF_BF16) MXQ(bf16);
  else MXQ(f16);
#undef MXQ
  RF_LAUNCH_CHECK("rf_mxfp4_quantize");
}

extern "C" int rf_mxfp4_dequantize(int dtype, int M, int K, const uint8_t* codes, const uint8_t* scales, void* out,
                                   int64_t ldo, rf_stream_t stream) {
  RF_REQUIRE(dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16, "rf_mxfp4_dequantize: bad dtype %d", dtype);
  RF_REQUIRE(M >= 0 && K > 0 && K <= (1 << 24) && ldo >= K, "rf_mxfp4_dequantize: bad shape M=%d K=%d", M, K);
  if (M == 0) return RF_OK;
  RF_REQUIRE(out && codes && scales, "rf_mxfp4_dequantize: null pointer");
  const int es = dtype == RF_F32 ? 4 : 2;
  RF_REQUIRE((reinterpret_cast<uintptr_t>(out) & (es - 1)) == 0 && aligned16(codes),
             "rf_mxfp4_dequantize: misaligned rows or codes");
  const int KB = (K + 31) / 32, G = (K + 7) / 8;
  const bool vec = aligned16(out) && ldo * es % 16 == 0;
  const int64_t total = (int64_t)M * G, blocks = (total + 511) / 512;
  RF_REQUIRE(blocks * 256 <= 0xFFFFFFFFll, "rf_mxfp4_dequantize: %d rows are too many for a launch", M);
  hipStream_t st = as_stream(stream);
#define MXD(T) \
  k_mxfp4_dequantize<T><<<(unsigned)blocks, 256, 0, st>>>(total, G, K, KB, codes, scales, (T*)out, ldo, vec)
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
  RF_REQUIRE(M >= 0 && N >= 0 && K > 0 && K <= (1 << 24) && ldc >= N, "rf_mxfp4_gemm: bad shape M=%d N=%d K=%d", M, N,
             K);
  if (M == 0 || N == 0) return RF_OK;
  RF_REQUIRE(a_codes && a_scales && w_codes && w_scales && C, "rf_mxfp4_gemm: null pointer");
  RF_REQUIRE(!ra == !rw, "rf_mxfp4_gemm: ra and rw go together");
  const int es = out_dtype == RF_F32 ? 4 : 2;
  RF_REQUIRE(aligned16(a_codes) && aligned16(w_codes), "rf_mxfp4_gemm: codes must be 16-byte aligned");
  RF_REQUIRE((reinterpret_cast<uintptr_t>(C) & (4 * es - 1)) == 0 && ldc % 4 == 0,
             "rf_mxfp4_gemm: the result's rows must be aligned to four elements");
  RF_REQUIRE(ldc * es <= (1 << 26), "rf_mxfp4_gemm: rows of the result over 64 MB");  // 32-bit offsets over 17 rows
  RF_REQUIRE(aligned16(bias) && aligned16(rw), "rf_mxfp4_gemm: bias and rw must be 16-byte aligned");
  MxArgs a{};
  a.M = M; a.N = N; a.KB = (K + 31) / 32;
  a.ac = a_codes; a.as = a_scales; a.wc = w_codes; a.ws = w_scales;
  a.bias = bias; a.ra = ra; a.rw = rw; a.col_scale = col_scale; a.c = C; a.ldc = ldc;
  a.vec = aligned16(C) && ldc * es % 16 == 0;
  a.nTm = (int)((a.M + MX_T - 1) / MX_T);
  a.nTn = (int)((a.N + MX_T - 1) / MX_T);
  // row tiles whose codes fill half of an XCD's 4 MB of L2
  a.gm = (int)std::max<int64_t>(1, std::min<int64_t>(a.nTm, (2 << 20) / ((int64_t)MX_T * a.KB * 16)));
  // column tiles side by side (1, 4, 8: 428, 413, 416 us at 4096 x 125000 x 768 fp32; 8192^3 373, 379, 384)
  a.gn = 4;
  RF_REQUIRE((int64_t)a.nTm * a.nTn < 0x7FFFFFFF - MX_WGS, "rf_mxfp4_gemm: too many tiles");
  hipStream_t st = as_stream(stream);
  const bool dw = a.KB % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.as) | reinterpret_cast<uintptr_t>(a.ws)) & 3) == 0;
#define MXG(T) dw ? launch_gemm<T, true>(a, st) : launch_gemm<T, false>(a, st)
  if (out_dtype == RF_F32) MXG(float);
  else if (out_dtype == RF_BF16) MXG(bf16);
  else MXG(f16);
#undef MXG
  RF_LAUNCH_CHECK("rf_mxfp4_gemm");
}
