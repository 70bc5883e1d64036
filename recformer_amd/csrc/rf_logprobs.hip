// What the softmax of a logits row says and how it learns, beside the cross entropy of rf_rowops.hip:
// log probabilities of given entries, the entropy, the k best alternatives, a teacher's best logits to
// learn from, and the gradients of all of them. For a row x of N logits and an inverse temperature it,
//
//   m = max_c x_c,  t_c = (x_c - m) it,  s = sum_c e^t_c,  logp_c = t_c - ln s,  p_c = e^logp_c
//   H = ln s - (sum_c e^t_c t_c) / s                        (both terms >= 0: nothing cancels)
//   top k: the k largest x_c, the lower index first among equals
//   distillation: q = softmax(teacher logits it) over the row's K listed ids (id -1 or logit -inf: not
//     listed), loss = sum_k q_k (ln q_k - logp_id_k)
//   gradients:  dx_c = it (a p_c + b p_c logp_c + sum of w_j over the listed entries j with id_j = c)
//     log probabilities (weights g_j) and entropy (weight h): a = -sum_j g_j - h H, b = -h, w_j = g_j
//     distillation (weight g): a = g (0 for a row that lists nothing), b = 0, w_j = -g q_j
//
// -inf logits (masked columns) have p = 0 and add nothing. A row that is all -inf has no distribution:
// log probabilities -inf, entropy 0, gradient 0. NaN or +inf in a row makes its numbers NaN (its top ids
// stay defined: NaN first). Entries equal to ignore_index count 0 and get no gradient; any other id
// outside [0, N) makes its number NaN.
//
// HBM bound: the forward reads the row once, the backward reads it once and writes it once. A workgroup
// holds its slice of a row in registers (up to LP_R 16-byte chunks a thread), so the maximum, the sums and the
// alternatives all come from one read, and no running rescale is needed. Sums and exponents are fp32.
// Rows longer than a workgroup holds are cut into slices whose (m, s, sum e^t t) and k best are joined by a
// second launch; no atomics on memory, so results do not depend on scheduling.
#include "rf_common.h"

#include <algorithm>

namespace rf {

constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;
constexpr float LP_NINF = -__builtin_inff();
constexpr int LP_R = 8;         // 16-byte chunks of a row per thread
constexpr int LP_KMAX = 256;    // alternatives
constexpr int LP_LIST = 1024;   // given entries / teacher entries per row
constexpr int LP_NMAX = 0x7FFFFFFF - (1 << 16);  // columns: a workgroup's numbers past the end of a row fit 32 bits
constexpr float LP_ITMAX = 2e38f;                // it log2(e) is finite

// ---- elements of a row -----------------------------------------------------------------------
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename T> struct Row;
template <> struct Row<float> {
  static constexpr int V = 4;
  static constexpr uint32_t FILL = 0xFF800000u;
  static constexpr bool ROUND = true;  // its values do not all fit bf16
  static __device__ __forceinline__ float at(const u32x4& r, int e) { return __uint_as_float(r[e]); }
};
template <> struct Row<bf16> {
  static constexpr int V = 8;
  static constexpr uint32_t FILL = 0xFF80FF80u;
  static constexpr bool ROUND = false;
  static __device__ __forceinline__ float at(const u32x4& r, int e) {
    return __uint_as_float(e & 1 ? r[e >> 1] & 0xFFFF0000u : r[e >> 1] << 16);
  }
};
template <> struct Row<f16> {
  static constexpr int V = 8;
  static constexpr uint32_t FILL = 0xFC00FC00u;
  static constexpr bool ROUND = true;
  static __device__ __forceinline__ float at(const u32x4& r, int e) {
    const uint32_t w = r[e >> 1];  // (a bit cast of the vector's element itself would read element 0)
    return (float)__builtin_bit_cast(f16x2, w)[e & 1];
  }
};

template <typename T>
__device__ __forceinline__ float chunk_max(const u32x4& r) {  // NaN is passed over
  float v = Row<T>::at(r, 0);
#pragma unroll
  for (int e = 1; e < Row<T>::V; ++e) v = fmaxf(v, Row<T>::at(r, e));
  return v;
}

// A row starts `off` elements into its first aligned 16-byte chunk; chunk j holds the columns
// [j V - off, j V - off + V). Chunks that reach over an end of the row are read element by element.
template <typename T>
__device__ __forceinline__ int row_off(const T* x) {
  return (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
}
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* x, int c0, int N) {
  constexpr int V = Row<T>::V;
  if (c0 >= 0 && c0 <= N - V) return *reinterpret_cast<const u32x4*>(x + c0);
  T v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = c0 + e >= 0 && c0 + e < N ? x[c0 + e] : from_f32<T>(LP_NINF);
  u32x4 r;
  __builtin_memcpy(&r, v, 16);
  return r;
}

// order of the alternatives: larger key first; -0 = +0, NaN above +inf
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  if (k == 0xFFFFFFFFu) return __builtin_nanf("");
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// (key, column) as one number: larger = earlier in the list
__device__ __forceinline__ uint64_t entry_of(float v, uint32_t col) {
  return (uint64_t)key_of(v) << 32 | (uint32_t)~col;
}

// ---- workgroup reductions ----------------------------------------------------------------------
// the waves' results joined by every wave from LDS, a value a lane (read side by side, sixteen values would not
// fit the registers beside a row)
template <int TPB>
__device__ __forceinline__ float waves_max(const float* red) {
  constexpr int W = TPB / 64;
  float v = red[threadIdx.x & (W - 1)];
#pragma unroll
  for (int o = W >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
template <int TPB>
__device__ __forceinline__ float waves_sum(const float* red) {
  constexpr int W = TPB / 64;
  float v = red[threadIdx.x & (W - 1)];
#pragma unroll
  for (int o = W >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int TPB>
__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return waves_max<TPB>(red);
}
template <int TPB>
__device__ __forceinline__ void block_sum2(float& a, float& b, float* red) {
  a = wave_sum(a);
  b = wave_sum(b);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = a;
    red[16 + (threadIdx.x >> 6)] = b;
  }
  __syncthreads();
  a = waves_sum<TPB>(red);
  b = waves_sum<TPB>(red + 16);
}

// ---- the k best of a workgroup's entries -------------------------------------------------------
template <int TPB>
struct SelectLds {
  static constexpr int CAP = TPB == 1024 ? 2048 : TPB == 256 ? 1024 : 512;  // candidates, at least LP_KMAX
  uint64_t cand[CAP];
  // the threads' largest keys; the histogram of the exact search
  __attribute__((aligned(16))) uint32_t key[TPB < 256 ? 256 : TPB];
  int count;
  uint32_t tau;
  uint64_t prefix;
  int rem, done;
};

// the upper 16 bits of the k-th largest of a wave's keys (0 where it holds fewer)
template <int PER>
__device__ __forceinline__ uint32_t upper_bits(const uint32_t (&g)[PER], int k) {
  uint32_t tau = 0;
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t c = tau | 1u << bit;
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) cnt += __popcll(__ballot(g[i] >= c));
    if (cnt >= k) tau = c;
  }
  return tau;
}

// The k best of a workgroup's entries, in three steps with a barrier after each: every thread enters the key
// of its largest value into s.key (and thread 0 clears s.count); one wave finds s.tau; every thread collects
// what passes.
//
// The k-th largest of the threads' maxima is a lower bound of the k-th largest entry (k threads hold one at
// least as large), and few entries lie above it: G groups of threads let about G ln(G / (G - k)) through (56
// for k = 50 and G = 256, and G = 1024 would take four times the counting to save 4). Its upper 16 bits do. Where
// fewer than k threads hold entries the bound is 0 and everything passes.
template <int TPB>
__device__ __forceinline__ void find_tau(SelectLds<TPB>& s, int lane, int k) {
  uint32_t tau;
  if (TPB == 1024 && k <= 64) {  // groups of four threads
    uint32_t g[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 q = *reinterpret_cast<const u32x4*>(&s.key[(i * 64 + lane) * 4 % (TPB < 256 ? 256 : TPB)]);
      g[i] = max(max(q[0], q[1]), max(q[2], q[3]));
    }
    tau = upper_bits(g, k);
  } else if (TPB == 1024) {  // of two: 355 pass for k = 256
    uint32_t g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = (i * 64 + lane) * 2 % (TPB < 256 ? 256 : TPB);
      g[i] = max(s.key[at], s.key[at + 1]);
    }
    tau = upper_bits(g, k);
  } else {
    uint32_t g[TPB / 64];
#pragma unroll
    for (int i = 0; i < TPB / 64; ++i) g[i] = s.key[i * 64 + lane];
    tau = upper_bits(g, k);
  }
  if (lane == 0) s.tau = tau;
}

// The exact search: collects into s.cand the min(k, n) best of src.all's n entries by the digits (8 bits from the top)
// of the last one taken; stops as soon as a digit's whole bin is taken. It is rare, and a function of its own so
// that its registers do not crowd out the short way's.
template <int TPB, typename Src>
__device__ __attribute__((noinline)) int collect_exact(const Src src, int k, int64_t n, SelectLds<TPB>* sel) {
  SelectLds<TPB>& s = *sel;
  const int t = threadIdx.x;
  const int kk = (int)(n < k ? n : k);
  uint64_t prefix = 0;
  int rem = kk, shift = 64;
  while (true) {
    __syncthreads();
    for (int i = t; i < 256; i += TPB) s.key[i] = 0;
    __syncthreads();
    src.all([&](uint64_t e) {
      if (shift != 64 && (e >> shift) != prefix) return;
      const int d = (int)(e >> (shift - 8)) & 255;
      const uint64_t here = __ballot(1);
      if (__ballot(d == __builtin_amdgcn_readfirstlane(d)) == here) {  // adds to one address would go one by one
        if ((t & 63) == __builtin_ctzll(here)) atomicAdd(&s.key[d], (uint32_t)__popcll(here));
      } else {
        atomicAdd(&s.key[d], 1u);
      }
    });
    __syncthreads();
    if (t < 64) {  // four digits a lane, the highest first
      int h[4], sum = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) sum += h[x] = (int)s.key[255 - 4 * t - x];
      int above = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(above, o, 64);
        if (t >= o) above += v;
      }
      above -= sum;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (above < rem && above + h[x] >= rem) {  // one lane's, once
          s.prefix = prefix << 8 | (uint64_t)(255 - 4 * t - x);
          s.rem = rem - above;
          s.done = h[x] == rem - above;
        }
        above += h[x];
      }
    }
    __syncthreads();
    prefix = s.prefix;
    rem = s.rem;
    shift -= 8;
    if (s.done || shift == 0) break;
  }
  const uint64_t least = prefix << shift;
  __syncthreads();
  if (t == 0) s.count = 0;
  __syncthreads();
  src.all([&](uint64_t e) {
    if (e < least) return;
    const int at = atomicAdd(&s.count, 1);
    if (at < SelectLds<TPB>::CAP) s.cand[at] = e;
  });
  __syncthreads();
  return min(s.count, SelectLds<TPB>::CAP);
}

// Collects into s.cand what passes s.tau, at least min(k, n) entries and among them the k best, and returns how
// many. src.each(tau, f) calls f(entry) for every entry of the calling thread whose key is >= tau,
// src.again().all(f) for all its entries; nan: some value is NaN (the float compares of src.each would miss it).
// Where more than CAP entries pass (many equal values, or the best all in few threads) the exact search follows.
template <int TPB, typename Src>
__device__ __forceinline__ int collect(const Src& src, bool nan, int k, int64_t n, SelectLds<TPB>& s) {
  auto take = [&](uint64_t e) {
    const int at = atomicAdd(&s.count, 1);
    if (at < SelectLds<TPB>::CAP) s.cand[at] = e;
  };
  if (!nan) {
    src.each(s.tau, take);
    __syncthreads();
    const int c = s.count;
    if (c <= SelectLds<TPB>::CAP) return c;
  }
  return collect_exact<TPB>(src.again(), k, n, &s);
}

// f(rank, entry) for the candidates in list order: entries are all different, so an entry's rank is the
// number of larger ones. Counted by one lane each (several lanes an entry took 4% longer at 4915 x 50265 top 20),
// by two where there are many.
template <int TPB, int L, typename F>
__device__ __forceinline__ void rank_by(const SelectLds<TPB>& s, int c, int k, F f) {  // L lanes an entry
  for (int i = threadIdx.x / L; i < c; i += TPB / L) {
    const uint64_t e = s.cand[i];
    int r = 0, j = 4 * (threadIdx.x % L);
    for (; j + 4 <= c; j += 4 * L) {  // reads of four together: their latencies overlap
      const uint64_t a0 = s.cand[j], a1 = s.cand[j + 1], a2 = s.cand[j + 2], a3 = s.cand[j + 3];
      r += (a0 > e) + (a1 > e) + (a2 > e) + (a3 > e);
    }
    for (; j < c; ++j) r += s.cand[j] > e;
    if (L == 2) r += __builtin_amdgcn_mov_dpp(r, 0xB1, 0xF, 0xF, true);  // the neighbour's
    if (r < k && (L == 1 || !(threadIdx.x & 1))) f(r, e);
  }
}
template <int TPB, typename F>
__device__ __forceinline__ void rank_candidates(const SelectLds<TPB>& s, int c, int k, F f) {
  if (TPB == 1024 && c > 128) rank_by<TPB, 2>(s, c, k, f);
  else rank_by<TPB, 1>(s, c, k, f);
}

// ---- what a finished row gives -----------------------------------------------------------------
struct LpArgs {
  int M, N, S, cps;          // rows, columns, slices per row, chunks per slice
  int64_t ld;
  float it, c2;              // inverse temperature; it log2(e)
  const int64_t* ids;        // given entries (M, C), or the teacher's (M, K)
  int nids;
  int64_t ignore;
  const float* tval;         // teacher logits (M, K); NULL: log probabilities
  int k;                     // alternatives
  float* logp;               // (M, C), or the distillation loss per row (M)
  float* entropy;            // (M) or NULL
  float* top_logp;           // (M, k)
  int64_t* top_ids;
  float* stats;              // (M, 4): m, 1 / s, teacher maximum, 1 / teacher sum
  float* part;               // (M S, 4): m, s, sum e^t t log2(e), -
  uint64_t* pent;            // (M S, k) entries, 0 = none
};

// The thread's entry of a row's list (entry t; the lists' rest is read where it is needed): loaded before the
// row, its logit after it, so that the row's end does not wait for them.
template <bool TEACH>
struct Listed {
  int32_t id;  // -1: ignored or not used, -2: out of range
  float t, x;  // teacher logit; logit of the row
  __device__ __forceinline__ void load(const LpArgs& a, int r, int j) {
    const int64_t k = j < a.nids ? a.ids[(int64_t)r * a.nids + j] : -1;
    id = k == (TEACH ? -1 : a.ignore) ? -1 : k >= 0 && k < a.N ? (int32_t)k : -2;
    if (TEACH) t = j < a.nids ? a.tval[(int64_t)r * a.nids + j] : 0.f;
  }
  template <typename T>
  __device__ __forceinline__ void look(const T* __restrict__ row) {
    x = id >= 0 ? to_f32(row[id]) : __builtin_nanf("");
  }
};

// m, s and h = sum e^t t log2(e) of row r are known to the whole workgroup
template <int TPB, bool TEACH, typename T>
__device__ __forceinline__ void finish_row(const LpArgs& a, int r, const T* __restrict__ row, float m, float s, float h,
                                           const Listed<TEACH>& own, float* red) {
  const int t = threadIdx.x;
  const bool empty = s == 0.f;
  const float ls = empty ? 0.f : __builtin_amdgcn_logf(s) * LP_LN2;
  // own.x is NaN for an id out of range
  auto logp = [&](float v) { return v != v ? v : empty || v == LP_NINF ? (s != s ? s : LP_NINF) : (v - m) * a.it - ls; };
  auto each = [&](auto f) {
    if (t < a.nids) f(t, own);
    for (int j = t + TPB; j < a.nids; j += TPB) {
      Listed<TEACH> l;
      l.load(a, r, j);
      l.look(row);
      f(j, l);
    }
  };
  float tm = 0.f, trs = 0.f;
  if constexpr (TEACH) {
    auto top = [&](float mx, const Listed<TEACH>& l) { return l.id != -1 ? fmaxf(mx, l.t) : mx; };
    float ts = 0.f, cross = 0.f;
    auto add = [&](const Listed<TEACH>& l) {
      if (l.id == -1) return;
      const float tz = (l.t - tm) * a.it;
      const float e = __builtin_amdgcn_exp2f(tz * LP_LOG2E);
      ts += e;
      if (e != 0.f) cross += e * (tz - logp(l.x));  // a teacher logit of -inf teaches nothing, whatever the student says
    };
    if (a.nids <= 64) {  // the first wave's entries: no barriers
      if (t >= 64) return;
      tm = wave_max(top(LP_NINF, own));
      if (tm == LP_NINF) tm = 0.f;
      add(own);
      ts = wave_sum(ts);
      cross = wave_sum(cross);
    } else {
      float mx = LP_NINF;
      each([&](int, const Listed<TEACH>& l) { mx = top(mx, l); });
      tm = block_max<TPB>(mx, red);
      if (tm == LP_NINF) tm = 0.f;
      each([&](int, const Listed<TEACH>& l) { add(l); });
      block_sum2<TPB>(ts, cross, red);
    }
    trs = ts == 0.f ? 0.f : 1.f / ts;
    // sum q (tz - ln ts - logp) with q = e / ts
    if (t == 0) a.logp[r] = ts == 0.f ? 0.f : cross * trs - __builtin_amdgcn_logf(ts) * LP_LN2;
  } else {
    each([&](int j, const Listed<TEACH>& l) { a.logp[(int64_t)r * a.nids + j] = l.id == -1 ? 0.f : logp(l.x); });
    if (t == 0 && a.entropy) a.entropy[r] = empty ? 0.f : ls - h / s * LP_LN2;
  }
  if (t == 0 && a.stats) {
    float* st = a.stats + (int64_t)r * 4;
    st[0] = m;
    st[1] = empty ? 0.f : 1.f / s;
    st[2] = tm;
    st[3] = trs;
  }
}

template <int TPB>
__device__ __forceinline__ void write_top(const LpArgs& a, int r, float m, float s, const SelectLds<TPB>& sel, int c) {
  const bool empty = s == 0.f;
  const float ls = empty ? 0.f : __builtin_amdgcn_logf(s) * LP_LN2;
  rank_candidates<TPB>(sel, c, a.k, [&](int rank, uint64_t e) {
    const float v = value_of((uint32_t)(e >> 32));
    const int64_t o = (int64_t)r * a.k + rank;
    a.top_logp[o] = empty || v == LP_NINF ? (s != s ? s : LP_NINF) : (v - m) * a.it - ls;
    a.top_ids[o] = (int64_t)(uint32_t)~(uint32_t)e;
  });
}

// A slice of a row: the short way looks at the chunks a thread holds, the exact search reads the row again
// (it is rare, and unrolled over the registers its code would crowd out the rest).
template <typename T, int TPB>
struct RowSrc {
  const T* x;
  u32x4* raw;
  const uint32_t* top;  // the chunks' maxima rounded up to bf16
  int j0, jn, off, N;  // the slice's chunks [j0, j0 + jn)
  template <typename F>
  __device__ __forceinline__ void each(uint32_t tau, F f) const {
    constexpr int V = Row<T>::V;
    // keys at or below -inf's: every column; otherwise an ordinary float compare
    const float lim = tau <= 0x007FFFFFu ? LP_NINF : value_of(tau);
    int base = (j0 + (int)threadIdx.x) * V - off, have = jn - (int)threadIdx.x;
    asm volatile("" : "+v"(base), "+v"(have));
#pragma unroll
    for (int i = 0; i < LP_R; ++i) {
      if (i * TPB < have && __uint_as_float(i & 1 ? top[i / 2] & 0xFFFF0000u : top[i / 2] << 16) >= lim) {
        asm volatile("" : "+v"(raw[i]));
        const int c0 = base + i * TPB * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float v = Row<T>::at(raw[i], e);
          if (v >= lim && c0 + e >= 0 && c0 + e < N) f(entry_of(v, (uint32_t)(c0 + e)));
        }
      }
    }
  }
  struct Again {
    const T* x;
    int64_t c0, c1;
    template <typename F>
    __device__ __forceinline__ void all(F f) const {
      for (int64_t c = c0 + threadIdx.x; c < c1; c += TPB) f(entry_of(to_f32(x[c]), (uint32_t)c));
    }
  };
  __device__ __forceinline__ Again again() const {
    constexpr int V = Row<T>::V;
    return {x, max((int64_t)j0 * V - off, (int64_t)0), min((int64_t)(j0 + jn) * V - off, (int64_t)N)};
  }
};

// ---- one slice of a row ------------------------------------------------------------------------
// Loads, maximum, exponentials and alternatives follow one another within a workgroup; two of 1024 threads a CU
// (64 registers) let one load while the other computes. Reading bounds it for fp32 (128 x 1M: 88 us, 5.8 TB/s);
// 16-bit rows come within a tenth or two of that (4915 x 50265 bf16: 98 us, 5.1 TB/s), and what comes on top shows:
// the entropy's two operations an element (110 us), the barriers and the one-wave search of the alternatives (top 20
// 130 us, with the entropy 133, top 256 216 and 224; 128 x 1M fp32 top 50 with the entropy 110). Launches one after
// another over three inputs in turn.
// With alternatives the 1024 threads' 64 registers do not hold it all: four of a thread's go to scratch memory, for
// bf16 one of them in every thread, which writes 20 MB at 4915 x 50265 where the results are 1.3 MB.
template <typename T, int TPB, bool ENT, bool TOP, bool TEACH>
__global__ void __launch_bounds__(TPB, TPB == 1024 ? 8 : 4) k_logprobs(LpArgs a, const T* __restrict__ logits) {
  constexpr int V = Row<T>::V;
  __shared__ float redm[16], reds[32];
  __shared__ SelectLds<TPB> sel;
  const int t = threadIdx.x;
  const int r = blockIdx.x / a.S, sl = blockIdx.x % a.S;
  const T* x = logits + (int64_t)r * a.ld;
  const int off = row_off(x);
  const int nch = (int)(((int64_t)a.N + off + V - 1) / V);
  const int j0 = min(sl * a.cps, nch), jn = min(a.cps, nch - j0);
  Listed<TEACH> own;
  if (a.S == 1) own.load(a, r, t);
  u32x4 raw[LP_R];
#pragma unroll
  for (int i = 0; i < LP_R; ++i) {
    const int j = i * TPB + t;
    if (j < jn) raw[i] = load_chunk(x, (j0 + j) * V - off, a.N);
    else raw[i] = u32x4{Row<T>::FILL, Row<T>::FILL, Row<T>::FILL, Row<T>::FILL};
  }
  float tmax = LP_NINF;
  uint32_t top[LP_R / 2];  // the chunks' maxima rounded up to bf16, two a word
#pragma unroll
  for (int i = 0; i < LP_R; ++i) {
    const float v = chunk_max<T>(raw[i]);
    tmax = fmaxf(tmax, v);
    if (TOP) {
      const uint32_t b = __float_as_uint(v), up = Row<T>::ROUND ? (b >> 31 ? b : b + 0xFFFFu) : b;
      top[i / 2] = i & 1 ? top[i / 2] | (up & 0xFFFF0000u) : up >> 16;
    }
  }
  if (a.S == 1) own.look(x);
  const int wave = t >> 6;
  const float wmax = wave_max(tmax);
  if ((t & 63) == 0) redm[wave] = wmax;
  if (TOP) {
    sel.key[t] = key_of(tmax);
    if (t == 0) sel.count = 0;
  }
  __syncthreads();
  float m = waves_max<TPB>(redm);
  if (m == LP_NINF) m = 0.f;
  if (TOP && wave == TPB / 64 - 1) find_tau<TPB>(sel, t & 63, a.k);
  // per element: subtract, scale, v_exp, one add, and for the entropy a clamp (so that 0 * -inf stays 0; e^t is 0
  // from 2^-150 on) and an fma
  // (the empty asm keeps the values packed between the passes: unpacked they would not fit the registers)
  float s = 0.f, h = 0.f;
#pragma unroll
  for (int i = 0; i < LP_R; ++i) {
    if (i * TPB < jn) {
      asm volatile("" : "+v"(raw[i]));
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float u = (Row<T>::at(raw[i], e) - m) * a.c2;
        const float p = __builtin_amdgcn_exp2f(u);
        s += p;
        if (ENT) h = fmaf(p, fmaxf(u, -200.f), h);
      }
    }
  }
  s = wave_sum(s);
  if (ENT) h = wave_sum(h);
  if ((t & 63) == 0) {
    reds[wave] = s;
    if (ENT) reds[16 + wave] = h;
  }
  __syncthreads();
  s = waves_sum<TPB>(reds);
  h = ENT ? waves_sum<TPB>(reds + 16) : 0.f;
  if (!(s < __builtin_inff())) s = __builtin_nanf("");  // NaN or +inf in the row
  if (a.S == 1) {
    finish_row<TPB, TEACH>(a, r, x, m, s, h, own, reds);
  } else if (t == 0) {
    float* p = a.part + (int64_t)blockIdx.x * 4;
    p[0] = s == 0.f ? LP_NINF : m;
    p[1] = s;
    p[2] = h;
  }
  if (TOP) {
    const int64_t first = max((int64_t)j0 * V - off, (int64_t)0);
    const int64_t n = max(min((int64_t)(j0 + jn) * V - off, (int64_t)a.N) - first, (int64_t)0);
    const RowSrc<T, TPB> src{x, raw, top, j0, jn, off, a.N};
    const int c = collect<TPB>(src, s != s, a.k, n, sel);
    if (a.S == 1) {
      write_top<TPB>(a, r, m, s, sel, c);
    } else {
      uint64_t* o = a.pent + (int64_t)blockIdx.x * a.k;
      rank_candidates<TPB>(sel, c, a.k, [&](int rank, uint64_t e) { o[rank] = e; });
      for (int i = c + t; i < a.k; i += TPB) o[i] = 0;
    }
  }
}

// ---- the slices of a row joined ----------------------------------------------------------------
// A workgroup a row. Latency: 4 us for the sums (16 x 200000), 8 with 50 alternatives of each slice.
template <int TPB>
struct ListSrc {
  const uint64_t* ent;
  uint32_t S, k;
  // the lists' first entries before their second ones: a thread's entries are of different ranks, so the threads'
  // maxima are the best of all lists (in the lists' own order the bound let 2048 of 16 lists of 256 through)
  template <typename F>
  __device__ __forceinline__ void each(uint32_t tau, F f) const {
    for (uint32_t i = threadIdx.x; i < S * k; i += TPB) {
      const uint64_t e = ent[i % S * k + i / S];
      if (e != 0 && (uint32_t)(e >> 32) >= tau) f(e);
    }
  }
  __device__ __forceinline__ ListSrc again() const { return *this; }
  template <typename F>
  __device__ __forceinline__ void all(F f) const { each(0u, f); }
};

template <typename T, int TPB, bool TOP, bool TEACH>
__global__ void __launch_bounds__(TPB) k_logprobs_join(LpArgs a, const T* __restrict__ logits) {
  __shared__ float red[32];
  __shared__ SelectLds<TPB> sel;
  const int t = threadIdx.x, r = blockIdx.x;
  const T* x = logits + (int64_t)r * a.ld;
  Listed<TEACH> own;
  own.load(a, r, t);
  own.look(x);
  const float* part = a.part + (int64_t)r * a.S * 4;
  float m = LP_NINF;
  for (int i = t; i < a.S; i += TPB) m = fmaxf(m, part[4 * i]);
  m = block_max<TPB>(m, red);
  if (m == LP_NINF) m = 0.f;
  float s = 0.f, h = 0.f;
  for (int i = t; i < a.S; i += TPB) {
    const float mi = part[4 * i], si = part[4 * i + 1];
    if (si == 0.f) continue;  // a slice with nothing in it
    const float d = (mi - m) * a.c2;  // the slice's exponents move by d: sum e^(u + d) (u + d)
    const float f = __builtin_amdgcn_exp2f(d);
    s = fmaf(si, f, s);
    h = fmaf(f, fmaf(fmaxf(d, -200.f), si, part[4 * i + 2]), h);
  }
  block_sum2<TPB>(s, h, red);
  finish_row<TPB, TEACH>(a, r, x, m, s, h, own, red);
  if (TOP) {
    const ListSrc<TPB> src{a.pent + (int64_t)r * a.S * a.k, (uint32_t)a.S, (uint32_t)a.k};
    uint64_t best = 0;
    src.all([&](uint64_t e) { best = max(best, e); });
    sel.key[t] = (uint32_t)(best >> 32);
    if (t == 0) sel.count = 0;
    __syncthreads();
    if (t < 64) find_tau<TPB>(sel, t, a.k);
    __syncthreads();
    const int c = collect<TPB>(src, false, a.k, (int64_t)a.S * a.k, sel);
    write_top<TPB>(a, r, m, s, sel, c);
  }
}

// ---- mean of the rows' losses over the rows that list something --------------------------------
// loss = scale sum(rows) / n, coef = scale / n with n = #{r : 1 / teacher sum != 0}; one workgroup, so
// the order of the sum is fixed (0 / 0 = NaN where no row lists anything, as the mean cross entropy has it). Latency:
// 4.5 us for 4915 rows, and in proportion to M from there on (34 us for 100000, 311 for 1M)
__global__ void __launch_bounds__(1024) k_rows_mean(int M, const float* __restrict__ rows,
                                                    const float* __restrict__ stats, float scale,
                                                    float* __restrict__ loss, float* __restrict__ coef) {
  __shared__ float red[32];
  float a = 0.f, n = 0.f;
  for (int r = threadIdx.x; r < M; r += 1024) {
    a += rows[r];
    n += stats[4 * (int64_t)r + 3] != 0.f ? 1.f : 0.f;
  }
  block_sum2<1024>(a, n, red);
  if (threadIdx.x == 0) {
    *loss = a * scale / n;
    *coef = scale / n;
  }
}

// ---- gradients ---------------------------------------------------------------------------------
constexpr int LB_R = 4;

struct LpBwdArgs {
  int M, N, S, cps;
  int64_t ld, ldd;
  float it, c2;
  const int64_t* ids;
  int nids;
  int64_t ignore;
  const float* tval;    // teacher logits; NULL: log probabilities
  const float* g;       // (M, C) weights of the log probabilities, or one weight of the loss; may be NULL
  const float* coef;    // distillation: a factor of that weight
  const float* entropy; // (M), with g_ent
  const float* g_ent;   // (M) weights of the entropy or NULL
  const float* stats;   // (M, 4)
};

// One slice of a row: read, e^t / s, write. The listed entries are then written again by one thread each
// (after a barrier; the first of equal ids adds all their weights in list order), so nothing is added
// atomically. HBM bound: 4915 x 50265 bf16 166 us (6.0 TB/s), 128 x 1M fp32 205 (5.0 TB/s); LB_R chunks a thread
// keep enough loads in flight beside the stores.
// PAST: the gradient is written past the caches.
template <typename T, int TPB, bool ENT, bool PAST>
__global__ void __launch_bounds__(TPB) k_logprobs_bwd(LpBwdArgs a, const T* __restrict__ logits,
                                                         T* __restrict__ dlogits) {
  constexpr int V = Row<T>::V;
  __shared__ float red[32];
  constexpr int LIST = TPB == 64 ? 64 : LP_LIST;
  __shared__ int32_t sid[LIST];
  __shared__ float sw[LIST];
  const int t = threadIdx.x;
  const int r = blockIdx.x / a.S, sl = blockIdx.x % a.S;
  const T* x = logits + (int64_t)r * a.ld;
  T* dx = dlogits + (int64_t)r * a.ldd;
  const int off = row_off(x);  // dx starts as far into its chunk (checked by the caller)
  const int nch = (int)(((int64_t)a.N + off + V - 1) / V);
  const int j0 = min(sl * a.cps, nch), jn = min(a.cps, nch - j0);
  u32x4 raw[LB_R];
#pragma unroll
  for (int i = 0; i < LB_R; ++i) {
    const int j = i * TPB + t;
    if (j < jn) raw[i] = load_chunk(x, (j0 + j) * V - off, a.N);
  }
  const float m = a.stats[4 * (int64_t)r], rs = a.stats[4 * (int64_t)r + 1];
  const bool empty = rs == 0.f;
  const float nan = __builtin_nanf("");
  float ca = 0.f, cb = 0.f;
  if (a.tval) {
    const float tm = a.stats[4 * (int64_t)r + 2], trs = a.stats[4 * (int64_t)r + 3];
    const float g = a.g[0] * a.coef[0];
    float bad = 0.f, unused = 0.f;
    for (int j = t; j < a.nids; j += TPB) {
      const int64_t id = a.ids[(int64_t)r * a.nids + j];
      const float q = id == -1 ? 0.f : __builtin_amdgcn_exp2f((a.tval[(int64_t)r * a.nids + j] - tm) * a.c2) * trs;
      const bool in = id >= 0 && id < a.N;
      if (!in && id != -1 && q != 0.f) bad = nan;
      sid[j] = in && q != 0.f ? (int32_t)id : -1;
      sw[j] = -g * q;
    }
    block_sum2<TPB>(bad, unused, red);
    ca = trs == 0.f ? 0.f : g + bad;
  } else {
    float sum = 0.f, unused = 0.f;
    for (int j = t; j < a.nids; j += TPB) {
      const int64_t id = a.ids[(int64_t)r * a.nids + j];
      const bool in = id >= 0 && id < a.N;
      const float g = a.g && id != a.ignore ? a.g[(int64_t)r * a.nids + j] : 0.f;
      sum += in || id == a.ignore ? (id == a.ignore ? 0.f : g) : nan;
      sid[j] = in && id != a.ignore ? (int32_t)id : -1;
      sw[j] = g;
    }
    block_sum2<TPB>(sum, unused, red);
    ca = -sum;
    if (ENT) {
      cb = -a.g_ent[r];
      ca = fmaf(cb, a.entropy[r], ca);
    }
  }
  const float lrs = empty ? 0.f : __builtin_amdgcn_logf(rs) * LP_LN2;  // -ln s
  // the gradient over it: the temperature comes last, since it c alone may be past fp32's range (0 * inf in the
  // columns of p = 0, inf - inf where the weights of a listed entry and of p cancel)
  ca *= rs;
  cb *= rs;
  auto grad = [&](float v) {
    const float u = (v - m) * a.c2;
    return __builtin_amdgcn_exp2f(u) * (ENT ? fmaf(cb, fmaf(fmaxf(u, -200.f), LP_LN2, lrs), ca) : ca);
  };
#pragma unroll
  for (int i = 0; i < LB_R; ++i) {
    const int j = i * TPB + t;
    if (j < jn) {
      const int64_t c0 = (int64_t)(j0 + j) * V - off;
      T o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = from_f32<T>(empty ? 0.f : a.it * grad(Row<T>::at(raw[i], e)));
      if (c0 >= 0 && c0 + V <= a.N) {
        u32x4 w;
        __builtin_memcpy(&w, o, 16);
        if (PAST) __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(dx + c0));
        else *reinterpret_cast<u32x4*>(dx + c0) = w;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (c0 + e >= 0 && c0 + e < a.N) dx[c0 + e] = o[e];
      }
    }
  }
  if (empty) return;
  __syncthreads();
  const int64_t first = (int64_t)j0 * V - off, last = (int64_t)(j0 + jn) * V - off;
  for (int j = t; j < a.nids; j += TPB) {
    const int32_t id = sid[j];
    if (id < 0 || id < first || id >= last) continue;
    float w = 0.f;
    bool head = true;
    for (int i = 0; i < a.nids; ++i)
      if (sid[i] == id) {
        head &= i >= j;
        w += sw[i];
      }
    if (head) dx[id] = from_f32<T>(a.it * (w + grad(to_f32(x[id]))));
  }
}

// ---- host --------------------------------------------------------------------------------------
static int lp_vec(int dtype) { return dtype == RF_F32 ? 4 : 8; }

// Slices per row and chunks per slice. A slice is at most what a 1024-thread workgroup holds. A row that one
// workgroup holds is not cut, however few the rows: the join's launch costs more than the shorter slices give (uncut
// against 8 KB slices: 64 x 10000 fp32 top 50 8.7 and 13.6 us, 300 x 50265 top 20 15.0 and 21.7; the other way
// only for a row or two without alternatives, 1 x 50265 7.5 and 6.5). Rows that are joined anyway, and fewer than
// two workgroups a CU, are cut further, down to LP_MIN_CHUNKS chunks (1 x 70000: 6.4 us, 9.1 uncut, 4 x 1M bf16
// 7.3 and 11.0), as long as the join reads at most LP_JOIN entries a row (1 x 1M fp32 top 50 17.6 us, 27.9 with
// 16384; top 256 34.1 and 38.8).
constexpr int LP_CUS = 256, LP_MIN_CHUNKS = 512, LP_JOIN = 4096;
static void lp_plan(int dtype, int M, int N, int k, int* S, int* cps) {
  const int V = lp_vec(dtype);
  const int64_t nch = ((int64_t)N + 2 * V - 2) / V;  // of a row that starts anywhere in a chunk
  int64_t s = (nch + 1024 * LP_R - 1) / (1024 * LP_R);
  if (s > 1) {
    const int64_t want = std::min({(2 * LP_CUS + (int64_t)M - 1) / M, nch / LP_MIN_CHUNKS,
                                   (int64_t)LP_JOIN / std::max(k, 1)});
    s = std::max(s, want);
  }
  *cps = (int)((nch + s - 1) / s);
  *S = (int)((nch + *cps - 1) / *cps);
}

// Threads of a workgroup. One wave a row where it has a chunk a thread, or up to LP_R where rows fill the card (64
// against 256 threads, bf16 top 10: 8192 x 500 13.3 and 28.2 us, 8192 x 4000 23.7 and 30.7, 512 x 500 6.0 and
// 7.1; but 1024 x 4000 9.2 and 8.3, 64 x 2000 fp32 8.6 and 6.4); a wave's 64 maxima bound up to 32
// alternatives well. 256 threads (against 1024: 2048 x 10000 top 20 16 and 34 us, top 128 29 and 54) up to 128
// alternatives; for more their 256 maxima bound badly (2048 x 10000 top 224: 91 and 80 us, 64 x 16000 55 and 17).
static int lp_threads(const LpArgs& a) {
  if (a.S == 1 && a.k <= 32 && (a.cps <= 64 || (a.cps <= 64 * LP_R && a.M >= 2048))) return 64;
  return a.cps <= 256 * LP_R && a.k <= 128 ? 256 : 1024;
}

template <typename T, bool ENT, bool TOP, bool TEACH>
static void lp_launch(const LpArgs& a, const void* x, hipStream_t st) {
  const T* p = (const T*)x;
  const unsigned grid = (unsigned)((int64_t)a.M * a.S);
  const int tpb = lp_threads(a);
  if (tpb == 64) k_logprobs<T, 64, ENT, TOP, TEACH><<<grid, 64, 0, st>>>(a, p);
  else if (tpb == 256) k_logprobs<T, 256, ENT, TOP, TEACH><<<grid, 256, 0, st>>>(a, p);
  else k_logprobs<T, 1024, ENT, TOP, TEACH><<<grid, 1024, 0, st>>>(a, p);
  if (a.S > 1) {
    // 256 threads for short lists (1 x 100000 bf16 top 5: 10.0 us, 10.7 with 1024), 1024 for long ones (1 x 1M fp32 top
    // 50: 17.5 us, 21.6 with 256)
    if (!TOP || (a.S * a.k <= 2048 && a.k <= 64)) k_logprobs_join<T, 256, TOP, TEACH><<<a.M, 256, 0, st>>>(a, p);
    else k_logprobs_join<T, 1024, TOP, TEACH><<<a.M, 1024, 0, st>>>(a, p);
  }
}

static int lp_forward(const char* name, int dtype, const LpArgs& in, const void* logits, void* ws, hipStream_t st) {
  LpArgs a = in;
  RF_REQUIRE(dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16, "%s: bad dtype %d", name, dtype);
  RF_REQUIRE(a.M >= 0 && a.N > 0 && a.N <= LP_NMAX && a.ld >= a.N, "%s: bad shape M=%d N=%d ld=%lld", name, a.M, a.N,
             (long long)a.ld);
  RF_REQUIRE(a.it > 0.f && a.it <= LP_ITMAX, "%s: inverse temperature %g must be positive and finite", name, a.it);
  RF_REQUIRE(a.nids >= 0 && a.nids <= LP_LIST, "%s: %d entries per row (0 to %d)", name, a.nids, LP_LIST);
  RF_REQUIRE(a.k >= 0 && a.k <= LP_KMAX && a.k <= a.N, "%s: k=%d must be in [0, min(N, %d)]", name, a.k, LP_KMAX);
  if (a.M == 0) return RF_OK;
  RF_REQUIRE(logits && (a.nids == 0 || (a.ids && a.logp)) && (a.k == 0 || (a.top_logp && a.top_ids)),
             "%s: null pointer", name);
  RF_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (dtype == RF_F32 ? 3 : 1)) == 0, "%s: misaligned logits", name);
  lp_plan(dtype, a.M, a.N, a.k, &a.S, &a.cps);
  const int tpb = lp_threads(a);
  RF_REQUIRE((int64_t)a.M * a.S * tpb <= 0xFFFFFFFFll && (a.S == 1 || (int64_t)a.M * 1024 <= 0xFFFFFFFFll),
             "%s: %d rows of %d slices are too many for a launch", name, a.M, a.S);
  if (a.S > 1) {
    RF_REQUIRE(ws && (reinterpret_cast<uintptr_t>(ws) & 15) == 0, "%s: workspace missing or not 16-byte aligned", name);
    a.part = (float*)ws;
    a.pent = (uint64_t*)((char*)ws + (size_t)a.M * a.S * 16);
  }
  const bool ent = a.entropy != nullptr, top = a.k > 0;
#define LP_T(T)                                                        \
  if (a.tval) lp_launch<T, false, false, true>(a, logits, st);         \
  else if (ent && top) lp_launch<T, true, true, false>(a, logits, st); \
  else if (ent) lp_launch<T, true, false, false>(a, logits, st);       \
  else if (top) lp_launch<T, false, true, false>(a, logits, st);       \
  else lp_launch<T, false, false, false>(a, logits, st)
  if (dtype == RF_F32) { LP_T(float); }
  else if (dtype == RF_BF16) { LP_T(bf16); }
  else { LP_T(f16); }
#undef LP_T
  RF_LAUNCH_CHECK(name);
}

static int lp_backward(const char* name, int dtype, const LpBwdArgs& in, const void* logits, void* dlogits,
                       hipStream_t st) {
  LpBwdArgs a = in;
  RF_REQUIRE(dtype == RF_F32 || dtype == RF_BF16 || dtype == RF_F16, "%s: bad dtype %d", name, dtype);
  RF_REQUIRE(a.M >= 0 && a.N > 0 && a.N <= LP_NMAX && a.ld >= a.N && a.ldd >= a.N, "%s: bad shape", name);
  RF_REQUIRE(a.it > 0.f && a.it <= LP_ITMAX, "%s: inverse temperature %g must be positive and finite", name, a.it);
  RF_REQUIRE(a.nids >= 0 && a.nids <= LP_LIST, "%s: %d entries per row (0 to %d)", name, a.nids, LP_LIST);
  if (a.M == 0) return RF_OK;
  RF_REQUIRE(logits && dlogits && a.stats && (a.nids == 0 || a.ids), "%s: null pointer", name);
  const int V = lp_vec(dtype), es = dtype == RF_F32 ? 4 : 2;
  RF_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (es - 1)) == 0 &&
                 ((reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dlogits)) & 15) == 0 &&
                 (a.ld - a.ldd) % V == 0,
             "%s: the gradient's rows must be aligned as the logits' rows are", name);
  const int64_t nch = ((int64_t)a.N + 2 * V - 2) / V;
  // one wave a row where that holds it (256 threads: 8192 x 500 bf16 with 20 teacher entries 17.7 us instead of 10.9,
  // 100000 x 100 170 instead of 75)
  const int tpb = nch <= 64 * LB_R && a.nids <= 64 ? 64 : 256;
  a.S = (int)((nch + tpb * LB_R - 1) / (tpb * LB_R));
  a.cps = (int)((nch + a.S - 1) / a.S);
  RF_REQUIRE((int64_t)a.M * a.S * tpb <= 0xFFFFFFFFll, "%s: %d rows of %d slices are too many for a launch", name,
             a.M, a.S);
  const unsigned grid = (unsigned)((int64_t)a.M * a.S);
  // A gradient that the products behind it find in the caches (256 MB) is kept there, a larger one only pushes the
  // next logits out: distillation of 4915 x 50265 bf16 forward and backward 287 us, 302 through the caches, with both
  // products behind it 824 and 838, 2457 rows (247 MB) 643 and 646; but 1200 rows (121 MB) 465 and 420.
  const bool past = (int64_t)a.M * a.N * es > (int64_t)192 << 20;
#define LB_K(T, TPB, ENT)                                                                                              \
  if (past) k_logprobs_bwd<T, TPB, ENT, true><<<grid, TPB, 0, st>>>(a, (const T*)logits, (T*)dlogits);                \
  else k_logprobs_bwd<T, TPB, ENT, false><<<grid, TPB, 0, st>>>(a, (const T*)logits, (T*)dlogits)
#define LB_T(T)                                    \
  if (tpb == 64 && a.g_ent) { LB_K(T, 64, true); } \
  else if (tpb == 64) { LB_K(T, 64, false); }      \
  else if (a.g_ent) { LB_K(T, 256, true); }        \
  else { LB_K(T, 256, false); }
  if (dtype == RF_F32) { LB_T(float); }
  else if (dtype == RF_BF16) { LB_T(bf16); }
  else { LB_T(f16); }
#undef LB_T
#undef LB_K
  RF_LAUNCH_CHECK(name);
}

}  // namespace rf

using namespace rf;

extern "C" size_t rf_logprobs_workspace(int dtype, int M, int N, int k) {
  if (M <= 0 || N <= 0 || k < 0) return 0;
  int S, cps;
  lp_plan(dtype, M, N, k, &S, &cps);
  return S > 1 ? (size_t)M * S * (16 + 8 * (size_t)k) : 0;
}

extern "C" int rf_token_logprobs_fwd(int dtype, int M, int N, const void* logits, int64_t ldx, float inv_temp,
                                     const int64_t* tokens, int C, int64_t ignore_index, int k, float* logp,
                                     float* entropy, float* top_logp, int64_t* top_ids, float* stats, void* workspace,
                                     rf_stream_t stream) {
  LpArgs a{};
  a.M = M; a.N = N; a.ld = ldx; a.it = inv_temp; a.c2 = (float)((double)inv_temp * 1.4426950408889634);
  a.ids = tokens; a.nids = C; a.ignore = ignore_index; a.k = k;
  a.logp = logp; a.entropy = entropy; a.top_logp = top_logp; a.top_ids = top_ids; a.stats = stats;
  return lp_forward("rf_token_logprobs_fwd", dtype, a, logits, workspace, as_stream(stream));
}

extern "C" int rf_token_logprobs_bwd(int dtype, int M, int N, const void* logits, int64_t ldx, float inv_temp,
                                     const float* stats, const int64_t* tokens, int C, int64_t ignore_index,
                                     const float* g_logp, const float* entropy, const float* g_entropy, void* dlogits,
                                     int64_t ldd, rf_stream_t stream) {
  RF_REQUIRE(!g_entropy || entropy, "rf_token_logprobs_bwd: the entropy's gradient needs the entropy");
  LpBwdArgs a{};
  a.M = M; a.N = N; a.ld = ldx; a.ldd = ldd; a.it = inv_temp; a.c2 = (float)((double)inv_temp * 1.4426950408889634);
  a.ids = tokens; a.nids = C; a.ignore = ignore_index; a.g = g_logp; a.entropy = entropy; a.g_ent = g_entropy;
  a.stats = stats;
  return lp_backward("rf_token_logprobs_bwd", dtype, a, logits, dlogits, as_stream(stream));
}

extern "C" int rf_topk_distill_fwd(int dtype, int M, int N, const void* logits, int64_t ldx, float inv_temp,
                                   const float* teacher, const int64_t* ids, int K, float scale, float* rows,
                                   float* stats, float* loss, float* coef, void* workspace, rf_stream_t stream) {
  RF_REQUIRE(K >= 1, "rf_topk_distill_fwd: K=%d teacher entries", K);
  RF_REQUIRE(M <= 0 || (teacher && rows && stats), "rf_topk_distill_fwd: null pointer");
  RF_REQUIRE(!loss == !coef, "rf_topk_distill_fwd: loss and coef go together");
  LpArgs a{};
  a.M = M; a.N = N; a.ld = ldx; a.it = inv_temp; a.c2 = (float)((double)inv_temp * 1.4426950408889634);
  a.ids = ids; a.nids = K; a.tval = teacher; a.logp = rows; a.stats = stats;
  const int rc = lp_forward("rf_topk_distill_fwd", dtype, a, logits, workspace, as_stream(stream));
  if (rc != RF_OK || !loss) return rc;
  k_rows_mean<<<1, 1024, 0, as_stream(stream)>>>(M, rows, stats, scale, loss, coef);
  RF_LAUNCH_CHECK("rf_topk_distill_fwd");
}

extern "C" int rf_topk_distill_bwd(int dtype, int M, int N, const void* logits, int64_t ldx, float inv_temp,
                                   const float* stats, const float* teacher, const int64_t* ids, int K, const float* g,
                                   const float* coef, void* dlogits, int64_t ldd, rf_stream_t stream) {
  RF_REQUIRE(K >= 1, "rf_topk_distill_bwd: K=%d teacher entries", K);
  RF_REQUIRE(M <= 0 || (teacher && g && coef), "rf_topk_distill_bwd: null pointer");
  LpBwdArgs a{};
  a.M = M; a.N = N; a.ld = ldx; a.ldd = ldd; a.it = inv_temp; a.c2 = (float)((double)inv_temp * 1.4426950408889634);
  a.ids = ids; a.nids = K; a.tval = teacher; a.g = g; a.coef = coef; a.stats = stats;
  return lp_backward("rf_topk_distill_bwd", dtype, a, logits, dlogits, as_stream(stream));
}
