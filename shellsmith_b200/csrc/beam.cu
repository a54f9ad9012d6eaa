// Beam selection over (beams x vocabulary) and the reordering of per-sequence state rows.
//
// No reference counterpart (its sampler draws one token per request); a step of
// several beams over the same cache needs both next to the decode path.
//
// Selection. With m_k, L_k the maximum and the log of the sum of e^(x - m_k) of beam
// k's logits, the score of token v is score_k + ((x - m_k) - L_k), computed in fp32;
// the n best of all K * V scores come out by (score descending, flat index
// ascending), an order without ties. A NaN score counts as -inf. A finished beam
// offers one candidate, (pad token, score_k).
//
// B200 mapping: HBM-bound, the logits are read once. scan_kernel: a CTA streams a segment
// of one row, each warp every eighth block of 4 x 16 bytes a lane, the next block's loads
// in flight while one is summed. Every lane keeps its own running maximum and sum. Beside
// them the CTA keeps a list of granules (16 bytes of logits), to which its warps add
// without waiting for one another: those whose maximum is not below a bound that n + 1
// logits have reached, so that most granules cost their maximum and one comparison. A
// warp starts with the (n + 1)-th largest of its first block's 128 maxima; whenever the
// list has grown, the warp that notices takes the (n + 1)-th largest maximum of its newest
// entries as the next bound. Both bisect over order-preserving integer keys by ballots. At
// the segment's end the listed granules' logits are cut to the n + 1 largest. Within a row
// the score is monotone in the logit, so no other logit can be among the n best, save by
// the rounding of scores below. merge_kernel, one CTA per group: the rows' statistics, the
// scores of all segments' candidates, a threshold over them in the same way, and the rank
// of each survivor.
//
// Equal logits: of the granules whose maximum equals a warp's first bound its first block
// keeps the n + 1 of lowest index and later blocks, whose indices are higher, none, so a
// row masked with one value costs nothing. A list that overflows all the same (long runs
// of one large value; eight warps' n + 1 first granules from n = 64 on, with the refreshes
// from about 30 on in long segments) is made anew from the logits, tile by tile in index
// order (ordered_list), exact but slow: 32 groups of 8 over 250,001 52 us with n = 16, 510 to 593 with 32 to
// 64; 8 of 5 over 50,001 fp32 20, 31 and 167 with 16, 32 and 64 (nothing finished).
//
// ex2.approx (two units in the last place) makes the terms of the sums, which are fp32: the
// score's error against 64 bits stays at an fp32 rounding's (3.4e-8 where a plain form in
// fp32 has 3.5e-8, at worst 2.8e-8 where it has 2.4e-8).
//
// Scores of different logits can round to the same fp32 number (a large |score_k|),
// and then the lower index wins even against a larger logit. A segment's dropped logits
// are at most its last kept one t, and one equal to t has a higher index; if the next
// value below t still scores as much as the n-th best, merge_kernel rescans the group's
// logits for scores equal to it, in index order, until it has enough.
//
// Measured (B200): 32 groups of 8 beams over 250,001 bf16 tokens, a fifth of the rows
// finished (106 MB), 38.5 us, 2.8 TB/s: the scan's 18.6 million warp instructions fill 60 %
// of the issue slots and its exponentials 43 % of their unit, while DRAM is 39 % busy. No
// unit is full: its time is the chains of dependent steps, not memory (three bulk-copied
// blocks a warp in flight instead of the one in registers took 43.2 us). 8 groups of 5 over
// 50,001 fp32 tokens 14.1 us, 1 of 4 over 32,768 9.9 us: two launches, a block's bound and the merge.
#include <math_constants.h>

#include <algorithm>

#include "common.cuh"

namespace sc {
namespace {

constexpr int kScanThreads = 256;
constexpr int kMergeThreads = 256;
constexpr int kMaxSelect = 64;       // n
constexpr int kScanWarps = kScanThreads / 32;
constexpr int kVecs = 4;             // 16-byte loads of a lane per block
// Candidates of a segment. ordered_list leaves up to 2 (n + 1) before it cuts, and a tile
// then appends up to a granule's logits (8 at most) a thread.
constexpr int kScanList = 2 * (kMaxSelect + 1) + kScanThreads * 8;
// Segments per SM: the case of 256 rows above took 38.5 us with 4, 48 with 2 and 47 with 8.
constexpr int kSegWaves = 4;
constexpr int kGranules = 512;       // listed granules
constexpr int kNewest = 128;         // list entries that make a bound
constexpr int kRankList = 256;       // lists up to here are ranked in one go
constexpr int kMergeCache = 4096;    // candidates whose keys merge_kernel keeps
constexpr int kMergeList = 1024;
constexpr int kMergeAhead = 4;       // items of a thread that are loaded at once
constexpr int kMaxBeams = 64;

// Order-preserving unsigned keys of finite values and +inf; 0 for -inf and NaN.
__device__ __forceinline__ uint32_t score_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 -> +0
  const uint32_t k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return x > -CUDART_INF_F ? k : 0u;  // false for NaN
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct Logits;
template <>
struct Logits<uint16_t> {  // bf16
  static constexpr int kPerVec = 8;
  static constexpr int kBits = 16;  // significant high bits of a key
  using Top = __nv_bfloat162;  // the maxima of a granule's even and odd logits
  __device__ static Top tops(const uint4& u) {  // NaN only where all are
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    return __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  }
  __device__ static Top join_tops(Top a, Top b) { return __hmax2(a, b); }
  __device__ static float largest(Top t) { return fmaxf(__low2float(t), __high2float(t)); }
  // x + shift of a pair of logits, in fp32.
  __device__ static uint64_t shifted(const uint4& u, int e, float shift) {
    const uint32_t w = e < 2 ? u.x : e < 4 ? u.y : e < 6 ? u.z : u.w;
    float lo, hi;
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "add.rn.f32.bf16 %0, a, %3;\n\t"
        "add.rn.f32.bf16 %1, b, %3;\n\t}"
        : "=f"(lo), "=f"(hi)
        : "r"(w), "f"(shift));
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
    return p;
  }
  __device__ static float value(uint16_t x) { return bf16_to_f(x); }
  __device__ static float get(const uint4& u, int e) {
    const uint32_t w = e < 2 ? u.x : e < 4 ? u.y : e < 6 ? u.z : u.w;
    return (e & 1) ? bf16_hi(w) : bf16_lo(w);
  }
  __device__ static uint4 fill() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  __device__ static void put(uint4& u, int e, uint16_t x) {
    uint32_t& w = e < 2 ? u.x : e < 4 ? u.y : e < 6 ? u.z : u.w;
    w = (e & 1) ? (w & 0xffffu) | ((uint32_t)x << 16) : (w & 0xffff0000u) | x;
  }
  // A bf16's key keeps its high 16 bits: the low ones of a negative value's would be set.
  __device__ static uint32_t key(float x) { return score_key(x) & 0xffff0000u; }
  __device__ static float unkey(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fff0000u) : (~k & 0xffff0000u));
  }
  __device__ static float below(float x) { return unkey(key(x) - 0x10000u); }  // the next value
};
template <>
struct Logits<float> {
  static constexpr int kPerVec = 4;
  static constexpr int kBits = 32;
  using Top = float;
  __device__ static Top tops(const uint4& u) {
    return fmaxf(fmaxf(get(u, 0), get(u, 1)), fmaxf(get(u, 2), get(u, 3)));
  }
  __device__ static Top join_tops(Top a, Top b) { return fmaxf(a, b); }
  __device__ static float largest(Top t) { return t; }
  __device__ static uint64_t shifted(const uint4& u, int e, float shift) {
    uint64_t p;
    asm("{\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %2};\n\t"
        "mov.b64 b, {%3, %3};\n\t"
        "add.rn.f32x2 %0, a, b;\n\t}"
        : "=l"(p)
        : "f"(get(u, e)), "f"(get(u, e + 1)), "f"(shift));
    return p;
  }
  __device__ static float value(float x) { return x; }
  __device__ static float get(const uint4& u, int e) {
    return __uint_as_float(e == 0 ? u.x : e == 1 ? u.y : e == 2 ? u.z : u.w);
  }
  __device__ static uint4 fill() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  __device__ static void put(uint4& u, int e, float x) {
    uint32_t& w = e == 0 ? u.x : e == 1 ? u.y : e == 2 ? u.z : u.w;
    w = __float_as_uint(x);
  }
  __device__ static uint32_t key(float x) { return score_key(x); }
  __device__ static float unkey(uint32_t k) { return key_value(k); }
  __device__ static float below(float x) { return unkey(key(x) - 1u); }
};

// Two fp32 lanes in one register pair: one instruction for two sums or products.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ void unpair(uint64_t p, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// (max, sum of e^(x - max)) of two disjoint sets. A NaN sum stays NaN; a set whose
// maximum is -inf is empty unless its sum is NaN.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float M = fmaxf(m, m2);
  const float a = s == 0.f ? 0.f : (m == M ? s : s * expf(m - M));
  const float b = s2 == 0.f ? 0.f : (m2 == M ? s2 : s2 * expf(m2 - M));
  m = M;
  s = a + b;
}

// Cuts the CTA's list (unsorted, `total` > `want` entries) to its `want` largest keys,
// equal ones by the lower index, in place; returns the smallest key left. The key by
// bisection; of a run of equal ones as many as fit stay, the lowest indices first.
template <int kBits>
__device__ uint32_t cut_list(uint32_t* list_k, int* list_v, int total, int want, int* scratch) {
  uint32_t cut = 0u;
#pragma unroll 1
  for (int b = 31; b >= 32 - kBits; --b) {
    const uint32_t next = cut | (1u << b);
    int c = 0;
    for (int i = threadIdx.x; i < total; i += kScanThreads) c += list_k[i] >= next;
    c = __reduce_add_sync(0xffffffffu, c);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = c;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < kScanThreads / 32; ++w) all += scratch[w];
    if (all >= want) cut = next;
    __syncthreads();
  }
  constexpr int kMost = (kScanList + kScanThreads - 1) / kScanThreads;
  uint32_t k[kMost];
  int v[kMost];
  uint32_t keep = 0u;
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    const int i = threadIdx.x + j * kScanThreads;
    k[j] = i < total ? list_k[i] : 0u;
    v[j] = i < total ? list_v[i] : 0;
    if (i >= total || k[j] < cut) continue;
    int before = 0;
    if (k[j] == cut)
      for (int o = 0; o < total; ++o)
        before += list_k[o] > cut || (list_k[o] == cut && list_v[o] < v[j]);
    if (before < want) keep |= 1u << j;
  }
  __syncthreads();
  if (threadIdx.x == 0) scratch[0] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kMost; ++j)
    if (keep >> j & 1u) {
      const int at = atomicAdd(&scratch[0], 1);
      list_k[at] = k[j];
      list_v[at] = v[j];
    }
  __syncthreads();
  return cut;
}

struct SelectArgs {
  const void* logits;
  long long row_stride;          // elements between rows
  const float* scores;           // [G, K]
  const uint8_t* finished;       // [G, K] or NULL
  float2* stats;                 // [rows][segs] (max, sum)
  float* floors;                 // [rows][segs] last kept logit where some were dropped, else -inf
  uint2* kept;                   // [rows][segs][n + 1] (logit bits, token), -inf: none
  float* out_scores;             // [G, n]
  int32_t *parents, *tokens;
  int G, K, V, n, segs, seg_blocks, pad;
};

// A row that offers no logit: finished, or its score is -inf or NaN.
__device__ __forceinline__ bool row_idle(const SelectArgs& a, int row) {
  return (a.finished != nullptr && a.finished[row]) || !(a.scores[row] > -CUDART_INF_F);
}

// One of the warp's keys that at least `want` of them reach: the want-th largest, but for
// at most 1/1024 of their span (which a bound may be below). 0 if fewer keys than that are
// not 0. A lane holds kPer of them.
template <int kPer>
__device__ __forceinline__ uint32_t warp_nth(const uint32_t* k, int want) {
  constexpr unsigned kAll = 0xffffffffu;
  uint32_t hi = 0u, lo = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    hi = max(hi, k[i]);
    lo = k[i] != 0u ? min(lo, k[i]) : lo;
  }
  hi = __reduce_max_sync(kAll, hi);
  lo = __reduce_min_sync(kAll, lo);
  const auto reach = [&](uint32_t t) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) c += k[i] >= t;
    return (int)__reduce_add_sync(kAll, (unsigned)c);
  };
  if (reach(1u) < want) return 0u;
  if (reach(hi) >= want) return hi;
  uint32_t step = hi - lo;  // at least want keys reach lo, fewer reach lo + step
#pragma unroll 1
  for (int i = 0; i < 10 && step > 1u; ++i) {
    const uint32_t half = step >> 1;
    if (reach(lo + half) >= want) {
      lo += half;
      step -= half;
    } else {
      step = half;
    }
  }
  uint32_t t = 0xffffffffu;  // the smallest key that reaches it, an actual one
#pragma unroll
  for (int i = 0; i < kPer; ++i) t = k[i] >= lo ? min(t, k[i]) : t;
  return __reduce_min_sync(kAll, t);
}

// (m, s) of the warp's lanes joined: one maximum, one rescaling and one sum.
__device__ __forceinline__ void warp_join(float& m, float& s) {
  constexpr unsigned kAll = 0xffffffffu;
  const uint32_t b = __float_as_uint(m);
  const uint32_t top = __reduce_max_sync(kAll, (b & 0x80000000u) ? ~b : (b | 0x80000000u));
  const float M = key_value(top);
  // An empty lane (s = 0) stays 0; a lane at the maximum is not rescaled (inf - inf).
  s = s == 0.f || m == M ? s : s * expf(m - M);
  m = M;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(kAll, s, off);
}

// The candidates of granules [g_begin, g_end) in index order, the CTA in step: a tile of a
// granule a thread at a time, the list cut whenever a tile might not fit. Returns its
// length (at least min(want, candidates); cut_list does the rest).
template <typename T>
__device__ __noinline__ int ordered_list(const T* base, int lead, int V, int g_begin, int g_end,
                                         uint32_t* list_k, int* list_v, int want, int* scratch,
                                         int* n_list) {
  using L = Logits<T>;
  constexpr int E = L::kPerVec;
  static_assert(kScanList >= 2 * (kMaxSelect + 1) + kScanThreads * E, "a tile past the last cut");
  if (threadIdx.x == 0) *n_list = 0;
  __syncthreads();
  uint32_t bound = 0u;
  for (int g0 = g_begin; g0 < g_end; g0 += kScanThreads) {
    const int v0 = (g0 + (int)threadIdx.x) * E - lead;
    uint32_t k[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      k[e] = g0 + (int)threadIdx.x < g_end && v0 + e >= 0 && v0 + e < V ? L::key(L::value(base[v0 + e]))
                                                                       : 0u;
    // Every thread has read the count before one appends: the branch holds barriers, and a
    // warp that came late would see what the early ones appended.
    const int total = *n_list;
    __syncthreads();
    if (total > 2 * want) {  // uniform
      bound = max(bound, cut_list<L::kBits>(list_k, list_v, total, want, scratch));
      if (threadIdx.x == 0) *n_list = want;
      __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (k[e] > bound) {
        const int at = atomicAdd(n_list, 1);
        list_k[at] = k[e];
        list_v[at] = v0 + e;
      }
    __syncthreads();
  }
  return *n_list;
}

// Three CTAs an SM: the case of 256 rows above took 38.5 us, with four (64 registers) 44.8.
template <typename T>
__global__ void __launch_bounds__(kScanThreads, 3) scan_kernel(const SelectArgs a) {
  using L = Logits<T>;
  constexpr int E = L::kPerVec;
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr unsigned kAll = 0xffffffffu;
  constexpr int kBlock = 32 * kVecs;  // granules of a warp's block
  __shared__ uint4 gran[kGranules];          // listed granules, their first element's index
  __shared__ int gran_v[kGranules];          // and the key of their maximum
  __shared__ uint32_t gran_k[kGranules];
  __shared__ uint32_t list_k[kScanList];
  __shared__ int list_v[kScanList];
  __shared__ uint32_t shared_bound;          // n + 1 logits of the segment reach it
  __shared__ int n_gran, n_list, refresh_at;
  __shared__ float red_m[kScanWarps], red_s[kScanWarps];
  __shared__ int scratch[kScanWarps];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.y, want = a.n + 1;
  const size_t seg = (size_t)row * a.segs + blockIdx.x;
  // Aligned 16-byte granules over the row; the first and the last may hold elements
  // outside it, which are read one by one.
  const T* base = reinterpret_cast<const T*>(a.logits) + (long long)row * a.row_stride;
  const int lead = (int)((reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T));
  const T* start = base - lead;  // granule g covers elements E g - lead .. of the row
  const int granules = (a.V + lead + E - 1) / E;
  const int g_begin = (int)blockIdx.x * a.seg_blocks * kScanWarps * kBlock;
  const int g_end = min(granules, g_begin + a.seg_blocks * kScanWarps * kBlock);
  int g0 = g_begin + warp * kBlock + lane;
  const auto load = [&](int g, uint4* r) {
    if (g - lane + kBlock <= g_end && (g - lane) * E - lead >= 0 &&
        (g - lane + kBlock) * E - lead <= a.V) {  // uniform: a whole block
#pragma unroll
      for (int j = 0; j < kVecs; ++j)
        r[j] = __ldcs(reinterpret_cast<const uint4*>(start) + g + 32 * j);
    } else {
#pragma unroll
      for (int j = 0; j < kVecs; ++j) {
        const int gj = g + 32 * j, v0 = gj * E - lead;
        r[j] = L::fill();
        if (gj < g_end)
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (v0 + e >= 0 && v0 + e < a.V) L::put(r[j], e, base[v0 + e]);
      }
    }
  };
  constexpr int kRound = kScanWarps * kBlock;
  uint4 r[kVecs], next[kVecs];
  load(g0, r);  // before the row's flags are known, which takes as long
  if (row_idle(a, row)) return;  // uniform over the CTA; merge_kernel skips the row too
  for (int i = tid; i < kGranules; i += kScanThreads) gran_k[i] = 0u;  // 0: not written yet
  if (tid == 0) {
    shared_bound = 0u;
    n_gran = n_list = 0;
    refresh_at = 2 * want;
  }
  __syncthreads();
  // This lane's maximum and the sum of e^(x - m). x - m comes before the change of base: a
  // product with log2 e would add its rounding to the largest terms (and overflow at the
  // type's ends).
  float m = -CUDART_INF_F, s = 0.f;
  float own = -CUDART_INF_F;  // this warp's first bound: later granules count above it
  bool first = true;
#pragma unroll 1
  for (; g0 - lane < g_end; g0 += kRound) {
    load(g0 + kRound, next);
    typename L::Top tops[kVecs];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) tops[j] = L::tops(r[j]);
    const float all = L::largest(L::join_tops(L::join_tops(tops[0], tops[1]),
                                              L::join_tops(tops[2], tops[3])));
    static_assert(kVecs == 4, "joined above");
    const auto top = [&](int j) { return L::largest(tops[j]); };
    if (all > m) {
      s *= m == -CUDART_INF_F ? 1.f : ex2((m - all) * kLog2e);  // a NaN sum stays
      m = all;
    }
    const float shift = m == -CUDART_INF_F ? 0.f : -m;
    uint64_t sums[2] = {pair(s, 0.f), pair(0.f, 0.f)};
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float y0, y1;
        unpair(mul2(L::shifted(r[j], e, shift), pair(kLog2e, kLog2e)), y0, y1);
        sums[e / 2 % 2] = add2(sums[e / 2 % 2], pair(ex2(y0), ex2(y1)));
      }
    float s0, s1;
    unpair(add2(sums[0], sums[1]), s0, s1);
    s = s0 + s1;
    unsigned hot = 0u;  // granules of this lane that go on the list
    if (!first) {
      const uint32_t least_k = *reinterpret_cast<volatile uint32_t*>(&shared_bound);
      const float least = least_k == 0u ? -CUDART_INF_F : L::unkey(least_k);
      if (__any_sync(kAll, all > own && all >= least)) {
#pragma unroll
        for (int j = 0; j < kVecs; ++j) hot |= (top(j) > own && top(j) >= least) ? 1u << j : 0u;
      }
    } else {
      first = false;
      uint32_t k[kVecs];
#pragma unroll
      for (int j = 0; j < kVecs; ++j) k[j] = L::key(top(j));
      const uint32_t t = warp_nth<kVecs>(k, want);
      if (t != 0u) own = L::unkey(t);
      if (lane == 0) atomicMax(&shared_bound, t);
      int equals = 0;
#pragma unroll
      for (int j = 0; j < kVecs; ++j) {
        const unsigned eq = __ballot_sync(kAll, k[j] == t && t != 0u);
        const int rank = equals + __popc(eq & ((1u << lane) - 1u));
        hot |= (k[j] > t || ((eq >> lane & 1u) && rank < want)) ? 1u << j : 0u;
        equals += __popc(eq);
      }
    }
    if (__any_sync(kAll, hot != 0u)) {
      if (hot != 0u) {
        int at = atomicAdd(&n_gran, __popc(hot));
#pragma unroll
        for (int j = 0; j < kVecs; ++j)
          if (hot >> j & 1u) {
            if (at < kGranules) {  // an overflow is seen at the end
              gran[at] = r[j];
              gran_v[at] = (g0 + 32 * j) * E - lead;
              gran_k[at] = L::key(top(j));
            }
            ++at;
          }
      }
      // Has the list grown enough for a better bound, and is it this warp that makes it? (Every
      // n + 1 entries; every 2 (n + 1): 39.5 us instead of 38.4.)
      int now = 0;
      if (lane == 0) {
        now = *reinterpret_cast<volatile int*>(&n_gran);
        const int due = *reinterpret_cast<volatile int*>(&refresh_at);
        if (now < due || atomicCAS(&refresh_at, due, now + want) != due) now = 0;
      }
      now = min(__shfl_sync(kAll, now, 0), kGranules);
      if (now != 0) {
        uint32_t k[kNewest / 32];
#pragma unroll
        for (int i = 0; i < kNewest / 32; ++i) {
          const int at = now - 1 - lane - 32 * i;
          k[i] = at >= 0 ? *reinterpret_cast<volatile uint32_t*>(&gran_k[at]) : 0u;
        }
        const uint32_t t = warp_nth<kNewest / 32>(k, want);
        if (lane == 0) atomicMax(&shared_bound, t);
      }
    }
#pragma unroll
    for (int j = 0; j < kVecs; ++j) r[j] = next[j];
  }
  warp_join(m, s);
  if (lane == 0) {
    red_m[warp] = m;
    red_s[warp] = s;
  }
  __syncthreads();
  // The listed granules' logits that are not below the last bound.
  const int grans = n_gran;
  const uint32_t least = max(shared_bound, 1u);
  for (int i = tid; i < min(grans, kGranules); i += kScanThreads) {
    if (gran_k[i] < least) continue;
    const uint4 g = gran[i];
    uint32_t key[E];
    unsigned hits = 0u;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      key[e] = L::key(L::get(g, e));
      hits |= key[e] >= least ? 1u << e : 0u;
    }
    int at = atomicAdd(&n_list, __popc(hits));
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (hits >> e & 1u) {
        if (at < kScanList) {
          list_k[at] = key[e];
          list_v[at] = gran_v[i] + e;
        }
        ++at;
      }
  }
  __syncthreads();
  int total = n_list;
  __syncthreads();
  if (grans > kGranules || total > kScanList)
    total = ordered_list(base, lead, a.V, g_begin, g_end, list_k, list_v, want, scratch, &n_list);
  if (total > kRankList) {
    cut_list<L::kBits>(list_k, list_v, total, want, scratch);
    total = want;
  }
  // One entry a thread, ranked by counting the better ones; the n + 1 best go out in order.
  uint2* kept = a.kept + seg * want;
  const uint32_t key = tid < total ? list_k[tid] : 0u;
  const int v = tid < total ? list_v[tid] : 0;
  if (tid < total) {
    int rank = 0;
#pragma unroll 4
    for (int o = 0; o < total; ++o) {
      const uint32_t ko = list_k[o];
      rank += ko > key || (ko == key && list_v[o] < v);
    }
    if (rank < want) kept[rank] = make_uint2(__float_as_uint(L::unkey(key)), (uint32_t)v);
    // Where logits were dropped at all, n + 1 are left, and none dropped is above the last.
    if (rank == a.n) a.floors[seg] = L::unkey(key);
  }
  for (int i = total + tid; i < want; i += kScanThreads) kept[i] = make_uint2(0xff800000u, 0u);
  if (total < want && tid == 0) a.floors[seg] = -CUDART_INF_F;
  if (warp == kScanWarps - 1) {
    m = lane < kScanWarps ? red_m[lane] : -CUDART_INF_F;
    s = lane < kScanWarps ? red_s[lane] : 0.f;
    warp_join(m, s);
    if (lane == 0) a.stats[seg] = make_float2(m, s);
  }
}

// Sum of c over the CTA.
__device__ __forceinline__ int block_total(int c, int* scratch) {
  c = __reduce_add_sync(0xffffffffu, c);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = c;
  __syncthreads();
  int all = 0;
  for (int w = 0; w < kMergeThreads / 32; ++w) all += scratch[w];
  __syncthreads();
  return all;
}

template <typename T>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const SelectArgs a) {
  using L = Logits<T>;
  __shared__ float row_m[kMaxBeams], row_l[kMaxBeams], row_s[kMaxBeams];
  __shared__ bool row_on[kMaxBeams];
  __shared__ unsigned long long cache[kMergeCache], list[kMergeList];
  __shared__ int scratch[kMergeThreads / 32];
  __shared__ int n_list, ambiguous, strictly;
  __shared__ uint32_t last_score, threshold, best_k[kMergeThreads];
  pdl_wait();
  pdl_trigger();
  const int g = blockIdx.x, K = a.K, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) n_list = ambiguous = strictly = 0, last_score = 0u;
  // Items: the segments' candidates, then one per beam for the finished ones. A thread's
  // first ones and its first floor are loaded beside the rows' statistics; those of an idle
  // row are not used.
  const int per = a.n + 1, segs = K * a.segs, cands = segs * per, items = cands + K;
  const uint2* kept = a.kept + (size_t)g * cands;
  const float* floors = a.floors + (size_t)g * segs;
  uint2 ahead[kMergeAhead];
#pragma unroll
  for (int x = 0; x < kMergeAhead; ++x) {
    const int i = threadIdx.x + x * kMergeThreads;
    ahead[x] = i < cands ? kept[i] : make_uint2(0u, 0u);
  }
  const float floor_ahead = (int)threadIdx.x < segs ? floors[threadIdx.x] : 0.f;
  for (int k = warp; k < K; k += kMergeThreads / 32) {
    const int row = g * K + k;
    float m = -CUDART_INF_F, s = 0.f;
    const float2* stats = a.stats + (size_t)row * a.segs;
    const float2 st0 = lane < a.segs ? stats[lane] : make_float2(m, s);
    const bool on = !row_idle(a, row);
    if (on) {
      join(m, s, st0.x, st0.y);
      for (int c = lane + 32; c < a.segs; c += 32) {
        const float2 st = stats[c];
        join(m, s, st.x, st.y);
      }
    }
    warp_join(m, s);
    if (lane == 0) {
      row_m[k] = m;
      row_l[k] = logf(s);
      row_s[k] = a.scores[row];
      row_on[k] = on;
    }
  }
  __syncthreads();
  const auto score = [&](int k, float x) { return row_s[k] + ((x - row_m[k]) - row_l[k]); };
  // (score, lower index first) as one key; 0 for -inf and NaN.
  const auto full_key = [&](int k, float sc, int v) -> unsigned long long {
    const uint32_t key = score_key(sc);
    return key == 0u ? 0ull
                     : ((unsigned long long)key << 32) | (0xffffffffu - ((uint32_t)k * a.V + v));
  };
  const auto keyed = [&](int i, uint2 c) -> unsigned long long {
    if (i >= cands) {
      const int k = i - cands;
      const bool fin = a.finished != nullptr && a.finished[g * K + k];
      return fin ? full_key(k, row_s[k], a.pad) : 0ull;
    }
    const int k = i / (a.segs * per);
    return row_on[k] ? full_key(k, score(k, __uint_as_float(c.x)), (int)c.y) : 0ull;
  };
  const auto make = [&](int i) { return keyed(i, i < cands ? kept[i] : make_uint2(0u, 0u)); };
  const bool cached = items <= kMergeCache;
  unsigned long long best = 0ull;
  const auto see = [&](int i, unsigned long long key) {
    if (cached) cache[i] = key;
    best = key > best ? key : best;
  };
#pragma unroll
  for (int x = 0; x < kMergeAhead; ++x) {
    const int i = threadIdx.x + x * kMergeThreads;
    if (i < items) see(i, keyed(i, ahead[x]));
  }
  for (int i = threadIdx.x + kMergeAhead * kMergeThreads; i < items; i += kMergeThreads)
    see(i, make(i));
  const auto item = [&](int i) { return cached ? cache[i] : make(i); };  // own items only
  // At least n items reach about the n-th largest of the threads' best scores.
  best_k[threadIdx.x] = (uint32_t)(best >> 32);
  __syncthreads();
  if (warp == 0) {
    uint32_t k[kMergeThreads / 32];
#pragma unroll
    for (int i = 0; i < kMergeThreads / 32; ++i) k[i] = best_k[lane + 32 * i];
    const uint32_t bound = warp_nth<kMergeThreads / 32>(k, a.n);
    if (lane == 0) threshold = bound;
  }
  __syncthreads();
  const uint32_t t = threshold;
  unsigned long long floor_key = (unsigned long long)t << 32;
  int c = 0;
  if (best >= floor_key)
    for (int i = threadIdx.x; i < items; i += kMergeThreads) {
      const unsigned long long key = item(i);
      if (key != 0ull && key >= floor_key) {
        const int at = atomicAdd(&n_list, 1);
        if (at < kMergeList) list[at] = key;
      }
    }
  __syncthreads();
  if (n_list > kMergeList) {  // the n largest keys exactly
    floor_key = 0ull;
    for (int b = 63; b >= 0; --b) {
      const unsigned long long next = floor_key | (1ull << b);
      c = 0;
      for (int i = threadIdx.x; i < items; i += kMergeThreads) c += item(i) >= next;
      if (block_total(c, scratch) >= a.n) floor_key = next;
    }
    if (threadIdx.x == 0) n_list = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < items; i += kMergeThreads) {
      const unsigned long long key = item(i);
      if (key != 0ull && key >= floor_key) list[atomicAdd(&n_list, 1)] = key;
    }
    __syncthreads();
  }
  const int total = n_list;
  float* os = a.out_scores + (size_t)g * a.n;
  int32_t* op = a.parents + (size_t)g * a.n;
  int32_t* ot = a.tokens + (size_t)g * a.n;
  const auto emit = [&](int rank, float sc, uint32_t flat) {
    os[rank] = sc;
    op[rank] = (int32_t)(flat / (uint32_t)a.V);
    ot[rank] = (int32_t)(flat % (uint32_t)a.V);
  };
  for (int i = threadIdx.x; i < total; i += kMergeThreads) {
    const unsigned long long key = list[i];
    int rank = 0;
    for (int o = 0; o < total; ++o) rank += list[o] > key;
    if (rank < a.n) emit(rank, key_value((uint32_t)(key >> 32)), 0xffffffffu - (uint32_t)key);
    if (rank == a.n - 1) last_score = (uint32_t)(key >> 32);
  }
  __syncthreads();
  const uint32_t last = last_score;
  if (total < a.n) {
    // Every finite candidate is out; the rest are -inf, lowest index first.
    if (threadIdx.x == 0) {
      uint32_t flat = 0;
      for (int rank = total; rank < a.n; ++flat) {
        bool taken = false;
        for (int i = 0; i < total; ++i) taken |= 0xffffffffu - (uint32_t)list[i] == flat;
        if (!taken) emit(rank++, -CUDART_INF_F, flat);
      }
    }
    return;
  }
  // A dropped logit that rounds to the n-th best score may have a lower index.
  for (int sgm = threadIdx.x; sgm < segs; sgm += kMergeThreads) {
    const int k = sgm / a.segs;
    if (!row_on[k]) continue;
    const float fl = sgm < kMergeThreads ? floor_ahead : floors[sgm];
    if (fl > -CUDART_INF_F && score_key(score(k, L::below(fl))) >= last) ambiguous = 1;
  }
  for (int i = threadIdx.x; i < total; i += kMergeThreads)
    if ((uint32_t)(list[i] >> 32) > last) atomicAdd(&strictly, 1);
  __syncthreads();
  if (!ambiguous) return;
  const float target = key_value(last);
  int have = strictly;
  for (int k = 0; k < K && have < a.n; ++k) {
    const int row = g * K + k;
    if (!row_on[k]) {
      const bool fin = a.finished != nullptr && a.finished[row];
      if (fin && row_s[k] == target) {
        if (threadIdx.x == 0) emit(have, target, (uint32_t)k * a.V + a.pad);
        ++have;
      }
      continue;
    }
    const T* base = reinterpret_cast<const T*>(a.logits) + (long long)row * a.row_stride;
    for (int v0 = 0; v0 < a.V && have < a.n; v0 += kMergeThreads) {
      const int v = v0 + threadIdx.x;
      const bool hit = v < a.V && score(k, L::value(base[v])) == target;
      const unsigned mask = __ballot_sync(0xffffffffu, hit);
      if (lane == 0) scratch[warp] = __popc(mask);
      __syncthreads();
      int at = have + __popc(mask & ((1u << lane) - 1u)), sum = 0;
      for (int w = 0; w < kMergeThreads / 32; ++w) {
        if (w < warp) at += scratch[w];
        sum += scratch[w];
      }
      if (hit && at < a.n) emit(at, target, (uint32_t)k * a.V + v);
      have += sum;
      __syncthreads();
    }
  }
}

// Segments of a row, in whole rounds of blocks (one a warp): as many as the GPU holds at
// once, so that every segment is long and its first bound and its end pay.
struct Segments {
  int blocks, count;  // rounds of blocks per segment, segments per row
};
template <typename T>
Segments select_segments(long long rows, int V) {
  const int per = kScanThreads * kVecs * Logits<T>::kPerVec;
  const int rounds = (int)(((long long)V + Logits<T>::kPerVec - 1 + per - 1) / per);  // + the lead
  const long long most = 148ll * kSegWaves / rows;
  Segments s;
  s.blocks = most >= rounds ? 1 : (int)((rounds + (most < 1 ? 1 : most) - 1) / (most < 1 ? 1 : most));
  s.count = (rounds + s.blocks - 1) / s.blocks;
  return s;
}

// ---------------------------------------------------------------- reordering of rows
// Child j of group g continues beam parents[g][j]. The first child of a beam keeps the
// beam's slot; each later child takes the slot of a beam without children, in ascending
// order of both. A slot that is read is never written, so the copies run in place and
// in any order.
//
// One launch: every CTA makes the whole plan for itself (a warp a group, beams as 64-bit
// masks; a few hundred cycles) and then takes its share of the places to copy, a place
// being one source's 32 KB piece of a layer, read once and written to each of its
// destinations. Larger batches make the plan in slices that fit shared memory.
constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 8;       // 16-byte loads in flight per thread
constexpr int kPlanBeams = 1024;   // beams planned at once

struct ReorderPools {
  uint8_t* base[4];
  long long chunks[4];  // 16-byte chunks per row
  long long first[5];   // pieces before pool p, of one row
  int count;
};

__global__ void __launch_bounds__(kCopyThreads)
    reorder_kernel(const __grid_constant__ ReorderPools pools, const int32_t* __restrict__ slots,
                   const int32_t* __restrict__ parents, int32_t* __restrict__ new_slots, int G,
                   int K, int rows, unsigned int* status) {
  constexpr unsigned kAll = 0xffffffffu;
  constexpr int kUnit = kCopyThreads * kCopyVecs;
  // Per copied source, at K / 2 places a group: its row, where its destinations start and
  // how many there are. `order` lists the places in use, in the same order in every CTA.
  __shared__ int src_row[kPlanBeams / 2], src_at[kPlanBeams / 2], src_n[kPlanBeams / 2];
  __shared__ int dst_row[kPlanBeams], in_group[kPlanBeams], order[kPlanBeams / 2];
  __shared__ int n_src;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const uint64_t beams = K == 64 ? ~0ull : (1ull << K) - 1ull;
  const int slice = kPlanBeams / K;  // groups planned at once
  const bool writes = blockIdx.x == 0;
  for (int g0 = 0; g0 < G; g0 += slice) {
    for (int g = g0 + (threadIdx.x >> 5); g < min(G, g0 + slice); g += kCopyThreads / 32) {
      const int32_t* mine = slots + (size_t)g * K;
      int p[2], slot[2], own[2];
      uint64_t used = 0, later = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = lane + 32 * i;
        p[i] = j < K ? parents[(size_t)g * K + j] : -1;
        own[i] = j < K ? mine[j] : -1;  // beam j's own row
        const bool ok = p[i] >= 0 && p[i] < K;
        if (j < K && !ok && writes) flag_device(status, DEV_BAD_INDEX);
        // A child is a later one if its beam has a child among the lower lanes or, in the
        // second round, among the first 32.
        const unsigned same = __match_any_sync(kAll, ok ? p[i] : -1);
        const bool again = ok && ((same & ((1u << lane) - 1u)) != 0u || (used >> p[i] & 1ull));
        later |= (uint64_t)__ballot_sync(kAll, again) << (32 * i);
        const uint64_t bit = ok ? 1ull << p[i] : 0ull;
        used |= (uint64_t)__reduce_or_sync(kAll, (unsigned)bit) |
                ((uint64_t)__reduce_or_sync(kAll, (unsigned)(bit >> 32)) << 32);
      }
      const uint64_t dead = beams & ~used;
      const auto row_of = [&](int b) {  // all lanes; b in [0, 64)
        const int lo = __shfl_sync(kAll, own[0], b & 31), hi = __shfl_sync(kAll, own[1], b & 31);
        return b < 32 ? lo : hi;
      };
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = lane + 32 * i;
        const bool ok = p[i] >= 0 && p[i] < K;
        const bool copy = later >> j & 1ull;
        const int src = row_of(ok ? p[i] : 0);
        uint64_t d = dead;  // as many beams without children as later children, at least
        if (copy)
          for (int skip = __popcll(later & ((1ull << j) - 1ull)); skip > 0; --skip) d &= d - 1;
        const int to = row_of(copy && d != 0 ? __ffsll(d) - 1 : 0);
        slot[i] = !ok ? -1 : copy ? to : src;
        const bool bad = ok && (src < 0 || src >= rows || slot[i] < 0 || slot[i] >= rows);
        if (bad && writes) flag_device(status, DEV_BAD_INDEX);
        if (j < K && writes) new_slots[(size_t)g * K + j] = slot[i];
        if (!copy || bad) slot[i] = -1;
      }
      // Beams with copies, one after the other.
      int at = (g - g0) * (K / 2), to = (g - g0) * K;
      for (uint64_t left = used; left != 0; left &= left - 1) {
        const int b = __ffsll(left) - 1;
        const uint64_t mine_b =
            (uint64_t)__ballot_sync(kAll, slot[0] >= 0 && p[0] == b) |
            ((uint64_t)__ballot_sync(kAll, slot[1] >= 0 && p[1] == b) << 32);
        if (mine_b == 0) continue;
        const int row = row_of(b), cnt = __popcll(mine_b);
        if (lane == 0) {
          src_row[at] = row;
          src_at[at] = to;
          src_n[at] = cnt;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = lane + 32 * i;
          if (mine_b >> j & 1ull) dst_row[to + __popcll(mine_b & ((1ull << j) - 1ull))] = slot[i];
        }
        ++at;
        to += cnt;
      }
      if (lane == 0) in_group[g - g0] = at - (g - g0) * (K / 2);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      int before = 0;
      for (int x = 0; x < min(slice, G - g0); x += 32) {
        const int cnt = x + lane < min(slice, G - g0) ? in_group[x + lane] : 0;
        int incl = cnt;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int y = __shfl_up_sync(kAll, incl, off);
          if (lane >= off) incl += y;
        }
        for (int i = 0; i < cnt; ++i) order[before + incl - cnt + i] = (x + lane) * (K / 2) + i;
        before += __shfl_sync(kAll, incl, 31);
      }
      if (lane == 0) n_src = before;
    }
    __syncthreads();
    const int n = n_src;
    const long long units = pools.first[pools.count] * n;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
      const long long part = u / n;
      const int i = order[u - part * n];
      int p = 0;
      while (p + 1 < pools.count && part >= pools.first[p + 1]) ++p;
      const long long per_row = (pools.chunks[p] + kUnit - 1) / kUnit;
      const long long at = part - pools.first[p];
      const int layer = (int)(at / per_row);
      const long long c0 = (at - layer * per_row) * kUnit + threadIdx.x;
      uint4* base = reinterpret_cast<uint4*>(pools.base[p]) + (size_t)layer * rows * pools.chunks[p];
      const uint4* src = base + (size_t)src_row[i] * pools.chunks[p];
      uint4 v[kCopyVecs];
#pragma unroll
      for (int x = 0; x < kCopyVecs; ++x)
        if (c0 + x * kCopyThreads < pools.chunks[p]) v[x] = src[c0 + x * kCopyThreads];
      for (int d = 0; d < src_n[i]; ++d) {
        uint4* dst = base + (size_t)dst_row[src_at[i] + d] * pools.chunks[p];
#pragma unroll
        for (int x = 0; x < kCopyVecs; ++x)
          if (c0 + x * kCopyThreads < pools.chunks[p]) dst[c0 + x * kCopyThreads] = v[x];
      }
    }
    __syncthreads();
  }
}

template <typename T>
cudaError_t launch_select(const SelectArgs& a, cudaStream_t s) {
  const cudaError_t err =
      launch_pdl(scan_kernel<T>, dim3(a.segs, a.G * a.K), dim3(kScanThreads), 0, s, a);
  if (err != cudaSuccess) return err;
  return launch_pdl(merge_kernel<T>, dim3(a.G), dim3(kMergeThreads), 0, s, a);
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// The parts of the workspace: stats, floors, candidates.
size_t select_layout(long long segs, int n, size_t* at) {
  const size_t sizes[3] = {sizeof(float2) * (size_t)segs, sizeof(float) * (size_t)segs,
                           sizeof(uint2) * (size_t)segs * (n + 1)};
  size_t o = 0;
  for (int i = 0; i < 3; ++i) {
    if (at != nullptr) at[i] = o;
    o += round256(sizes[i]);
  }
  return o;
}

}  // namespace
}  // namespace sc

extern "C" size_t sc_beam_select_workspace(int groups, int beams, int vocab, int n,
                                           int logits_fp32) {
  if (groups <= 0 || beams <= 0 || vocab <= 0 || n <= 0 || n > sc::kMaxSelect) return 0;
  const long long rows = (long long)groups * beams;
  const sc::Segments seg = logits_fp32 ? sc::select_segments<float>(rows, vocab)
                                       : sc::select_segments<uint16_t>(rows, vocab);
  return sc::select_layout(rows * seg.count, n, nullptr);
}

extern "C" int sc_beam_select(const void* logits, int logits_fp32, int64_t row_stride,
                              const float* scores, const uint8_t* finished, int pad_token,
                              float* out_scores, int32_t* parents, int32_t* tokens,
                              void* workspace, size_t workspace_bytes, int groups, int beams,
                              int vocab, int n, void* stream) {
  const char* name = "sc_beam_select";
  SC_REQUIRE(groups >= 0 && beams > 0 && vocab > 0 && row_stride >= vocab, SC_ERR_INVALID,
             "%s: bad groups=%d beams=%d vocab=%d row_stride=%lld", name, groups, beams, vocab,
             (long long)row_stride);
  SC_REQUIRE(beams <= sc::kMaxBeams, SC_ERR_UNSUPPORTED, "%s: %d beams, at most %d", name, beams,
             sc::kMaxBeams);
  // Indices are 32-bit; the scan looks up to two rounds of blocks past a row's end for them.
  SC_REQUIRE((long long)beams * vocab <= (1ll << 31) - (1ll << 14), SC_ERR_UNSUPPORTED,
             "%s: beams * vocab = %lld, at most 2^31 - 2^14", name, (long long)beams * vocab);
  SC_REQUIRE(n > 0 && n <= sc::kMaxSelect && n <= (long long)beams * vocab, SC_ERR_UNSUPPORTED,
             "%s: n=%d not in 1..min(%d, beams * vocab)", name, n, sc::kMaxSelect);
  SC_REQUIRE(finished == nullptr || (pad_token >= 0 && pad_token < vocab), SC_ERR_INVALID,
             "%s: pad_token=%d outside the vocabulary", name, pad_token);
  if (groups == 0) return SC_OK;
  SC_REQUIRE((long long)groups * beams <= 65535, SC_ERR_UNSUPPORTED, "%s: %lld rows, at most 65535",
             name, (long long)groups * beams);
  SC_REQUIRE(logits && scores && out_scores && parents && tokens && workspace, SC_ERR_INVALID,
             "%s: null pointer", name);
  SC_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (logits_fp32 ? 4 : 2) == 0 &&
                 reinterpret_cast<uintptr_t>(workspace) % 256 == 0,
             SC_ERR_INVALID, "%s: misaligned logits or workspace (256 bytes)", name);
  const size_t need = sc_beam_select_workspace(groups, beams, vocab, n, logits_fp32);
  SC_REQUIRE(workspace_bytes >= need, SC_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", name,
             workspace_bytes, need);
  const long long rows = (long long)groups * beams;
  const sc::Segments seg = logits_fp32 ? sc::select_segments<float>(rows, vocab)
                                       : sc::select_segments<uint16_t>(rows, vocab);
  size_t at[3];
  sc::select_layout(rows * seg.count, n, at);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  sc::SelectArgs a;
  a.segs = seg.count;
  a.seg_blocks = seg.blocks;
  a.logits = logits;
  a.row_stride = row_stride;
  a.scores = scores;
  a.finished = finished;
  a.stats = reinterpret_cast<float2*>(ws + at[0]);
  a.floors = reinterpret_cast<float*>(ws + at[1]);
  a.kept = reinterpret_cast<uint2*>(ws + at[2]);
  a.out_scores = out_scores;
  a.parents = parents;
  a.tokens = tokens;
  a.G = groups;
  a.K = beams;
  a.V = vocab;
  a.n = n;
  a.pad = pad_token;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = logits_fp32 ? sc::launch_select<float>(a, s)
                                      : sc::launch_select<uint16_t>(a, s);
  if (err != cudaSuccess)
    return sc::set_error(SC_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
  return sc::check_launch(name);
}

extern "C" int sc_reorder_rows(void* const* pools, const int64_t* row_bytes, const int* layers,
                               int npools, int rows, const int32_t* slots, const int32_t* parents,
                               int32_t* new_slots, int groups, int beams, void* stream) {
  const char* name = "sc_reorder_rows";
  SC_REQUIRE(npools >= 0 && npools <= 4 && rows > 0 && groups >= 0 && beams > 0, SC_ERR_INVALID,
             "%s: bad npools=%d rows=%d groups=%d beams=%d", name, npools, rows, groups, beams);
  SC_REQUIRE(beams <= sc::kMaxBeams, SC_ERR_UNSUPPORTED, "%s: %d beams, at most %d", name, beams,
             sc::kMaxBeams);
  if (groups == 0) return SC_OK;
  SC_REQUIRE(slots && parents && new_slots && (npools == 0 || (pools && row_bytes && layers)),
             SC_ERR_INVALID, "%s: null pointer", name);
  sc::ReorderPools p = {};
  p.count = npools;
  for (int i = 0; i < npools; ++i) {
    SC_REQUIRE(pools[i] && reinterpret_cast<uintptr_t>(pools[i]) % 16 == 0 && row_bytes[i] > 0 &&
                   row_bytes[i] % 16 == 0 && layers[i] >= 0,
               SC_ERR_INVALID, "%s: pool %d: 16-byte aligned rows of a multiple of 16 bytes", name, i);
    p.base[i] = static_cast<uint8_t*>(pools[i]);
    p.chunks[i] = row_bytes[i] / 16;
    const long long unit = sc::kCopyThreads * sc::kCopyVecs;
    p.first[i + 1] = p.first[i] + layers[i] * ((p.chunks[i] + unit - 1) / unit);
  }
  // About eight places a CTA, in 8 to 32 CTAs an SM: short CTAs that come and go copied 2.1
  // GB at 6.4 TB/s where one resident wave, all reading and all writing at the same time,
  // reached 5.1; under eight an SM the plan that each of them makes costs more (151 MB: 35
  // us with 32 an SM, 26.6 with 8).
  const long long most = p.first[npools] * groups * (beams / 2);
  const int ctas = (int)std::min(most < 1 ? 1 : most, std::max(148ll * 8, std::min(148ll * 32, most / 8)));
  const cudaError_t err = sc::launch_pdl(sc::reorder_kernel, dim3(ctas), dim3(sc::kCopyThreads), 0,
                                         static_cast<cudaStream_t>(stream), p, slots, parents,
                                         new_slots, groups, beams, rows, sc::device_status_word());
  if (err != cudaSuccess)
    return sc::set_error(SC_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
  return sc::check_launch(name);
}
