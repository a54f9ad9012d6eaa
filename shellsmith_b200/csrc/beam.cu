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
// B200 mapping: HBM-bound, the logits are read once. scan_kernel: a CTA holds a chunk
// of one row in registers, makes the chunk's (max, sum) and keeps every logit at or
// above a threshold that at least n + 1 of the chunk reach: the (n + 1)-th largest of
// its 256 threads' maxima (n + 1 distinct logits reach it; found by bisection over
// the order-preserving integer keys, one block count per bit). Within a row the score
// is monotone in the logit, so no other logit can be among the n best, save by the
// rounding of scores below. merge_kernel, one CTA per group: the rows' statistics,
// the scores of all kept logits, a threshold over them in the same way, and the rank
// of each survivor by counting.
//
// Scores of different logits can round to the same fp32 number (a large |score_k|),
// and then the lower index wins even against a larger logit. A chunk's dropped logits
// are all below its threshold t; if the next value below t still scores as much as
// the n-th best, merge_kernel rescans the group's logits for scores equal to it, in
// index order, until it has enough.
#include <math_constants.h>

#include "common.cuh"

namespace sc {
namespace {

constexpr int kScanThreads = 256;
constexpr int kMergeThreads = 512;
constexpr int kMaxSelect = 64;       // n
constexpr int kSegment = 160;        // kept logits of one chunk (>= kMaxSelect + 1)
constexpr int kScanList = 4096 + 80; // a chunk's survivors before they are cut to kSegment
constexpr int kMergeList = 2048;
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

// (max, sum of e^(x - max)) of two disjoint sets. A NaN sum stays NaN; a set whose
// maximum is -inf is empty unless its sum is NaN.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float M = fmaxf(m, m2);
  const float a = s == 0.f ? 0.f : (m == M ? s : s * expf(m - M));
  const float b = s2 == 0.f ? 0.f : (m2 == M ? s2 : s2 * expf(m2 - M));
  m = M;
  s = a + b;
}

// Largest key t (its low 32 - kBits bits zero) such that at least `want` threads hold
// a key >= t; 0 when fewer than `want` hold any. Bits are set from the top.
template <int kBits>
__device__ __forceinline__ uint32_t nth_key(uint32_t key, int want) {
  uint32_t t = 0;
#pragma unroll 1
  for (int b = 31; b >= 32 - kBits; --b) {
    const uint32_t next = t | (1u << b);
    if (__syncthreads_count(key >= next) >= want) t = next;
  }
  return t;
}

struct SelectArgs {
  const void* logits;
  long long row_stride;          // elements between rows
  const float* scores;           // [G, K]
  const uint8_t* finished;       // [G, K] or NULL
  float2* stats;                 // [rows][chunks] (max, sum)
  int* counts;                   // [rows][chunks] kept
  float* floors;                 // [rows][chunks] threshold where logits were dropped, else -inf
  float* kept_x;                 // [rows][chunks][kSegment]
  int32_t* kept_v;
  float* out_scores;             // [G, n]
  int32_t *parents, *tokens;
  int G, K, V, n, chunks, pad;
};

// A row that offers no logit: finished, or its score is -inf or NaN.
__device__ __forceinline__ bool row_idle(const SelectArgs& a, int row) {
  return (a.finished != nullptr && a.finished[row]) || !(a.scores[row] > -CUDART_INF_F);
}

template <typename T, int kVecs>
__global__ void __launch_bounds__(kScanThreads) scan_kernel(const SelectArgs a) {
  using L = Logits<T>;
  constexpr int E = L::kPerVec;
  __shared__ uint32_t list_k[kScanList];
  __shared__ int list_v[kScanList];
  __shared__ int n_above, n_equal, n_out;
  __shared__ float red_m[kScanThreads / 32], red_s[kScanThreads / 32];
  __shared__ int scan_w[kScanThreads / 32];
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.y, chunk = blockIdx.x;
  const size_t seg = (size_t)row * a.chunks + chunk;
  if (row_idle(a, row)) {  // uniform over the CTA
    if (threadIdx.x == 0) {
      a.counts[seg] = 0;
      a.floors[seg] = -CUDART_INF_F;
    }
    return;
  }
  if (threadIdx.x == 0) n_above = n_equal = n_out = 0;
  // Aligned 16-byte granules over the row; the first and the last may hold elements
  // outside it, which are read one by one.
  const T* base = reinterpret_cast<const T*>(a.logits) + (long long)row * a.row_stride;
  const int lead = (int)((reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T));
  const T* start = base - lead;  // granule g covers elements E g - lead .. of the row
  const int g0 = chunk * kScanThreads * kVecs + threadIdx.x;
  uint4 r[kVecs];
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int v0 = (g0 + j * kScanThreads) * E - lead;
    if (v0 >= 0 && v0 + E <= a.V) {
      r[j] = __ldcs(reinterpret_cast<const uint4*>(start) + g0 + j * kScanThreads);
    } else {
      r[j] = L::fill();
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (v0 + e >= 0 && v0 + e < a.V) L::put(r[j], e, base[v0 + e]);
    }
  }
  float m = -CUDART_INF_F, s = 0.f;
#pragma unroll
  for (int j = 0; j < kVecs; ++j)
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, L::get(r[j], e));
  // x - m is taken before the change of base: the largest terms then carry no error of
  // the product with log2 e. Where every x is -inf (or NaN) the sum tells them apart.
  const float ref = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll
  for (int j = 0; j < kVecs; ++j)
#pragma unroll
    for (int e = 0; e < E; ++e) s += ex2((L::get(r[j], e) - ref) * 1.4426950408889634f);

  const uint32_t mine = L::key(m);
  const uint32_t t = nth_key<L::kBits>(mine, a.n + 1);
  // Logits above t: at most n threads hold any, so they fit the list.
  const auto push = [&](int at, uint32_t k, int j, int e) {
    list_k[at] = k;
    list_v[at] = (g0 + j * kScanThreads) * E - lead + e;
  };
  int eq = 0;
  if (mine >= t && mine != 0u) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t k = L::key(L::get(r[j], e));
        if (k > t) push(atomicAdd(&n_above, 1), k, j, e);
        eq += k == t && t != 0u;
      }
    if (eq) atomicAdd(&n_equal, eq);
  }
  float wm = m, ws = s;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, wm, off);
    const float s2 = __shfl_xor_sync(0xffffffffu, ws, off);
    join(wm, ws, m2, s2);
  }
  if ((threadIdx.x & 31) == 0) {
    red_m[threadIdx.x >> 5] = wm;
    red_s[threadIdx.x >> 5] = ws;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kScanThreads / 32; ++w) join(wm, ws, red_m[w], red_s[w]);
    a.stats[seg] = make_float2(wm, ws);
  }
  const int above = n_above, equal = n_equal;
  int total = above + equal;
  if (total <= kSegment) {
    if (eq) {
#pragma unroll
      for (int j = 0; j < kVecs; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (L::key(L::get(r[j], e)) == t) push(above + atomicAdd(&n_out, 1), t, j, e);
    }
  } else {
    // Of the equal ones the n + 1 of lowest index are enough: any other has as much as
    // these and comes after them. Granule j of the threads in order is index order.
    int have = 0;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      if (have > a.n) break;  // uniform
      int c = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) c += t != 0u && L::key(L::get(r[j], e)) == t;
      int incl = c;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, off);
        if ((threadIdx.x & 31) >= off) incl += y;
      }
      if ((threadIdx.x & 31) == 31) scan_w[threadIdx.x >> 5] = incl;
      __syncthreads();
      int at = have + incl - c, sum = 0;
      for (int w = 0; w < kScanThreads / 32; ++w) {
        if (w < (int)(threadIdx.x >> 5)) at += scan_w[w];
        sum += scan_w[w];
      }
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (t != 0u && L::key(L::get(r[j], e)) == t) {
          if (at <= a.n) push(above + at, t, j, e);
          ++at;
        }
      have += sum;
      __syncthreads();
    }
    total = above + min(have, a.n + 1);
  }
  __syncthreads();
  // Cut to the segment: the n + 1 largest (equal ones: lowest index) of the list.
  uint32_t cut = t;
  if (total > kSegment) {
    cut = 0;
#pragma unroll 1
    for (int b = 31; b >= 32 - L::kBits; --b) {
      const uint32_t next = cut | (1u << b);
      int c = 0;
      for (int i = threadIdx.x; i < total; i += kScanThreads) c += list_k[i] >= next;
      c = __reduce_add_sync(0xffffffffu, c);
      if ((threadIdx.x & 31) == 0) scan_w[threadIdx.x >> 5] = c;
      __syncthreads();
      int all = 0;
      for (int w = 0; w < kScanThreads / 32; ++w) all += scan_w[w];
      if (all > a.n) cut = next;
      __syncthreads();
    }
    if (threadIdx.x == 0) n_out = 0;
    __syncthreads();
  }
  float* kx = a.kept_x + seg * kSegment;
  int32_t* kv = a.kept_v + seg * kSegment;
  if (total <= kSegment) {
    for (int i = threadIdx.x; i < total; i += kScanThreads) {
      kx[i] = L::unkey(list_k[i]);
      kv[i] = list_v[i];
    }
  } else {
    for (int i = threadIdx.x; i < total; i += kScanThreads) {
      const uint32_t k = list_k[i];
      bool keep = k > cut;
      if (k == cut) {  // rank among the equal ones and those above
        int rank = 0;
        for (int o = 0; o < total; ++o) rank += list_k[o] > cut || (list_k[o] == cut && list_v[o] < list_v[i]);
        keep = rank <= a.n;
      }
      if (keep) {
        const int at = atomicAdd(&n_out, 1);
        kx[at] = L::unkey(k);
        kv[at] = list_v[i];
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.counts[seg] = total <= kSegment ? total : n_out;
    a.floors[seg] = cut == 0u ? -CUDART_INF_F : L::unkey(cut);  // 0: every candidate is kept
  }
}

// The number of keys >= bound over the CTA's threads' items, for the bisections below.
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
  __shared__ float row_m[kMaxBeams], row_l[kMaxBeams];
  __shared__ unsigned long long list[kMergeList];
  __shared__ int scratch[kMergeThreads / 32];
  __shared__ int n_list, ambiguous;
  pdl_wait();
  pdl_trigger();
  const int g = blockIdx.x, K = a.K, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) n_list = ambiguous = 0;
  for (int k = warp; k < K; k += kMergeThreads / 32) {
    const int row = g * K + k;
    float m = -CUDART_INF_F, s = 0.f;
    if (!row_idle(a, row))
      for (int c = lane; c < a.chunks; c += 32) {
        const float2 st = a.stats[(size_t)row * a.chunks + c];
        join(m, s, st.x, st.y);
      }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, off);
      const float s2 = __shfl_xor_sync(0xffffffffu, s, off);
      join(m, s, m2, s2);
    }
    if (lane == 0) {
      row_m[k] = m;
      row_l[k] = logf(s);
    }
  }
  __syncthreads();
  const auto score = [&](int k, float x) {
    return a.scores[g * K + k] + ((x - row_m[k]) - row_l[k]);
  };
  // (score, lower index first) as one key; 0 for -inf and NaN.
  const auto full_key = [&](int k, float sc, int v) -> unsigned long long {
    const uint32_t key = score_key(sc);
    return key == 0u ? 0ull
                     : ((unsigned long long)key << 32) | (0xffffffffu - ((uint32_t)k * a.V + v));
  };
  const int segs = K * a.chunks;
  // Items: the kept logits of segment i / kSegment, then one per finished beam.
  const auto each = [&](auto&& f) {
    for (int sgm = warp; sgm < segs; sgm += kMergeThreads / 32) {
      const int k = sgm / a.chunks;
      const size_t seg = (size_t)g * segs + sgm;
      const int cnt = a.counts[seg];
      for (int i = lane; i < cnt; i += 32)
        f(full_key(k, score(k, a.kept_x[seg * kSegment + i]), a.kept_v[seg * kSegment + i]));
    }
    if (a.finished != nullptr)
      for (int k = threadIdx.x; k < K; k += kMergeThreads)
        if (a.finished[g * K + k]) f(full_key(k, a.scores[g * K + k], a.pad));
  };
  unsigned long long best = 0ull;
  each([&](unsigned long long key) { best = key > best ? key : best; });
  // At least n items reach the n-th largest of the threads' best scores.
  uint32_t t = nth_key<32>((uint32_t)(best >> 32), a.n);
  int c = 0;
  each([&](unsigned long long key) { c += key != 0ull && (uint32_t)(key >> 32) >= t; });
  unsigned long long floor_key = (unsigned long long)t << 32;
  if (block_total(c, scratch) > kMergeList) {  // the n largest keys exactly
    floor_key = 0ull;
    for (int b = 63; b >= 0; --b) {
      const unsigned long long next = floor_key | (1ull << b);
      c = 0;
      each([&](unsigned long long key) { c += key >= next; });
      if (block_total(c, scratch) >= a.n) floor_key = next;
    }
  }
  each([&](unsigned long long key) {
    if (key != 0ull && key >= floor_key) list[atomicAdd(&n_list, 1)] = key;
  });
  __syncthreads();
  const int total = n_list;
  float* os = a.out_scores + (size_t)g * a.n;
  int32_t* op = a.parents + (size_t)g * a.n;
  int32_t* ot = a.tokens + (size_t)g * a.n;
  const auto emit = [&](int rank, float sc, uint32_t flat) {
    os[rank] = sc;
    op[rank] = (int32_t)(flat / (uint32_t)a.V);
    ot[rank] = (int32_t)(flat % (uint32_t)a.V);
  };
  __shared__ uint32_t last_score;
  __shared__ int strictly;
  if (threadIdx.x == 0) last_score = 0u, strictly = 0;
  __syncthreads();
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
    const float fl = a.floors[(size_t)g * segs + sgm];
    if (fl > -CUDART_INF_F && score_key(score(sgm / a.chunks, L::below(fl))) >= last) ambiguous = 1;
  }
  for (int i = threadIdx.x; i < total; i += kMergeThreads)
    if ((uint32_t)(list[i] >> 32) > last) atomicAdd(&strictly, 1);
  __syncthreads();
  if (!ambiguous) return;
  const float target = key_value(last);
  int have = strictly;
  for (int k = 0; k < K && have < a.n; ++k) {
    const int row = g * K + k;
    if (row_idle(a, row)) {
      const bool fin = a.finished != nullptr && a.finished[row];
      if (fin && a.scores[row] == target) {
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

// Chunks of 8 granules a thread amortise the bisection; small calls take 2, so that
// their few rows spread over more SMs.
template <typename T>
int select_vecs(long long rows, int V) {
  return rows * V <= (long long)148 * kScanThreads * Logits<T>::kPerVec * 8 ? 2 : 8;
}
template <typename T>
int chunk_count(int V, int vecs) {
  const int per = kScanThreads * vecs * Logits<T>::kPerVec;
  return (int)(((long long)V + Logits<T>::kPerVec - 1 + per - 1) / per);  // + the lead of an unaligned row
}

// ---------------------------------------------------------------- reordering of rows
// Child j of group g continues beam parents[g][j]. The first child of a beam keeps the
// beam's slot; each later child takes the slot of a beam without children, in ascending
// order of both. A slot that is read is never written, so the copies run in place and
// in any order.
constexpr int kPlanThreads = 256;
constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 4;  // 16-byte loads in flight per thread

struct ReorderPools {
  uint8_t* base[4];
  long long chunks[4];  // 16-byte chunks per row
  int layers[4];
  long long first[5];   // work units before pool p, per copied row
  int count;
};

// One warp per group, lane l its children l and l + 32; sets of beams are 64-bit masks.
__global__ void __launch_bounds__(kPlanThreads)
    reorder_plan_kernel(const int32_t* __restrict__ slots, const int32_t* __restrict__ parents,
                        int32_t* __restrict__ new_slots, int2* __restrict__ copies,
                        int* __restrict__ n_copies, int G, int K, int rows, unsigned int* status) {
  constexpr unsigned kAll = 0xffffffffu;
  pdl_wait();
  pdl_trigger();
  __shared__ int total;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const uint64_t beams = K == 64 ? ~0ull : (1ull << K) - 1ull;
  for (int g = threadIdx.x >> 5; g < G; g += kPlanThreads / 32) {
    const int32_t* mine = slots + (size_t)g * K;
    int p[2];
    uint64_t used = 0, later = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = lane + 32 * i;
      p[i] = j < K ? parents[(size_t)g * K + j] : -1;
      const bool ok = p[i] >= 0 && p[i] < K;
      if (j < K && !ok) flag_device(status, DEV_BAD_INDEX);
      // A child is a later one if its beam has a child among the lower lanes or lanes
      // 0-31 of the first round.
      const unsigned same = __match_any_sync(kAll, ok ? p[i] : -1);
      const bool again = ok && ((same & ((1u << lane) - 1u)) != 0u || (used >> p[i] & 1ull));
      later |= (uint64_t)__ballot_sync(kAll, again) << (32 * i);
      const uint64_t bit = ok ? 1ull << p[i] : 0ull;
      used |= (uint64_t)__reduce_or_sync(kAll, (unsigned)bit) |
              ((uint64_t)__reduce_or_sync(kAll, (unsigned)(bit >> 32)) << 32);
    }
    const uint64_t dead = beams & ~used;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = lane + 32 * i;
      if (j >= K) continue;
      int slot = -1;
      if (p[i] >= 0 && p[i] < K) {
        const int src = mine[p[i]];
        slot = src;
        if (later >> j & 1ull) {
          uint64_t d = dead;  // as many beams without children as later ones, at least
          for (int skip = __popcll(later & ((1ull << j) - 1ull)); skip > 0; --skip) d &= d - 1;
          slot = d != 0 ? mine[__ffsll(d) - 1] : -1;
          if (src >= 0 && src < rows && slot >= 0 && slot < rows)
            copies[atomicAdd(&total, 1)] = make_int2(src, slot);
        }
        if (src < 0 || src >= rows || slot < 0 || slot >= rows) flag_device(status, DEV_BAD_INDEX);
      }
      new_slots[(size_t)g * K + j] = slot;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) *n_copies = total;
}

__global__ void __launch_bounds__(kCopyThreads)
    reorder_copy_kernel(const __grid_constant__ ReorderPools pools, const int2* __restrict__ copies,
                        const int* __restrict__ n_copies, int rows) {
  pdl_wait();
  pdl_trigger();
  const int n = *n_copies;
  const long long units = pools.first[pools.count] * n;
  constexpr int kUnit = kCopyThreads * kCopyVecs;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const long long part = u / n;  // consecutive units: the copies of one place
    const int2 cp = copies[u - part * n];
    int p = 0;
    while (p + 1 < pools.count && part >= pools.first[p + 1]) ++p;
    const long long per_row = (pools.chunks[p] + kUnit - 1) / kUnit;
    const long long at = part - pools.first[p];
    const int layer = (int)(at / per_row);
    const long long c0 = (at - layer * per_row) * kUnit + threadIdx.x;
    uint4* base = reinterpret_cast<uint4*>(pools.base[p]) + (size_t)layer * rows * pools.chunks[p];
    const uint4* src = base + (size_t)cp.x * pools.chunks[p];
    uint4* dst = base + (size_t)cp.y * pools.chunks[p];
    uint4 v[kCopyVecs];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
      if (c0 + i * kCopyThreads < pools.chunks[p]) v[i] = src[c0 + i * kCopyThreads];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
      if (c0 + i * kCopyThreads < pools.chunks[p]) dst[c0 + i * kCopyThreads] = v[i];
  }
}

template <typename T>
cudaError_t launch_select(SelectArgs a, int vecs, cudaStream_t s) {
  const dim3 grid(a.chunks, a.G * a.K);
  cudaError_t err = launch_pdl(vecs == 2 ? scan_kernel<T, 2> : scan_kernel<T, 8>, grid,
                               dim3(kScanThreads), 0, s, a);
  if (err != cudaSuccess) return err;
  return launch_pdl(merge_kernel<T>, dim3(a.G), dim3(kMergeThreads), 0, s, a);
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// The parts of the workspace: stats, counts, floors, kept logits, kept tokens.
size_t select_layout(long long segs, size_t* at) {
  size_t o = 0;
  const size_t sizes[5] = {sizeof(float2) * (size_t)segs, sizeof(int) * (size_t)segs,
                           sizeof(float) * (size_t)segs, sizeof(float) * (size_t)segs * kSegment,
                           sizeof(int32_t) * (size_t)segs * kSegment};
  for (int i = 0; i < 5; ++i) {
    if (at != nullptr) at[i] = o;
    o += round256(sizes[i]);
  }
  return o;
}

}  // namespace
}  // namespace sc

extern "C" size_t sc_beam_select_workspace(int groups, int beams, int vocab, int logits_fp32) {
  if (groups <= 0 || beams <= 0 || vocab <= 0) return 0;
  const long long rows = (long long)groups * beams;
  const int vecs = logits_fp32 ? sc::select_vecs<float>(rows, vocab)
                               : sc::select_vecs<uint16_t>(rows, vocab);
  const int chunks = logits_fp32 ? sc::chunk_count<float>(vocab, vecs)
                                 : sc::chunk_count<uint16_t>(vocab, vecs);
  return sc::select_layout(rows * chunks, nullptr);
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
  SC_REQUIRE((long long)beams * vocab < (1ll << 31), SC_ERR_UNSUPPORTED,
             "%s: beams * vocab = %lld does not fit 31 bits", name, (long long)beams * vocab);
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
  const size_t need = sc_beam_select_workspace(groups, beams, vocab, logits_fp32);
  SC_REQUIRE(workspace_bytes >= need, SC_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", name,
             workspace_bytes, need);
  const long long rows = (long long)groups * beams;
  const int vecs = logits_fp32 ? sc::select_vecs<float>(rows, vocab)
                               : sc::select_vecs<uint16_t>(rows, vocab);
  sc::SelectArgs a;
  a.chunks = logits_fp32 ? sc::chunk_count<float>(vocab, vecs)
                         : sc::chunk_count<uint16_t>(vocab, vecs);
  size_t at[5];
  sc::select_layout(rows * a.chunks, at);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.logits = logits;
  a.row_stride = row_stride;
  a.scores = scores;
  a.finished = finished;
  a.stats = reinterpret_cast<float2*>(ws + at[0]);
  a.counts = reinterpret_cast<int*>(ws + at[1]);
  a.floors = reinterpret_cast<float*>(ws + at[2]);
  a.kept_x = reinterpret_cast<float*>(ws + at[3]);
  a.kept_v = reinterpret_cast<int32_t*>(ws + at[4]);
  a.out_scores = out_scores;
  a.parents = parents;
  a.tokens = tokens;
  a.G = groups;
  a.K = beams;
  a.V = vocab;
  a.n = n;
  a.pad = pad_token;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = logits_fp32 ? sc::launch_select<float>(a, vecs, s)
                                      : sc::launch_select<uint16_t>(a, vecs, s);
  if (err != cudaSuccess)
    return sc::set_error(SC_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
  return sc::check_launch(name);
}

extern "C" int sc_reorder_rows(void* const* pools, const int64_t* row_bytes, const int* layers,
                               int npools, int rows, const int32_t* slots, const int32_t* parents,
                               int32_t* new_slots, int32_t* copies, int groups, int beams,
                               void* stream) {
  const char* name = "sc_reorder_rows";
  SC_REQUIRE(npools >= 0 && npools <= 4 && rows > 0 && groups >= 0 && beams > 0, SC_ERR_INVALID,
             "%s: bad npools=%d rows=%d groups=%d beams=%d", name, npools, rows, groups, beams);
  SC_REQUIRE(beams <= sc::kMaxBeams, SC_ERR_UNSUPPORTED, "%s: %d beams, at most %d", name, beams,
             sc::kMaxBeams);
  if (groups == 0) return SC_OK;
  SC_REQUIRE(slots && parents && new_slots && copies && (npools == 0 || (pools && row_bytes && layers)),
             SC_ERR_INVALID, "%s: null pointer", name);
  SC_REQUIRE((long long)groups * beams <= (1 << 20), SC_ERR_UNSUPPORTED, "%s: %lld beams in all",
             name, (long long)groups * beams);
  SC_REQUIRE(reinterpret_cast<uintptr_t>(copies) % 8 == 0, SC_ERR_INVALID,
             "%s: copies must be 8-byte aligned", name);
  sc::ReorderPools p = {};
  p.count = npools;
  for (int i = 0; i < npools; ++i) {
    SC_REQUIRE(pools[i] && reinterpret_cast<uintptr_t>(pools[i]) % 16 == 0 && row_bytes[i] > 0 &&
                   row_bytes[i] % 16 == 0 && layers[i] >= 0,
               SC_ERR_INVALID, "%s: pool %d: 16-byte aligned rows of a multiple of 16 bytes", name, i);
    p.base[i] = static_cast<uint8_t*>(pools[i]);
    p.chunks[i] = row_bytes[i] / 16;
    p.layers[i] = layers[i];
    const long long unit = sc::kCopyThreads * sc::kCopyVecs;
    p.first[i + 1] = p.first[i] + layers[i] * ((p.chunks[i] + unit - 1) / unit);
  }
  // The plan's scratch: the copy count, then the (source, destination) pairs.
  int* n_copies = reinterpret_cast<int*>(copies);
  int2* pairs = reinterpret_cast<int2*>(copies + 2);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err = sc::launch_pdl(sc::reorder_plan_kernel, dim3(1), dim3(sc::kPlanThreads), 0, s,
                                   slots, parents, new_slots, pairs, n_copies, groups, beams, rows,
                                   sc::device_status_word());
  if (err == cudaSuccess && npools > 0 && p.first[npools] > 0)
    err = sc::launch_pdl(sc::reorder_copy_kernel, dim3(148 * 8), dim3(sc::kCopyThreads), 0, s, p,
                         static_cast<const int2*>(pairs), static_cast<const int*>(n_copies), rows);
  if (err != cudaSuccess)
    return sc::set_error(SC_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
  return sc::check_launch(name);
}
