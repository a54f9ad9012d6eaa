// Decode attention of sequences that share the pages of a long prefix.
//
// No reference counterpart (it runs one request at a time,
// studio_compute/mlx_decode.py:80-106); the math is that of split-K decode attention,
//   out[b,h] = softmax_j<L_b(scale q[b,h] . K_b[j]) V_b[j],
// with the first S_g pages of every sequence of group g the same. Softmax over a
// union splits into parts (m, sum, output) that merge exactly, so the prefix is
// attended once for the whole group and each sequence's own tail by itself:
//   prefix_kernel        Q of 128 (sequence, head) rows against a split of the prefix
//   the split-K kernel   one query a sequence against its own pages (paged_attention.cu)
//   merge_parts_kernel   the parts of each row -> bf16
// The first two run side by side (the second does not wait for the first to end).
//
// B200 mapping of prefix_kernel. Read once for 128 rows, a K/V byte carries 128
// multiply-adds, too many for the warp tensor path to keep up with HBM: tcgen05.
// One CTA per (split, kv head, tile of rows) and SM, six warps:
//   warps 0-3  one row a thread: scores out of TMEM, online softmax, P back into TMEM
//   warp 4     TMA: page ids from the block table, K and V tiles into rings of stages
//   warp 5     issues S = Q K^T (Q in TMEM) and O += P V (P in TMEM, over its scores)
// A stage holds kTok tokens of 16-token pages. The pool's rows are stored with their
// 16-byte chunks already permuted as the 128-byte swizzle wants them, so each 64-column
// slice of a page arrives by an unswizzled 16 x 128-byte TMA box and lands as two
// swizzle atoms; the slices of a tile's pages follow each other, which makes K a
// K-major and V an MN-major operand without a copy. S is double buffered: the scores of
// tile i + 1 are made while the softmax of tile i runs. O stays in TMEM and is rescaled
// only when a row's maximum grows by more than 2^8 over its reference (until then P may
// be as large as 2^8, which costs fp32 sums and bf16 P no accuracy).
// P is rounded to bf16 for the tensor cores, as in the split-K kernel; scores, maxima,
// sums and O are fp32.
#include <cudaTypedefs.h>
#include <math_constants.h>

#include <mutex>

#include "attention_internal.cuh"
#include "tc.cuh"

namespace sc {
namespace {

constexpr int kPageTok = 16;
constexpr int kRowsTile = 128;
constexpr int kSoftWarps = 4;
constexpr int kPrefixThreads = 192;
constexpr float kRescale = 8.f;  // log2 units

template <int D>
struct PrefixShape {
  static constexpr int TOK = D == 256 ? 64 : 128;  // tokens of a tile
  static constexpr int PAGES = TOK / kPageTok;
  static constexpr int SEGS = D / 64;              // 128-byte column slices
  static constexpr int TILE_BYTES = TOK * D * 2;   // K or V
  static constexpr int STAGES = 98304 / TILE_BYTES;
  static constexpr int SMEM = 2 * STAGES * TILE_BYTES + 1024 + 512;
  // TMEM columns: O, Q (two bf16 a column), two score buffers.
  static constexpr int T_Q = D, T_S = D + D / 2;
  static_assert(T_S + 2 * TOK <= 512, "TMEM plan");
  static_assert(2 * SMEM > 228 * 1024, "a second CTA per SM would wait for TMEM");
};

struct PrefixArgs {
  const uint16_t* q;
  const int32_t* block_table;
  const int32_t* ctx_len;
  const int4* tiles;        // first member, members, prefix pages, leader row
  const int32_t* members;   // rows of the batch
  float *part_out, *part_lse;
  long long num_pages;
  float scale_log2;
  int B, Hq, Hkv, G, max_pages, pages_per_split, num_splits;
  unsigned int* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                            int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(c0), "r"(c1), "r"(c2),
      "r"(c3)
      : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

template <int D>
__global__ void __launch_bounds__(kPrefixThreads, 1)
    prefix_kernel(const __grid_constant__ CUtensorMap pool, const PrefixArgs a) {
  using S = PrefixShape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                           ~uintptr_t(1023));
  uint64_t* kfull = reinterpret_cast<uint64_t*>(sm + 2 * S::STAGES * S::TILE_BYTES);
  uint64_t* vfull = kfull + S::STAGES;
  uint64_t* kfree = vfull + S::STAGES;
  uint64_t* vfree = kfree + S::STAGES;
  uint64_t* sfull = vfree + S::STAGES;  // [2] scores of a tile are in TMEM
  uint64_t* pfull = sfull + 2;          // [2] its P is
  uint64_t* ofull = pfull + 2;          // [2] O has taken it
  uint64_t* qfull = ofull + 2;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(qfull + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x, kvh = blockIdx.y;
  pdl_wait();
  pdl_trigger();

  const int4 tile = a.tiles[blockIdx.z];
  const int p0 = split * a.pages_per_split;
  if (p0 >= tile.z) return;  // uniform over the CTA
  if (tile.w < 0 || tile.w >= a.B || tile.z > a.max_pages || tile.y * a.G > kRowsTile) {
    if (tid == 0) flag_device(a.status, DEV_BAD_INDEX);
    return;
  }
  // A member attends here to the whole pages of its context; a page that its context
  // ends in is its tail's. Pages that no member attends to are not read.
  const auto pages_of = [&](int b) { return min(tile.z, max(a.ctx_len[b], 0) / kPageTok); };
  __shared__ int s_pages;
  if (tid == 0) s_pages = 0;
  __syncthreads();
  if (tid < tile.y) {
    const int b = a.members[tile.x + tid];
    if (b >= 0 && b < a.B)
      atomicMax(&s_pages, pages_of(b));
    else
      flag_device(a.status, DEV_BAD_INDEX);
  }
  __syncthreads();
  const int npages = min(p0 + a.pages_per_split, s_pages) - p0;
  if (npages <= 0) return;
  if (a.status != nullptr &&
      (*reinterpret_cast<volatile unsigned int*>(a.status) & DEV_WAIT_TIMEOUT))
    return;
  const int ntiles = (npages + S::PAGES - 1) / S::PAGES;

  if (tid == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(&kfull[i], 1);
      mbar_init(&vfull[i], 1);
      mbar_init(&kfree[i], 1);
      mbar_init(&vfree[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], kSoftWarps * 32);
      mbar_init(&ofull[i], 1);
    }
    mbar_init(qfull, kSoftWarps * 32);
    fence_mbar_init();
  }
  if (warp == 5) tc::tmem_alloc(s_tmem, 512);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *s_tmem;

  if (warp == 4) {
    // ---------------------------------------------------------------- TMA
    // Lane l moves slice l % SEGS of page l / SEGS of the tile, K and then V.
    const int32_t* row = a.block_table + (size_t)tile.w * a.max_pages + p0;
    constexpr int kBoxes = S::PAGES * S::SEGS;  // 16 for every D
    static_assert(kBoxes == 16 || kBoxes == 8, "one box a lane, K on one half, V on the other");
    const int box = lane & 15, which = lane >> 4;
    const bool moves = box < kBoxes;
    const int pg = box / S::SEGS, seg = box % S::SEGS;
    const auto page_of = [&](int i) {  // pages past the end repeat the last one (masked)
      return moves && i < ntiles ? row[min(i * S::PAGES + pg, npages - 1)] : 0;
    };
    int page = page_of(0);
    int issued = 0;
    for (int i = 0; i < ntiles; ++i) {
      const int next = page_of(i + 1);
      const int st = i % S::STAGES, round = i / S::STAGES;
      if (page < 0 || page >= a.num_pages) {
        flag_device(a.status, DEV_BAD_INDEX);
        page = 0;  // keep the copy in bounds; the status word reports the fault
      }
      bool ok = true;
      if (lane == 0 && round > 0)
        ok = mbar_wait_bounded(&kfree[st], (round - 1) & 1, a.status) &&
             mbar_wait_bounded(&vfree[st], (round - 1) & 1, a.status);
      if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&kfull[st], S::TILE_BYTES);
        mbar_arrive_expect_tx(&vfull[st], S::TILE_BYTES);
      }
      __syncwarp();
      if (moves) {
        const uint32_t dst = smem_addr(sm + (which * S::STAGES + st) * S::TILE_BYTES) +
                             seg * (S::TOK * 128) + pg * (kPageTok * 128);
        tma_load_4d(dst, &pool, 0, 0, seg, (page * a.Hkv + kvh) * 2 + which,
                    which ? &vfull[st] : &kfull[st]);
      }
      issued = i + 1;
      page = next;
    }
    // The last copy into each stage has landed before the CTA ends.
    if (lane == 0)
      for (int i = max(0, issued - S::STAGES); i < issued; ++i) {
        mbar_wait_bounded(&kfull[i % S::STAGES], (i / S::STAGES) & 1, a.status);
        mbar_wait_bounded(&vfull[i % S::STAGES], (i / S::STAGES) & 1, a.status);
      }
  } else if (warp == 5) {
    // ---------------------------------------------------------------- MMA
    if (lane == 0) {
      constexpr uint32_t kIdS = tc::idesc_bf16(kRowsTile, S::TOK, false, false);
      constexpr uint32_t kIdO = tc::idesc_bf16(kRowsTile, D, false, true);
      const auto scores = [&](int i) {
        const int st = i % S::STAGES;
        if (!mbar_wait_bounded(&kfull[st], (i / S::STAGES) & 1, a.status)) return false;
        tc::fence_after();
        const uint32_t kb = smem_addr(sm + st * S::TILE_BYTES);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc::mma_bf16_ts(tmem + S::T_S + (i & 1) * S::TOK, tmem + S::T_Q + 8 * kk,
                          tc::desc_kmajor(kb + (kk / 4) * (S::TOK * 128) + (kk % 4) * 32), kIdS,
                          kk > 0);
        tc::commit(&sfull[i & 1]);
        tc::commit(&kfree[st]);
        return true;
      };
      bool ok = mbar_wait_bounded(qfull, 0, a.status);
      tc::fence_after();
      ok = ok && scores(0);
      for (int i = 0; ok && i < ntiles; ++i) {
        if (i + 1 < ntiles) ok = scores(i + 1);
        const int st = i % S::STAGES;
        ok = ok && mbar_wait_bounded(&pfull[i & 1], (i >> 1) & 1, a.status) &&
             mbar_wait_bounded(&vfull[st], (i / S::STAGES) & 1, a.status);
        if (!ok) break;
        tc::fence_after();
        const uint32_t vb = smem_addr(sm + (S::STAGES + st) * S::TILE_BYTES);
#pragma unroll
        for (int kk = 0; kk < S::TOK / 16; ++kk)
          tc::mma_bf16_ts(tmem, tmem + S::T_S + (i & 1) * S::TOK + 8 * kk,
                          tc::desc_mnmajor(vb + kk * 2048, S::TOK * 128), kIdO, i > 0 || kk > 0);
        tc::commit(&vfree[st]);
        tc::commit(&ofull[i & 1]);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);  // this warp's TMEM lanes
    const int member = tid / a.G, h = tid - member * a.G;
    const int b = member < tile.y ? a.members[tile.x + member] : -1;
    const bool live = b >= 0 && b < a.B;
    const size_t out_row = live ? (size_t)b * a.Hq + kvh * a.G + h : 0;
    // Tokens of this split that the row attends to (its context may end inside the prefix).
    const int limit = live ? min(pages_of(b) - p0, npages) * kPageTok : 0;
    // A negative scale turns q, so that the largest score stays the largest; a zero one
    // clears it.
    const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    const uint32_t keep = a.scale_log2 == 0.f ? 0u : 0xffffffffu;
    const float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);
    {
      const uint4* src = reinterpret_cast<const uint4*>(a.q + out_row * D);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint4 u = live ? src[4 * c + x] : make_uint4(0u, 0u, 0u, 0u);
          w[4 * x] = u.x;
          w[4 * x + 1] = u.y;
          w[4 * x + 2] = u.z;
          w[4 * x + 3] = u.w;
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) w[x] = (w[x] ^ flip) & keep;
        tc::tmem_st16(mine + S::T_Q + 16 * c, w);
      }
      tc::tmem_wait_st();
      tc::fence_before();
      mbar_arrive(qfull);
    }
    float m = -CUDART_INF_F, l = 0.f;  // reference maximum (log2 units) and sum
    bool ok = true;
    for (int i = 0; i < ntiles; ++i) {
      ok = mbar_wait_bounded(&sfull[i & 1], (i >> 1) & 1, a.status);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc::fence_after();
      const uint32_t st = mine + S::T_S + (i & 1) * S::TOK;
      float x[S::TOK];
#pragma unroll
      for (int c = 0; c < S::TOK / 32; ++c) tc::tmem_ld32(st + 32 * c, x + 32 * c);
      const int left = limit - i * S::TOK;  // columns below it count
      if (left < S::TOK)
#pragma unroll
        for (int c = 0; c < S::TOK; ++c) x[c] = c < left ? x[c] : -CUDART_INF_F;
      float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
      for (int c = 0; c < S::TOK; ++c) mx[c & 3] = fmaxf(mx[c & 3], x[c]);
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
      const bool grows = top > m + kRescale || (m == -CUDART_INF_F && top > m);
      if (__any_sync(0xffffffffu, grows)) {
        const float to = grows ? top : m;
        const float f = m == to ? 1.f : ex2(m - to);  // 0 from -inf
        if (i > 0) {
          ok = mbar_wait_bounded(&ofull[(i - 1) & 1], ((i - 1) >> 1) & 1, a.status);
          if (!__all_sync(0xffffffffu, ok)) break;
          tc::fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tc::tmem_ld32(mine + 32 * c, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= f;
            tc::tmem_st32(mine + 32 * c, o);
          }
        }
        l *= f;
        m = to;
      }
      const float ref = m == -CUDART_INF_F ? 0.f : m;  // nothing seen yet: every p is 0
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < S::TOK / 32; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float y0 = ex2(fmaf(x[32 * c + 2 * e], scale, -ref));
          const float y1 = ex2(fmaf(x[32 * c + 2 * e + 1], scale, -ref));
          sum[(2 * e) & 3] += y0;
          sum[(2 * e + 1) & 3] += y1;
          w[e] = pack_bf16x2(y0, y1);
        }
        tc::tmem_st16(st + 16 * c, w);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tc::tmem_wait_st();
      tc::fence_before();
      mbar_arrive(&pfull[i & 1]);
    }
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      ok = mbar_wait_bounded(&ofull[(ntiles - 1) & 1], ((ntiles - 1) >> 1) & 1, a.status);
      tc::fence_after();
    }
    if (__all_sync(0xffffffffu, ok)) {
      const float inv = l > 0.f ? 1.f / l : 0.f;
      const size_t part = out_row * a.num_splits + split;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        tc::tmem_ld32(mine + 32 * c, o);
        if (live) {
          float4* dst = reinterpret_cast<float4*>(a.part_out + part * D + 32 * c);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[e] = make_float4(o[4 * e] * inv, o[4 * e + 1] * inv, o[4 * e + 2] * inv,
                                 o[4 * e + 3] * inv);
        }
      }
      if (live)
        a.part_lse[part] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f
                                   : (l == 0.f ? -CUDART_INF_F : l);  // a NaN stays one
    }
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (warp == 5) tc::tmem_dealloc(tmem, 512);
}

// The parts of each (sequence, head) row: those of its prefix, then its own tail's.
// D / 4 threads hold a float4 of the row each, the CTA's other threads take other parts;
// the weights e^(lse - M) are made once in shared memory.
constexpr int kMergeThreads2 = 256;
constexpr int kMergeMax = 1024;  // parts of one row

struct MergeArgs {
  const float *pre_out, *pre_lse, *tail_out, *tail_lse;
  const int32_t *ctx_len, *first_page;
  uint16_t* out;
  float* lse_out;
  int Hq, max_pages, pre_pps, pre_splits, tail_pps, tail_splits;
};

template <int D>
__global__ void __launch_bounds__(kMergeThreads2) merge_parts_kernel(const MergeArgs a) {
  constexpr int kCols = D / 4, kLanes = kMergeThreads2 / kCols;
  __shared__ float w[kMergeMax];
  __shared__ float red[kMergeThreads2 / 32], sums[kLanes];
  __shared__ float4 acc_s[kMergeThreads2];
  pdl_wait();
  pdl_trigger();
  const size_t row = blockIdx.x;
  const int b = (int)(row / a.Hq), tid = threadIdx.x;
  const int ctx = max(a.ctx_len[b], 0);
  const int skip = min(max(0, min(a.first_page[b], a.max_pages)), ctx / kPageTok);
  const int pages = min((ctx - skip * kPageTok + kPageTok - 1) / kPageTok, a.max_pages - skip);
  const int n_pre = min((skip + a.pre_pps - 1) / a.pre_pps, a.pre_splits);
  const int n = n_pre + min((pages + a.tail_pps - 1) / a.tail_pps, a.tail_splits);
  const auto lse_at = [&](int s) {
    return s < n_pre ? a.pre_lse[row * a.pre_splits + s] : a.tail_lse[row * a.tail_splits + s - n_pre];
  };
  float m = -CUDART_INF_F;
  for (int s = tid; s < n; s += kMergeThreads2) {
    w[s] = lse_at(s);
    m = fmaxf(m, w[s]);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if ((tid & 31) == 0) red[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMergeThreads2 / 32; ++i) m = fmaxf(m, red[i]);
  __syncthreads();
  const int col = tid % kCols, first = tid / kCols;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  for (int s = first; s < n; s += kLanes) {
    const float ls = w[s];
    if (ls == -CUDART_INF_F) continue;  // an empty part
    const float e = __expf(ls - m);
    const float* o = s < n_pre ? a.pre_out + (row * a.pre_splits + s) * D
                               : a.tail_out + (row * a.tail_splits + s - n_pre) * D;
    const float4 v = reinterpret_cast<const float4*>(o)[col];
    acc.x = fmaf(e, v.x, acc.x);
    acc.y = fmaf(e, v.y, acc.y);
    acc.z = fmaf(e, v.z, acc.z);
    acc.w = fmaf(e, v.w, acc.w);
    sum += e;
  }
  acc_s[tid] = acc;
  if (col == 0) sums[first] = sum;
  __syncthreads();
  if (tid < kCols) {
    float total = 0.f;
    for (int i = 0; i < kLanes; ++i) total += sums[i];
    for (int i = 1; i < kLanes; ++i) {
      const float4 v = acc_s[i * kCols + tid];
      acc.x += v.x;
      acc.y += v.y;
      acc.z += v.z;
      acc.w += v.w;
    }
    const float inv = n == 0 || total == 0.f ? 0.f : 1.f / total;
    uint2 u;
    u.x = pack_bf16x2(acc.x * inv, acc.y * inv);
    u.y = pack_bf16x2(acc.z * inv, acc.w * inv);
    reinterpret_cast<uint2*>(a.out + row * D)[tid] = u;
    if (tid == 0 && a.lse_out != nullptr)
      a.lse_out[row] = total == 0.f ? -CUDART_INF_F : m + logf(total);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// The pool as [block = (page, head, K|V)][64-column slice][token][64]: one box is the 16
// tokens of one slice, x always 0.
int encode_pool(CUtensorMap* map, const void* pool, int D, long long blocks) {
  auto fn = encode_fn();
  if (fn == nullptr)
    return set_error(SC_ERR_CUDA, "sc_shared_prefix_attention: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[4] = {64, kPageTok, (cuuint64_t)D / 64, (cuuint64_t)blocks};
  cuuint64_t strides[3] = {(cuuint64_t)D * 2, 128, (cuuint64_t)kPageTok * D * 2};
  cuuint32_t box[4] = {64, kPageTok, 1, 1};
  cuuint32_t step[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(pool), dims,
                        strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(SC_ERR_INVALID, "sc_shared_prefix_attention: tensor map rejected (%d)", (int)r);
  return SC_OK;
}

template <int D>
int launch_shared(const CUtensorMap& map, const PrefixArgs& p, const MergeArgs& m, int ntiles,
                  const sc_bf16* kv_pool, const int32_t* seq_order, float scale,
                  float* tail_out, float* tail_lse, cudaStream_t s) {
  const char* name = "sc_shared_prefix_attention";
  using S = PrefixShape<D>;
  static int configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    const cudaError_t err = cudaFuncSetAttribute(
        prefix_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (err != cudaSuccess)
      return set_error(SC_ERR_CUDA, "%s: smem attribute: %s", name, cudaGetErrorString(err));
    configured[dev] = 1;
  }
  cudaError_t err = launch_pdl(prefix_kernel<D>, dim3(p.num_splits, p.Hkv, ntiles),
                               dim3(kPrefixThreads), S::SMEM, s, map, p);
  if (err != cudaSuccess)
    return set_error(SC_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
  if (int rc = launch_decode_tail(p.q, kv_pool, p.num_pages, p.block_table, p.ctx_len, seq_order,
                                  m.first_page, p.B, p.Hq, p.Hkv, D, p.max_pages, m.tail_pps,
                                  m.tail_splits, scale, tail_out, tail_lse, s))
    return rc;
  err = launch_pdl(merge_parts_kernel<D>, dim3(p.B * p.Hq), dim3(kMergeThreads2), 0, s, m);
  if (err != cudaSuccess)
    return set_error(SC_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
  return check_launch(name);
}

}  // namespace
}  // namespace sc

extern "C" int sc_shared_prefix_attention(
    const sc_bf16* q, const sc_bf16* kv_pool, int64_t num_pages, const int32_t* block_table,
    const int32_t* ctx_len, const int32_t* seq_order, const int32_t* prefix_pages,
    const int32_t* tiles, const int32_t* members, int ntiles, int B, int Hq, int Hkv, int D, int P,
    int max_pages, int prefix_pages_per_split, int prefix_splits, int pages_per_split,
    int num_splits, float scale, float* prefix_out, float* prefix_lse, float* part_out,
    float* part_lse, sc_bf16* out, float* lse_out, void* stream) {
  const char* name = "sc_shared_prefix_attention";
  SC_REQUIRE(B >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0, SC_ERR_INVALID,
             "%s: bad heads Hq=%d Hkv=%d", name, Hq, Hkv);
  SC_REQUIRE(D == 64 || D == 128 || D == 256, SC_ERR_UNSUPPORTED, "%s: D=%d not in {64,128,256}",
             name, D);
  SC_REQUIRE(P == sc::kPageTok, SC_ERR_UNSUPPORTED, "%s: page size %d != 16", name, P);
  SC_REQUIRE(Hq / Hkv <= sc::kRowsTile, SC_ERR_UNSUPPORTED, "%s: %d query heads per kv head", name,
             Hq / Hkv);
  if (B == 0) return SC_OK;
  SC_REQUIRE(q && kv_pool && block_table && ctx_len && prefix_pages && tiles && members && out &&
                 prefix_out && prefix_lse && part_out && part_lse,
             SC_ERR_INVALID, "%s: null pointer", name);
  SC_REQUIRE(num_pages > 0 && max_pages > 0 && ntiles > 0 && prefix_pages_per_split > 0 &&
                 prefix_splits > 0 && pages_per_split > 0 && num_splits > 0,
             SC_ERR_INVALID, "%s: bad plan max_pages=%d ntiles=%d splits=%d x %d + %d x %d", name,
             max_pages, ntiles, prefix_splits, prefix_pages_per_split, num_splits, pages_per_split);
  SC_REQUIRE(prefix_splits + num_splits <= sc::kMergeMax, SC_ERR_INVALID,
             "%s: %d + %d splits, at most %d", name, prefix_splits, num_splits, sc::kMergeMax);
  SC_REQUIRE(B <= 65535 && ntiles <= 65535 && Hkv * ((Hq / Hkv + 7) / 8) <= 65535 &&
                 num_pages * Hkv * 2 < (1ll << 31),
             SC_ERR_INVALID, "%s: grid or pool too large", name);
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  SC_REQUIRE(aligned(q) && aligned(kv_pool) && aligned(out) && aligned(prefix_out) &&
                 aligned(part_out) && aligned(tiles),
             SC_ERR_INVALID, "%s: operands must be 16-byte aligned", name);
  CUtensorMap map;
  if (int rc = sc::encode_pool(&map, kv_pool, D, num_pages * Hkv * 2)) return rc;
  sc::PrefixArgs p;
  p.q = q;
  p.block_table = block_table;
  p.ctx_len = ctx_len;
  p.tiles = reinterpret_cast<const int4*>(tiles);
  p.members = members;
  p.part_out = prefix_out;
  p.part_lse = prefix_lse;
  p.num_pages = num_pages;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.max_pages = max_pages;
  p.pages_per_split = prefix_pages_per_split;
  p.num_splits = prefix_splits;
  p.status = sc::device_status_word();
  sc::MergeArgs m;
  m.pre_out = prefix_out;
  m.pre_lse = prefix_lse;
  m.tail_out = part_out;
  m.tail_lse = part_lse;
  m.ctx_len = ctx_len;
  m.first_page = prefix_pages;
  m.out = out;
  m.lse_out = lse_out;
  m.Hq = Hq;
  m.max_pages = max_pages;
  m.pre_pps = prefix_pages_per_split;
  m.pre_splits = prefix_splits;
  m.tail_pps = pages_per_split;
  m.tail_splits = num_splits;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto launch = D == 64    ? sc::launch_shared<64>
                      : D == 128 ? sc::launch_shared<128>
                                 : sc::launch_shared<256>;
  return launch(map, p, m, ntiles, kv_pool, seq_order, scale, part_out, part_lse, s);
}
