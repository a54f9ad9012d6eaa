// Decode attention of sequences that share the pages of a long prefix.
//
// No reference counterpart (it runs one request at a time,
// studio_compute/mlx_decode.py:80-106); the math is that of split-K decode attention,
//   out[b,h] = softmax_j<L_b(scale q[b,h] . K_b[j]) V_b[j],
// with the first S_g pages of every sequence of group g the same. Softmax over a
// union splits into parts (m, sum, output) that merge exactly, so the prefix is
// attended once for the whole group and each sequence's own tail by itself:
//   prefix_kernel        Q of 128 (sequence, head) rows against a split of the prefix
//   tail_kernel          one query a sequence against its own pages
//   merge_parts_kernel   the parts of each row -> bf16
// The first two run side by side: the second does not wait for the first to end, and a
// CTA of each fits on an SM, so that one's loads run under the other's products.
//
// B200 mapping of prefix_kernel. Read once for 128 rows, a K/V byte carries 128
// multiply-adds, too many for the warp tensor path to keep up with HBM: tcgen05.
// One CTA per (split, kv head, tile of rows) and SM, eleven warps:
//   warps 0-7  softmax: warp w holds rows 32 (w % 4) .. (its TMEM lanes), one a thread,
//              and half w / 4 of each tile's columns: scores out of TMEM, P back
//   warps 8, 9 TMA: page ids from the block table, K (V) tiles into a ring of stages
//   warp 10    issues S = Q K^T (Q in TMEM) and O += P V (P in TMEM, over its scores)
// A stage holds the pages of TOK tokens. The pool's rows are stored with their 16-byte
// chunks already permuted as the 128-byte swizzle wants them, so an unswizzled TMA box
// (8 or 16 tokens x 64 columns x D / 64 slices) lands as swizzle atoms and nothing is
// copied. K comes in boxes of half a page: its 8-token groups are then evenly spaced and
// one product covers the tile's tokens. V comes in boxes of a page, the 16 rows of one
// step of its product. The whole MMA warp walks the loop and one elected lane issues: its
// operands stay in uniform registers (a product of N = 64 then takes 32 cycles; issued
// from a lane's own branch it took 49). S is double buffered: the scores of
// tile i + 1 are made while the softmax of tile i runs. O stays in TMEM and is rescaled
// only when a row's maximum grows by more than 2^8 over its reference (until then P may
// be as large as 2^8, which costs fp32 sums and bf16 P no accuracy).
// P is rounded to bf16 for the tensor cores, as in the split-K kernel; scores, maxima,
// sums and O are fp32. The exponentials are ex2.approx here and __expf in the merge: a
// few units in the last place, far below P's rounding. A row whose context ends inside the
// prefix keeps its O from that page on: a page is a product, and a product can leave TMEM
// lanes as they are. Two stages (128 KB at D = 256) leave room for the tail's CTA.
//
// tail_kernel. HBM-bound, 8 query heads to a K/V byte: the warp tensor path is enough.
// Every warp is on its own: it takes a unit of work (a sequence, a kv head's group of up
// to 8 query heads, a chunk of pages_per_split pages) off a counter, streams the unit's
// pages through three stages with one bulk copy a page and writes the unit's partial from
// its registers. The next unit is taken and its first pages are ordered while the present
// one is computed, so the stream does not break between units. Scores are transposed,
// S^T[token, head] = K Q^T (M = 16 tokens = a page, N = 8 heads), and O^T += V^T P^T.
//
// Measured (B200, 16 query over 2 kv heads of 256 unless said):
//   8 groups of 8 sequences, prefixes of 16,272 and tails of U[1, 2048] tokens (402 MB)
//     73.9 us, 5.4 TB/s, 83 % of a plain copy's rate: HBM, but for 5 us of start and 8 of
//     the last CTAs' parts and the merge
//   128 sequences on 8,208 tokens, tails of U[1, 1024] (153 MB) 47.5 us: the prefix's eight
//     tiles read it from the L2 and their products, the tails' loads and both softmaxes
//     share the SMs for 40 us; the tails alone take 35
//   3 groups of 5 on 5,104, tails of U[1, 777], 24 over 8 heads of 128 (87 MB) 24.3 us
//   8 on 2,048, tails of U[1, 64] (5 MB) 12.4 us: the chain of three kernels (8 + 4 us)
#include <cudaTypedefs.h>
#include <math_constants.h>

#include <algorithm>
#include <mutex>

#include "tc.cuh"

namespace sc {
namespace {

constexpr int kPageTok = 16;
constexpr int kRowsTile = 128;
constexpr int kSoftThreads = 256;
constexpr int kTmaWarp = 8, kMmaWarp = 10;  // kTmaWarp: K, the next one: V
constexpr int kPrefixThreads = 352;
constexpr int kSoftBar = 1;      // named barrier of the softmax warps
constexpr float kRescale = 8.f;  // log2 units

template <int D>
struct PrefixShape {
  static constexpr int TOK = D == 256 ? 64 : 128;  // tokens of a tile
  static constexpr int PAGES = TOK / kPageTok;
  static constexpr int PAGE_BYTES = kPageTok * D * 2;  // K or V of a page
  static constexpr int TILE_BYTES = TOK * D * 2;   // K or V
  static constexpr int STAGES = 65536 / TILE_BYTES;
  static constexpr int SMEM = 2 * STAGES * TILE_BYTES + 2 * kRowsTile * 4 + 256;
  // The partials leave through shared memory, kPiece columns of a thread's row at a time.
  static constexpr int PIECE = D == 64 ? 32 : 64, PITCH = PIECE * 4 + 16;
  static_assert(kSoftThreads * PITCH <= 2 * STAGES * TILE_BYTES, "epilogue staging");
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
  int* counters;            // the tail's work counters, one per slab of rows
  long long num_pages;
  float scale_log2;
  int B, Hq, Hkv, G, max_pages, pages_per_split, num_splits, slabs;
  unsigned int* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// L2 policy of the K/V reads: first to go, so that the parts stay for the merge (8 groups
// of 8 sequences on 16k tokens 73.9 us, 76.1 without it, 75.6 with it for the prefix
// alone; 3 of 5 on 5k 24.1 and 25.9). The tiles of one prefix read a page at about the
// same time and lose nothing (128 sequences on one of 8k 47.9 and 47.7).
__device__ __forceinline__ uint64_t read_once() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}

__device__ __forceinline__ void bulk_g2s_once(void* dst, const void* src, uint32_t bytes,
                                              uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1], %2, [%3], %4;" ::"r"(smem_addr(dst)),
      "l"(src), "r"(bytes), "r"(smem_addr(bar)), "l"(policy)
      : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                            int c2, int c3, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(c0), "r"(c1), "r"(c2),
      "r"(c3), "l"(policy)
      : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}

// tc::mma_bf16_ts on the lane with `elected` set, from converged code.
__device__ __forceinline__ void mma_elected(uint32_t elected, uint32_t d_tmem, uint32_t a_tmem,
                                            uint64_t b_desc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :
      : "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate ? 1u : 0u),
        "r"(elected)
      : "memory");
}

// The same, but the rows (TMEM lanes) whose bits are set in `off` keep what D held.
__device__ __forceinline__ void mma_elected_rows(uint32_t elected, uint32_t d_tmem,
                                                 uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                                 const uint32_t (&off)[4], bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%6, %7, %8, %9}, p;\n\t}"
      :
      : "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate ? 1u : 0u),
        "r"(elected), "r"(off[0]), "r"(off[1]), "r"(off[2]), "r"(off[3])
      : "memory");
}

// Barrier of the softmax warps that ORs a predicate over them.
__device__ __forceinline__ bool soft_any(bool pred) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((int)pred), "r"(kSoftBar), "r"(kSoftThreads)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void soft_sync() {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(kSoftBar), "r"(kSoftThreads) : "memory");
}

// 112 registers: three of the eleven warps share a quarter of the SM's registers with a
// warp of the tail kernel (168 at D = 256), or no tail CTA would fit beside this one.
template <int D>
__global__ void __maxnreg__(112)
    prefix_kernel(const __grid_constant__ CUtensorMap half_pages,
                  const __grid_constant__ CUtensorMap whole_pages, const PrefixArgs a) {
  using S = PrefixShape<D>;
  // All shared memory is dynamic: it then starts at a multiple of 1024 bytes, as the
  // swizzled tiles need, and there is no room on the SM for slack beside a tail CTA.
  extern __shared__ __align__(1024) uint8_t sm[];
  float(*s_half)[kRowsTile] =  // a row's value of each column half
      reinterpret_cast<float(*)[kRowsTile]>(sm + 2 * S::STAGES * S::TILE_BYTES);
  uint64_t* kfull = reinterpret_cast<uint64_t*>(s_half + 2);
  uint64_t* vfull = kfull + S::STAGES;
  uint64_t* kfree = vfull + S::STAGES;
  uint64_t* vfree = kfree + S::STAGES;
  uint64_t* sfull = vfree + S::STAGES;  // [2] scores of a tile are in TMEM
  uint64_t* pfull = sfull + 2;          // [2] its P is
  uint64_t* ofull = pfull + 2;          // [2] O has taken it
  uint64_t* qfull = ofull + 2;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(qfull + 1);
  int& s_pages = *reinterpret_cast<int*>(s_tmem + 1);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform
  const int split = blockIdx.x, kvh = blockIdx.y;
  if (tid == 0) {
    s_pages = 0;
    for (int i = 0; i < S::STAGES; ++i) {
      mbar_init(&kfull[i], 1);
      mbar_init(&vfull[i], 1);
      mbar_init(&kfree[i], 1);
      mbar_init(&vfree[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], kSoftThreads);
      mbar_init(&ofull[i], 1);
    }
    mbar_init(qfull, kSoftThreads);
    fence_mbar_init();
  }
  pdl_wait();
  if (tid == 0 && blockIdx.x + blockIdx.y + blockIdx.z == 0) {
    // The tail starts once every CTA has triggered; its counters are zero by then.
    for (int i = 0; i < a.slabs; ++i) atomicExch(a.counters + i, 0);
    __threadfence();
  }
  __syncthreads();
  pdl_trigger();

  const int4 tile = a.tiles[blockIdx.z];
  const int p0 = split * a.pages_per_split;
  const bool misplaced = (smem_addr(sm) & 1023u) != 0;  // never seen; better void than wrong
  const bool bad =
      tile.w < 0 || tile.w >= a.B || tile.z > a.max_pages || tile.y * a.G > kRowsTile;
  if (p0 >= tile.z || misplaced || bad) {  // uniform over the CTA
    if (tid == 0 && p0 < tile.z)
      flag_device(a.status, bad ? DEV_BAD_INDEX : DEV_WAIT_TIMEOUT);
    return;
  }
  // All of TMEM, while the others load: after the wait (a CTA of the kernel before this one
  // might still have had to take its own); the kernels that start beside this one use none.
  if (warp == kMmaWarp) tc::tmem_alloc(s_tmem, 512);
  tc::fence_before();
  // What the first tile needs is ordered before the contexts are looked at. The softmax
  // warps read 16 rows of q each, a row by neighbouring lanes; the copy warps the ids of
  // the first tile's pages.
  constexpr int kChunks = D / 8, kRowsAtOnce = 32 / kChunks;  // 16-byte chunks of a row
  const auto row_of = [&](int r) {  // row r of the tile: its row of q, -1: none
    const int member = r / a.G, b = member < tile.y ? a.members[tile.x + member] : -1;
    return b >= 0 && b < a.B ? b * a.Hq + kvh * a.G + (r - member * a.G) : -1;
  };
  // A member attends here to the whole pages of its context; a page that its context
  // ends in is its tail's. Pages that no member attends to are not read.
  const auto pages_of = [&](int b) { return min(tile.z, max(a.ctx_len[b], 0) / kPageTok); };
  int reach = 0;
  if (tid < tile.y) {
    const int b = a.members[tile.x + tid];
    if (b >= 0 && b < a.B)
      reach = pages_of(b);
    else
      flag_device(a.status, DEV_BAD_INDEX);
  }
  uint4 q[kChunks / 2];
  int first_page = 0;
  const int which = warp == kTmaWarp ? 0 : 1;  // of the copy warps: K (half pages), V (pages)
  const int pg = which ? lane : lane >> 1;
  const int32_t* table = a.block_table + (size_t)tile.w * a.max_pages + p0;
  if (warp < kTmaWarp) {
    const int mine = lane < 16 ? row_of(16 * warp + lane) : -1;
#pragma unroll
    for (int j = 0; j < kChunks / 2; ++j) {
      const int from = __shfl_sync(0xffffffffu, mine, j * kRowsAtOnce + lane / kChunks);
      q[j] = from < 0 ? make_uint4(0u, 0u, 0u, 0u)
                      : reinterpret_cast<const uint4*>(a.q)[(size_t)from * kChunks + lane % kChunks];
    }
  } else if (warp < kMmaWarp && pg < S::PAGES && p0 + pg < tile.z) {
    first_page = table[pg];
  }
  if (reach > 0) atomicMax(&s_pages, reach);
  const bool stop = a.status != nullptr &&
                    (*reinterpret_cast<volatile unsigned int*>(a.status) & DEV_WAIT_TIMEOUT);
  // After a bounded wait has given up on this device, later CTAs stop at once.
  const bool stopped = __syncthreads_or(stop);
  tc::fence_after();
  const uint32_t tmem = *s_tmem;
  const int npages = min(p0 + a.pages_per_split, s_pages) - p0;
  if (stopped || npages <= 0) {
    if (warp == kMmaWarp) tc::tmem_dealloc(tmem, 512);
    return;
  }
  const int ntiles = (npages + S::PAGES - 1) / S::PAGES;

  // Every wait is bounded. After one has given up (the status word says so) a role runs
  // on without waiting, so that the others' barriers still complete; the results are void.
  bool ok = true;
  const auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (ok) ok = mbar_wait_bounded(bar, parity, a.status);
  };

  if (warp == kTmaWarp || warp == kTmaWarp + 1) {
    // ---------------------------------------------------------------- TMA
    // One box a lane: half pages of K, pages of V.
    const int boxes = which ? S::PAGES : 2 * S::PAGES;
    const int box_bytes = which ? S::PAGE_BYTES : S::PAGE_BYTES / 2;
    const bool moves = lane < boxes;
    uint64_t *full = which ? vfull : kfull, *freed = which ? vfree : kfree;
    const CUtensorMap* map = which ? &whole_pages : &half_pages;
    const auto page_of = [&](int i) {  // pages past the end repeat the last one (masked)
      return moves && i < ntiles ? table[min(i * S::PAGES + pg, npages - 1)] : 0;
    };
    const uint64_t once = read_once();
    const int last = npages - 1;
    int page = __shfl_sync(0xffffffffu, first_page, min(pg, last) * (which ? 1 : 2) & 31);
    if (!moves) page = 0;
    if (which) wait(qfull, 0);  // q lies where V goes
    for (int i = 0; i < ntiles; ++i) {
      const int next = page_of(i + 1);
      const int st = i % S::STAGES, round = i / S::STAGES;
      if (page < 0 || page >= a.num_pages) {
        flag_device(a.status, DEV_BAD_INDEX);
        page = 0;  // keep the copy in bounds; the status word reports the fault
      }
      if (i >= S::STAGES) wait(&freed[st], (round - 1) & 1);
      if (lane == 0) mbar_arrive_expect_tx(&full[st], S::TILE_BYTES);
      __syncwarp();
      if (moves)
        tma_load_4d(smem_addr(sm + (which * S::STAGES + st) * S::TILE_BYTES + lane * box_bytes),
                    map, 0, which ? 0 : 8 * (lane & 1), 0, (page * a.Hkv + kvh) * 2 + which,
                    &full[st], once);
      page = next;
    }
    __syncwarp();
    // The last copy into each stage has landed before the CTA ends.
    ok = true;
    if (lane == 0)
      for (int i = max(0, ntiles - S::STAGES); i < ntiles; ++i)
        wait(&full[i % S::STAGES], (i / S::STAGES) & 1);
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------------- MMA
    constexpr uint32_t kIdS = tc::idesc_bf16(kRowsTile, S::TOK, false, false);
    constexpr uint32_t kIdO = tc::idesc_bf16(kRowsTile, D, false, true);
    const uint32_t one = elect();
    const auto scores = [&](int i) {
      const int st = i % S::STAGES;
      wait(&kfull[st], (i / S::STAGES) & 1);
      tc::fence_after();
      __syncwarp();
      const uint32_t kb = smem_addr(sm + st * S::TILE_BYTES);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        mma_elected(one, tmem + S::T_S + (i & 1) * S::TOK, tmem + S::T_Q + 8 * kk,
                    tc::smem_desc(kb + (kk / 4) * 1024 + (kk % 4) * 32, 16, S::PAGE_BYTES / 2),
                    kIdS, kk > 0);
      if (one) {
        tc::commit(&sfull[i & 1]);
        tc::commit(&kfree[st]);
      }
      __syncwarp();
    };
    // A row's O takes the pages that the row attends to and no others: a page past its context
    // may hold an Inf or NaN that another member wrote, and 0 * Inf would be in its sum. Lane
    // j: the page of this split at which rows j, j + 32, j + 64 and j + 96 end.
    int end[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int row = row_of(lane + 32 * x);
      end[x] = row < 0 ? npages : min(pages_of(row / a.Hq) - p0, npages);
    }
    wait(qfull, 0);
    tc::fence_after();
    scores(0);
    const bool uneven = __any_sync(0xffffffffu, min(min(end[0], end[1]), min(end[2], end[3])) < npages);
    for (int i = 0; i < ntiles; ++i) {
      if (i + 1 < ntiles) scores(i + 1);
      const int st = i % S::STAGES;
      wait(&vfull[st], (i / S::STAGES) & 1);
      wait(&pfull[i & 1], (i >> 1) & 1);
      tc::fence_after();
      __syncwarp();
      const uint32_t vb = smem_addr(sm + (S::STAGES + st) * S::TILE_BYTES);
      const uint32_t pb = tmem + S::T_S + (i & 1) * S::TOK;
      const int page0 = i * S::PAGES, pages = npages - page0;
      if (!uneven && pages >= S::PAGES) {
#pragma unroll
        for (int kk = 0; kk < S::PAGES; ++kk)
          mma_elected(one, tmem, pb + 8 * kk, tc::smem_desc(vb + kk * S::PAGE_BYTES, 2048, 1024),
                      kIdO, i > 0 || kk > 0);
      } else {  // a product is a page: of the last tile those that are there
#pragma unroll 1
        for (int kk = 0; kk < min(S::PAGES, pages); ++kk) {
          uint32_t off[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) off[x] = __ballot_sync(0xffffffffu, end[x] <= page0 + kk);
          mma_elected_rows(one, tmem, pb + 8 * kk,
                           tc::smem_desc(vb + kk * S::PAGE_BYTES, 2048, 1024), kIdO, off,
                           i > 0 || kk > 0);
        }
      }
      if (one) {
        tc::commit(&ofull[i & 1]);
        tc::commit(&vfree[st]);
      }
      __syncwarp();
    }
    ok = true;  // no product is in flight when TMEM goes back
    wait(&ofull[(ntiles - 1) & 1], ((ntiles - 1) >> 1) & 1);
  } else {
    // ---------------------------------------------------------------- softmax
    constexpr int kCols = S::TOK / 2;   // this thread's columns of a tile
    constexpr int kOut = D / 2;         // and of O and Q
    const int half = warp >> 2, r = tid & (kRowsTile - 1);
    const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);  // this warp's TMEM lanes
    const int out_row = row_of(r);
    const bool live = out_row >= 0;
    const bool idle = !__any_sync(0xffffffffu, live);  // no row here: only the barriers
    // Pages of this split that the row attends to (its context may end inside the prefix).
    const int limit = live ? min(pages_of(out_row / a.Hq) - p0, npages) : 0;
    // A negative scale turns q, so that the largest score stays the largest; a zero one
    // clears it.
    const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    const uint32_t keep = a.scale_log2 == 0.f || !live ? 0u : 0xffffffffu;
    const float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);
    {
      // q turns from a row by 8 to 32 lanes to a row a lane in the V stages, whose copies
      // wait for it; chunk c of row r at c ^ r keeps both ways free of bank conflicts.
      uint8_t* turn = sm + S::STAGES * S::TILE_BYTES;
      const auto chunk = [&](int row, int c) {
        return reinterpret_cast<uint4*>(turn + row * (D * 2) + ((c ^ (row & (kChunks - 1))) * 16));
      };
#pragma unroll
      for (int j = 0; j < kChunks / 2; ++j)
        *chunk(16 * warp + j * kRowsAtOnce + lane / kChunks, lane % kChunks) = q[j];
      soft_sync();
#pragma unroll
      for (int c = 0; c < kOut / 32; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint4 u = *chunk(r, half * (kChunks / 2) + 4 * c + x);
          w[4 * x] = u.x;
          w[4 * x + 1] = u.y;
          w[4 * x + 2] = u.z;
          w[4 * x + 3] = u.w;
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) w[x] = (w[x] ^ flip) & keep;
        tc::tmem_st16(mine + S::T_Q + half * (kOut / 2) + 16 * c, w);
      }
      fence_proxy_async_smem();
      tc::tmem_wait_st();
      tc::fence_before();
      mbar_arrive(qfull);
    }
    float m = -CUDART_INF_F, l = 0.f;  // reference maximum (log2 units), this half's sum
    const auto grows = [&](float top) {
      return top > m + kRescale || (m == -CUDART_INF_F && top > m);
    };
    for (int i = 0; i < ntiles; ++i) {
      if (idle) {
        if (soft_any(false)) soft_sync();
        mbar_arrive(&pfull[i & 1]);
        continue;
      }
      wait(&sfull[i & 1], (i >> 1) & 1);
      tc::fence_after();
      const uint32_t st = mine + S::T_S + (i & 1) * S::TOK;
      float x[kCols];
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) tc::tmem_ld32(st + half * kCols + 32 * c, x + 32 * c);
      const int left = limit - i * S::PAGES - half * (S::PAGES / 2);  // pages that count
      if (left < S::PAGES / 2)
#pragma unroll
        for (int c = 0; c < kCols; ++c) x[c] = c / kPageTok < left ? x[c] : -CUDART_INF_F;
      float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
      for (int c = 0; c < kCols; ++c) mx[c & 3] = fmaxf(mx[c & 3], x[c]);
      float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
      // Past this barrier both halves have read their scores (P goes over them).
      tc::fence_before();
      const bool any = soft_any(grows(top));
      tc::fence_after();
      if (any) {
        s_half[half][r] = top;
        soft_sync();
        top = fmaxf(top, s_half[half ^ 1][r]);
        const float to = grows(top) ? top : m;
        const float f = m == to ? 1.f : ex2(m - to);  // 0 from -inf
        if (i > 0) {
          wait(&ofull[(i - 1) & 1], ((i - 1) >> 1) & 1);
          tc::fence_after();
#pragma unroll 1
          for (int c = 0; c < kOut / 32; ++c) {
            float o[32];
            tc::tmem_ld32(mine + half * kOut + 32 * c, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= f;
            tc::tmem_st32(mine + half * kOut + 32 * c, o);
          }
        }
        l *= f;
        m = to;
      }
      const float ref = m == -CUDART_INF_F ? 0.f : m;  // nothing seen yet: every p is 0
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kCols / 32; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float y0 = ex2(fmaf(x[32 * c + 2 * e], scale, -ref));
          const float y1 = ex2(fmaf(x[32 * c + 2 * e + 1], scale, -ref));
          sum[(2 * e) & 3] += y0;
          sum[(2 * e + 1) & 3] += y1;
          w[e] = pack_bf16x2(y0, y1);
        }
        tc::tmem_st16(st + half * (kCols / 2) + 16 * c, w);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tc::tmem_wait_st();
      tc::fence_before();
      mbar_arrive(&pfull[i & 1]);
    }
    wait(&ofull[(ntiles - 1) & 1], ((ntiles - 1) >> 1) & 1);
    tc::fence_after();
    soft_sync();  // s_half's last readers are done
    s_half[half][r] = l;
    soft_sync();
    l += s_half[half ^ 1][r];
    const float inv = l > 0.f ? 1.f / l : 0.f;
    // The parts leave through the stages, which no copy or product uses any more: a piece
    // of the warp's 32 rows, a row a lane, then a row by neighbouring lanes.
    constexpr int kLanes = S::PIECE / 4, kRowsOut = 32 / kLanes;  // of a row, of a store
    uint8_t* stage = sm + warp * 32 * S::PITCH;
    if (!idle && __all_sync(0xffffffffu, ok)) {
#pragma unroll 1
      for (int c = 0; c < kOut; c += S::PIECE) {
#pragma unroll
        for (int p = 0; p < S::PIECE / 32; ++p) {
          float o[32];
          tc::tmem_ld32(mine + half * kOut + c + 32 * p, o);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            reinterpret_cast<float4*>(stage + lane * S::PITCH + 128 * p)[e] = make_float4(
                o[4 * e] * inv, o[4 * e + 1] * inv, o[4 * e + 2] * inv, o[4 * e + 3] * inv);
        }
        __syncwarp();
#pragma unroll 8
        for (int i = 0; i < kLanes; ++i) {
          const int from = i * kRowsOut + lane / kLanes, col = lane % kLanes;
          const int to = __shfl_sync(0xffffffffu, out_row, from);
          const float4 v = reinterpret_cast<const float4*>(stage + from * S::PITCH)[col];
          if (to >= 0)
            reinterpret_cast<float4*>(a.part_out + ((size_t)to * a.num_splits + split) * D +
                                      half * kOut + c)[col] = v;
        }
        __syncwarp();
      }
    }
    if (live && half == 0)
      a.part_lse[(size_t)out_row * a.num_splits + split] =
          l > 0.f ? (m + log2f(l)) * 0.6931471805599453f
                  : (l == 0.f ? -CUDART_INF_F : l);  // a NaN stays one
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tc::tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------- the sequences' own pages
// Two warps with three pages each in flight; four with three halves of a page each (the same
// memory) took as long: 12.3 / 75.7 / 48.5 / 26.3 us for the cases above, where two took
// 12.2 / 76.1 / 47.8 / 25.8.
constexpr int kTailWarps = 2;
constexpr int kTailStages = 3;
constexpr int kTailHeads = 8;        // query heads of a unit
constexpr int kSlabRows = 1024;      // rows whose units one counter hands out

struct TailArgs {
  const uint16_t *q, *kv_pool;
  const int32_t *block_table, *ctx_len, *first_page;
  float *part_out, *part_lse;
  int* counters;
  long long num_pages;
  float scale_log2;
  int B, Hq, Hkv, G, HG, max_pages, pages_per_split, num_splits;
  unsigned int* status;
};

// A row's own pages, [skip, skip + pages) of its block table, and the tokens they hold.
struct OwnPages {
  int skip, pages, tokens;
};
__device__ __forceinline__ OwnPages own_pages(int ctx, int first_page, int max_pages) {
  OwnPages o;
  ctx = (int)max(0ll, min((long long)ctx, (long long)max_pages * kPageTok));
  // A page that the context ends in is never left to the prefix.
  o.skip = min(max(0, min(first_page, max_pages)), ctx / kPageTok);
  o.tokens = ctx - o.skip * kPageTok;
  o.pages = (o.tokens + kPageTok - 1) / kPageTok;
  return o;
}

// kLong: units of more than 32 pages, whose ids the warp's lanes read 32 at a time. With that in
// every launch 128 sequences on 8,208 tokens took 48.9 us, without 47.8.
template <int D, bool kLong>
__global__ void __maxnreg__(168) tail_kernel(const TailArgs a) {
  constexpr int ROW = D * 2, KV = kPageTok * ROW, STAGE = 2 * KV, KSTEPS = D / 16;
  constexpr unsigned kAll = 0xffffffffu;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* stage = smem + warp * kTailStages * STAGE;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kTailWarps * kTailStages * STAGE) +
                  warp * kTailStages;
  int* chunks_to = reinterpret_cast<int*>(  // chunks of the slab's rows up to 32 i + 31
      smem + kTailWarps * kTailStages * (STAGE + sizeof(uint64_t)));
  pdl_trigger();
  const int slab = blockIdx.y, row0 = slab * kSlabRows;
  const int rows = min(kSlabRows, a.B - row0);
  const int groups = a.Hkv * a.HG;
  const auto take = [&]() {
    int t = 0;
    if (lane == 0) t = atomicAdd(a.counters + slab, 1);
    return t;
  };
  const int t_first = take();
  if (lane == 0) {
    for (int i = 0; i < kTailStages; ++i) mbar_init(&bar[i], 1);
    fence_mbar_init();
  }
  const auto own_of = [&](int r) {
    return r < rows ? own_pages(a.ctx_len[row0 + r], a.first_page[row0 + r], a.max_pages)
                    : OwnPages{0, 0, 0};
  };
  const auto chunks_of = [&](const OwnPages& o) {
    return min((o.pages + a.pages_per_split - 1) / a.pages_per_split, a.num_splits);
  };
#pragma unroll 4
  for (int i = warp; 32 * i < rows; i += kTailWarps) {
    const int sum = (int)__reduce_add_sync(kAll, (unsigned)chunks_of(own_of(32 * i + lane)));
    if (lane == 0) chunks_to[i] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    int incl = 32 * lane < rows ? chunks_to[lane] : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(kAll, incl, off);
      if (lane >= off) incl += y;
    }
    chunks_to[lane] = incl;
  }
  __syncthreads();

  struct Unit {
    int b, kvh, head0, heads, split, n, tokens;  // n pages; tokens of them count
    int first;                                   // (kLong) the first one's place in the table
    int page;                                    // lane i: the id of page i of 32
  };
  // Unit t of the slab: chunk t / groups of the rows' chunks laid end to end. Uniform over
  // the warp; u.n == 0 past the last one.
  const auto resolve = [&](int t) {
    Unit u;
    t = __shfl_sync(kAll, t, 0);
    const int want = t / groups, hg = t - want * groups;
    u.n = 0;
    const unsigned past = __ballot_sync(kAll, want < chunks_to[lane]);
    if (past == 0u) return u;
    const int block = __ffs(past) - 1;
    const OwnPages o = own_of(32 * block + lane);
    const int mine = chunks_of(o);
    int incl = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(kAll, incl, off);
      if (lane >= off) incl += y;
    }
    const int left = want - (block > 0 ? chunks_to[block - 1] : 0);
    const int src = __ffs(__ballot_sync(kAll, left < incl)) - 1;
    const int chunk = left - (__shfl_sync(kAll, incl, src) - __shfl_sync(kAll, mine, src));
    const int skip = __shfl_sync(kAll, o.skip, src), pages = __shfl_sync(kAll, o.pages, src);
    const int tokens = __shfl_sync(kAll, o.tokens, src);
    const int p0 = chunk * a.pages_per_split;
    u.b = row0 + 32 * block + src;
    u.split = chunk;
    u.n = min(a.pages_per_split, pages - p0);
    u.tokens = min(u.n * kPageTok, tokens - p0 * kPageTok);
    if constexpr (kLong) u.first = skip + p0;
    u.page = lane < u.n ? a.block_table[(size_t)u.b * a.max_pages + skip + p0 + lane] : 0;
    u.kvh = hg / a.HG;
    u.head0 = u.kvh * a.G + (hg - u.kvh * a.HG) * kTailHeads;
    u.heads = min(kTailHeads, (u.kvh + 1) * a.G - u.head0);
    return u;
  };

  const uint64_t once = read_once();
  int issued = 0, consumed = 0;  // pages of all units, in order through the stages
  const auto issue = [&](Unit& u, int i) {
    if constexpr (kLong)
      if (i > 0 && (i & 31) == 0)
        u.page = i + lane < u.n
                     ? a.block_table[(size_t)u.b * a.max_pages + u.first + i + lane] : 0;
    int page = __shfl_sync(kAll, u.page, kLong ? i & 31 : i);
    if (lane == 0) {
      if (page < 0 || page >= a.num_pages) {
        flag_device(a.status, DEV_BAD_INDEX);
        page = 0;  // keep the copy in bounds; the status word reports the fault
      }
      const int s = issued % kTailStages;
      // The stage may hold rows that the warp cleared with ordinary stores (a page that its
      // context ended in); a __syncwarp stands between those and every issue.
      fence_proxy_async_smem();
      mbar_arrive_expect_tx(&bar[s], STAGE);
      bulk_g2s_once(
          stage + s * STAGE,
          reinterpret_cast<const uint8_t*>(a.kv_pool) + ((size_t)page * a.Hkv + u.kvh) * STAGE,
          STAGE, &bar[s], once);
    }
    ++issued;
  };
  const int mi = lane >> 3, r8 = lane & 7;
  const int tk = r8 + 8 * (mi & 1);   // token row this lane addresses for K
  const int tv = r8 + 8 * (mi >> 1);  // token row this lane addresses for V^T
  // After a bounded wait has given up on this device, later CTAs take no work.
  bool ok = a.status == nullptr ||
            !(*reinterpret_cast<volatile unsigned int*>(a.status) & DEV_WAIT_TIMEOUT);
  ok = __all_sync(kAll, ok);
  Unit cur;
  cur.n = 0;
  if (ok) cur = resolve(t_first);
  int cur_issued = 0;
  // Q^T as the B operand: b0 = q[n][16kk + 2c .. +1], b1 = q[n][16kk + 8 + 2c .. +1].
  uint32_t qf[KSTEPS][2];
  const auto load_q = [&](const Unit& u) {
    const int n = lane >> 2, c = lane & 3;
    const bool valid = n < u.heads;
    const uint16_t* qp = a.q + ((size_t)u.b * a.Hq + u.head0 + (valid ? n : 0)) * D;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      qf[kk][0] = valid ? *reinterpret_cast<const uint32_t*>(qp + 16 * kk + 2 * c) : 0u;
      qf[kk][1] = valid ? *reinterpret_cast<const uint32_t*>(qp + 16 * kk + 8 + 2 * c) : 0u;
    }
  };
  if (cur.n > 0) load_q(cur);
  while (ok && cur.n > 0) {
    while (issued - consumed < kTailStages && cur_issued < cur.n) issue(cur, cur_issued++);
    const int t_next = take();
    Unit nxt;
    nxt.n = 0;
    int nxt_issued = 0;
    bool have_next = false;
    float m0 = -CUDART_INF_F, m1 = -CUDART_INF_F;  // running max of heads 2c, 2c+1 (log2 units)
    float l0 = 0.f, l1 = 0.f;                      // this lane's partial sums
    float o[KSTEPS][4];
#pragma unroll
    for (int mt = 0; mt < KSTEPS; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
    for (int j = 0; j < cur.n; ++j) {
      if (cur_issued == cur.n && !have_next) {
        nxt = resolve(t_next);
        have_next = true;
        while (issued - consumed < kTailStages && nxt_issued < nxt.n) issue(nxt, nxt_issued++);
      }
      const int s = consumed % kTailStages;
      ok = mbar_wait_bounded(&bar[s], (consumed / kTailStages) & 1, a.status);
      ok = __all_sync(kAll, ok);
      if (!ok) break;
      const uint32_t kbase = smem_addr(stage + s * STAGE), vbase = kbase + KV;
      const int left = cur.tokens - j * kPageTok;  // tokens of the page that count
      if (left < kPageTok) {
        // Rows past the context hold whatever the pool held (possibly Inf/NaN bits); their
        // probability is 0, but 0 * Inf would poison the sum.
        uint4* vrows = reinterpret_cast<uint4*>(stage + s * STAGE + KV);
        for (int c = left * (ROW / 16) + lane; c < kPageTok * (ROW / 16); c += 32)
          vrows[c] = make_uint4(0u, 0u, 0u, 0u);
        __syncwarp();
      }
      float sa[2][4];  // two accumulators halve the dependent chain of the scores
#pragma unroll
      for (int x = 0; x < 2; ++x) sa[x][0] = sa[x][1] = sa[x][2] = sa[x][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) {
        const int chunk = 2 * kk + (mi >> 1);
        uint32_t a0, a1, a2, a3;
        ldsm_x4(kbase + tk * ROW + ((chunk ^ (tk & 7)) << 4), a0, a1, a2, a3);
        mma_bf16_16816(sa[kk & 1], a0, a1, a2, a3, qf[kk][0], qf[kk][1]);
      }
      const int tok = lane >> 2;
      const bool lo = tok < left, hi = tok + 8 < left;
      const float x0 = lo ? (sa[0][0] + sa[1][0]) * a.scale_log2 : -CUDART_INF_F;
      const float x1 = lo ? (sa[0][1] + sa[1][1]) * a.scale_log2 : -CUDART_INF_F;
      const float x2 = hi ? (sa[0][2] + sa[1][2]) * a.scale_log2 : -CUDART_INF_F;
      const float x3 = hi ? (sa[0][3] + sa[1][3]) * a.scale_log2 : -CUDART_INF_F;
      float t0 = fmaxf(x0, x2), t1 = fmaxf(x1, x3);
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) {
        t0 = fmaxf(t0, __shfl_xor_sync(kAll, t0, off));
        t1 = fmaxf(t1, __shfl_xor_sync(kAll, t1, off));
      }
      // The maxima are -inf while every score is (a key of -Inf): each p is 0 then.
      const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
      const float r0 = n0 == -CUDART_INF_F ? 0.f : n0, r1 = n1 == -CUDART_INF_F ? 0.f : n1;
      const float c0 = exp2f(m0 - r0), c1 = exp2f(m1 - r1);
      const float p0 = exp2f(x0 - r0), p1 = exp2f(x1 - r1);
      const float p2 = exp2f(x2 - r0), p3 = exp2f(x3 - r1);
      l0 = fmaf(l0, c0, p0 + p2);
      l1 = fmaf(l1, c1, p1 + p3);
      m0 = n0;
      m1 = n1;
      const uint32_t pb0 = movmatrix_t(pack_bf16x2(p0, p1));
      const uint32_t pb1 = movmatrix_t(pack_bf16x2(p2, p3));
#pragma unroll
      for (int mt = 0; mt < KSTEPS; ++mt) {
        o[mt][0] *= c0;
        o[mt][1] *= c1;
        o[mt][2] *= c0;
        o[mt][3] *= c1;
        const int chunk = 2 * mt + (mi & 1);
        uint32_t a0, a1, a2, a3;
        ldsm_x4_t(vbase + tv * ROW + ((chunk ^ (tv & 7)) << 4), a0, a1, a2, a3);
        mma_bf16_16816(o[mt], a0, a1, a2, a3, pb0, pb1);
      }
      ++consumed;
      __syncwarp();
      if (cur_issued < cur.n)
        issue(cur, cur_issued++);
      else if (have_next && nxt_issued < nxt.n)
        issue(nxt, nxt_issued++);
    }
    if (!ok) break;
    if (nxt.n > 0) load_q(nxt);  // arrives while the partial is written
#pragma unroll
    for (int off = 4; off <= 16; off <<= 1) {
      l0 += __shfl_xor_sync(kAll, l0, off);
      l1 += __shfl_xor_sync(kAll, l1, off);
    }
    // O^T: this lane holds dims d0 + 16 mt (+ 8) of heads h0, h0 + 1.
    const int d0 = lane >> 2, h0 = 2 * (lane & 3);
    const float i0 = l0 == 0.f ? 0.f : 1.f / l0, i1 = l1 == 0.f ? 0.f : 1.f / l1;
    const size_t part = ((size_t)cur.b * a.Hq + cur.head0 + h0) * a.num_splits + cur.split;
    float* w0 = a.part_out + part * D + d0;
    float* w1 = w0 + (size_t)a.num_splits * D;
    if (h0 < cur.heads) {
#pragma unroll
      for (int mt = 0; mt < KSTEPS; ++mt) {
        w0[16 * mt] = o[mt][0] * i0;
        w0[16 * mt + 8] = o[mt][2] * i0;
      }
      if (d0 == 0) a.part_lse[part] = (m0 + log2f(l0)) * 0.6931471805599453f;
    }
    if (h0 + 1 < cur.heads) {
#pragma unroll
      for (int mt = 0; mt < KSTEPS; ++mt) {
        w1[16 * mt] = o[mt][1] * i1;
        w1[16 * mt + 8] = o[mt][3] * i1;
      }
      if (d0 == 0) a.part_lse[part + a.num_splits] = (m1 + log2f(l1)) * 0.6931471805599453f;
    }
    cur = nxt;
    cur_issued = nxt_issued;
  }
  // A wait gave up (already flagged): the copies in flight land before the CTA ends.
  for (; consumed < issued; ++consumed)
    if (!mbar_wait_bounded(&bar[consumed % kTailStages], (consumed / kTailStages) & 1, a.status)) break;
  // The grid ends after the prefix kernel's, so that what waits for this one waits for
  // both. One CTA sees to that; the others leave their SMs.
  if (blockIdx.x == 0 && blockIdx.y == 0) pdl_wait();
}

// The parts of each (sequence, head) row: those of its prefix, then its own tail's.
// kWarps warps share a row (a warp's lane holds D / 32 of its columns) and take its parts
// in turn. Which parts are there follows from the row's context; the loads do not wait for
// that: every place is read, kAhead of them per warp before anything is known.
constexpr int kMergeThreads = 256;
constexpr int kMergeMax = 1024;  // parts of one row

struct MergeArgs {
  const float *pre_out, *pre_lse, *tail_out, *tail_lse;
  const int32_t *ctx_len, *first_page;
  uint16_t* out;
  float* lse_out;
  int rows, Hq, max_pages, pre_pps, pre_splits, tail_pps, tail_splits;
  unsigned int* status;
};

template <int D, int kWarps>
__global__ void __launch_bounds__(kMergeThreads) merge_parts_kernel(const MergeArgs a) {
  constexpr int kPer = D / 32;                       // columns of a lane
  constexpr int kRows = kMergeThreads / 32 / kWarps; // rows of the CTA
  constexpr int kAhead = D == 256 ? 3 : 4;
  constexpr unsigned kAll = 0xffffffffu;
  __shared__ float acc_s[kMergeThreads / 32][kWarps > 1 ? D : 1];
  __shared__ float sum_s[kMergeThreads / 32];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = warp % kWarps;
  const int row = min(blockIdx.x * kRows + warp / kWarps, a.rows - 1);  // the last one twice
  const int total = a.pre_splits + a.tail_splits;
  const size_t pre = (size_t)row * a.pre_splits, own = (size_t)row * a.tail_splits;
  const auto lse_at = [&](int s) {
    return s < a.pre_splits ? a.pre_lse[pre + s] : a.tail_lse[own + s - a.pre_splits];
  };
  const auto load = [&](int s, float* v) {
    const float* o = s < a.pre_splits ? a.pre_out + (pre + s) * D
                                      : a.tail_out + (own + s - a.pre_splits) * D;
    if constexpr (kPer == 2) {
      const float2 u = reinterpret_cast<const float2*>(o)[lane];
      v[0] = u.x;
      v[1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < kPer / 4; ++i) {
        const float4 u = reinterpret_cast<const float4*>(o)[lane + 32 * i];
        v[4 * i] = u.x;
        v[4 * i + 1] = u.y;
        v[4 * i + 2] = u.z;
        v[4 * i + 3] = u.w;
      }
    }
  };
  float v[kAhead][kPer];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (w + i * kWarps < total) load(w + i * kWarps, v[i]);
  const float raw = lane < total ? lse_at(lane) : -CUDART_INF_F;
  const int b = row / a.Hq, ctx = a.ctx_len[b], first_page = a.first_page[b];
  const OwnPages o = own_pages(ctx, first_page, a.max_pages);
  const int need_pre = (o.skip + a.pre_pps - 1) / a.pre_pps;
  const int need_own = (o.pages + a.tail_pps - 1) / a.tail_pps;
  // A context outside the block table, or more pages than the splits cover: clamped.
  if (lane == 0 && (ctx < 0 || (long long)ctx > (long long)a.max_pages * kPageTok ||
                    first_page < 0 || first_page > a.max_pages || need_pre > a.pre_splits ||
                    need_own > a.tail_splits))
    flag_device(a.status, DEV_BAD_INDEX);
  const auto there = [&](int s) {
    return s < a.pre_splits ? s < need_pre : s - a.pre_splits < need_own && s < total;
  };
  const float first = there(lane) ? raw : -CUDART_INF_F;
  float m = first;
  for (int s = lane + 32; s < total; s += 32)
    if (there(s)) m = fmaxf(m, lse_at(s));
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, off));
  float acc[kPer], sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  const auto add = [&](float ls, const float* x) {
    if (ls == -CUDART_INF_F) return;  // an empty part holds nothing (a NaN weight passes)
    const float e = __expf(ls - m);
    sum += e;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = fmaf(e, x[i], acc[i]);
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int s = w + i * kWarps;
    if (s < 32) {
      add(__shfl_sync(kAll, first, s), v[i]);
    } else if (there(s)) {
      add(lse_at(s), v[i]);
    }
  }
#pragma unroll 1
  for (int s0 = w + kAhead * kWarps; s0 < total; s0 += kAhead * kWarps) {
    float ls[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int s = s0 + i * kWarps;
      ls[i] = -CUDART_INF_F;
      if (there(s)) {
        load(s, v[i]);
        ls[i] = lse_at(s);
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) add(ls[i], v[i]);
  }
  if constexpr (kWarps > 1) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc_s[warp][i * 32 + lane] = acc[i];
    if (lane == 0) sum_s[warp] = sum;
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int p = 1; p < kWarps; ++p) {
      sum += sum_s[warp + p];
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] += acc_s[warp + p][i * 32 + lane];
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* out = a.out + (size_t)row * D;
  if constexpr (kPer == 2) {
    reinterpret_cast<uint32_t*>(out)[lane] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  } else {
#pragma unroll
    for (int i = 0; i < kPer / 4; ++i)
      reinterpret_cast<uint2*>(out)[lane + 32 * i] =
          make_uint2(pack_bf16x2(acc[4 * i] * inv, acc[4 * i + 1] * inv),
                     pack_bf16x2(acc[4 * i + 2] * inv, acc[4 * i + 3] * inv));
  }
  if (lane == 0 && a.lse_out != nullptr)
    a.lse_out[row] = sum == 0.f ? -CUDART_INF_F : m + logf(sum);
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

// The pool as [block = (page, head, K|V)][64-column slice][token][64]: a box is `tokens`
// (8 or 16) tokens of a block, x always 0.
int encode_pool(CUtensorMap* map, const void* pool, int D, long long blocks, int tokens) {
  auto fn = encode_fn();
  if (fn == nullptr)
    return set_error(SC_ERR_CUDA, "sc_shared_prefix_attention: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[4] = {64, kPageTok, (cuuint64_t)D / 64, (cuuint64_t)blocks};
  cuuint64_t strides[3] = {(cuuint64_t)D * 2, 128, (cuuint64_t)kPageTok * D * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)tokens, (cuuint32_t)D / 64, 1};
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
int launch_shared(const CUtensorMap* maps, const PrefixArgs& p, const MergeArgs& m, int ntiles,
                  const TailArgs& t, cudaStream_t s) {
  const char* name = "sc_shared_prefix_attention";
  using S = PrefixShape<D>;
  constexpr size_t tail_smem =
      (size_t)kTailWarps * kTailStages * (2 * S::PAGE_BYTES + sizeof(uint64_t)) + 32 * sizeof(int);
  static int configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    cudaError_t err = cudaFuncSetAttribute(
        prefix_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    // All of the SM's memory as shared memory: a tail CTA goes beside this one.
    if (err == cudaSuccess)
      err = cudaFuncSetAttribute(prefix_kernel<D>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                 cudaSharedmemCarveoutMaxShared);
    for (auto tail : {tail_kernel<D, false>, tail_kernel<D, true>}) {
      if (err == cudaSuccess)
        err = cudaFuncSetAttribute(tail, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)tail_smem);
      if (err == cudaSuccess)
        err = cudaFuncSetAttribute(tail, cudaFuncAttributePreferredSharedMemoryCarveout,
                                   cudaSharedmemCarveoutMaxShared);
    }
    if (err != cudaSuccess)
      return set_error(SC_ERR_CUDA, "%s: smem attribute: %s", name, cudaGetErrorString(err));
    configured[dev] = 1;
  }
  cudaError_t err = launch_pdl(prefix_kernel<D>, dim3(p.num_splits, p.Hkv, ntiles),
                               dim3(kPrefixThreads), S::SMEM, s, maps[0], maps[1], p);
  if (err != cudaSuccess)
    return set_error(SC_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
  // Two CTAs an SM (one while a prefix CTA is there), fewer where there is less work.
  const long long units = (long long)std::min(p.B, kSlabRows) * t.Hkv * t.HG * t.num_splits;
  const int ctas = (int)std::min(2ll * 148, (units + kTailWarps - 1) / kTailWarps);
  err = launch_pdl(t.pages_per_split > 32 ? tail_kernel<D, true> : tail_kernel<D, false>,
                   dim3(ctas, p.slabs), dim3(kTailWarps * 32), tail_smem, s, t);
  if (err != cudaSuccess)
    return set_error(SC_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
  // As many warps a row (a power of two, at most 8) as the GPU holds at once. 128 rows of 8
  // sequences took 12.4 us of the whole call with 8, 13.3 with 2, 14.8 with 1; 1,024 rows
  // 73.9 with 4, 75.3 with 2, 76.2 with 8; 2,048 rows 47.9 with 2, 51.7 with 8.
  const int fit = 148 * 40 / m.rows;
  const int share = fit >= 8 ? 8 : fit >= 4 ? 4 : fit >= 2 ? 2 : 1;
  const auto merge = share == 8   ? merge_parts_kernel<D, 8>
                     : share == 4 ? merge_parts_kernel<D, 4>
                     : share == 2 ? merge_parts_kernel<D, 2>
                                  : merge_parts_kernel<D, 1>;
  const int per_cta = kMergeThreads / 32 / share;
  err = launch_pdl(merge, dim3((m.rows + per_cta - 1) / per_cta), dim3(kMergeThreads), 0, s, m);
  if (err != cudaSuccess)
    return set_error(SC_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
  return check_launch(name);
}

}  // namespace
}  // namespace sc

extern "C" int sc_shared_prefix_attention(
    const sc_bf16* q, const sc_bf16* kv_pool, int64_t num_pages, const int32_t* block_table,
    const int32_t* ctx_len, const int32_t* prefix_pages,
    const int32_t* tiles, const int32_t* members, int ntiles, int B, int Hq, int Hkv, int D, int P,
    int max_pages, int prefix_pages_per_split, int prefix_splits, int pages_per_split,
    int num_splits, float scale, float* prefix_out, float* prefix_lse, float* part_out,
    float* part_lse, int32_t* counters, sc_bf16* out, float* lse_out, void* stream) {
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
                 prefix_out && prefix_lse && part_out && part_lse && counters,
             SC_ERR_INVALID, "%s: null pointer", name);
  SC_REQUIRE(num_pages > 0 && max_pages > 0 && ntiles > 0 && prefix_pages_per_split > 0 &&
                 prefix_splits > 0 && pages_per_split > 0 && num_splits > 0,
             SC_ERR_INVALID, "%s: bad plan max_pages=%d ntiles=%d splits=%d x %d + %d x %d", name,
             max_pages, ntiles, prefix_splits, prefix_pages_per_split, num_splits, pages_per_split);
  SC_REQUIRE(prefix_splits + num_splits <= sc::kMergeMax, SC_ERR_INVALID,
             "%s: %d + %d splits, at most %d", name, prefix_splits, num_splits, sc::kMergeMax);
  SC_REQUIRE(B <= 65535 && ntiles <= 65535 && Hkv <= 65535 && Hkv * ((Hq / Hkv + 7) / 8) <= 65535 &&
                 num_pages * Hkv * 2 < (1ll << 31),
             SC_ERR_INVALID, "%s: grid or pool too large", name);
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  SC_REQUIRE(aligned(q) && aligned(kv_pool) && aligned(out) && aligned(prefix_out) &&
                 aligned(part_out) && aligned(tiles),
             SC_ERR_INVALID, "%s: operands must be 16-byte aligned", name);
  CUtensorMap maps[2];  // half pages (K), pages (V)
  for (int i = 0; i < 2; ++i)
    if (int rc = sc::encode_pool(&maps[i], kv_pool, D, num_pages * Hkv * 2, 8 * (i + 1))) return rc;
  sc::PrefixArgs p;
  p.q = q;
  p.block_table = block_table;
  p.ctx_len = ctx_len;
  p.tiles = reinterpret_cast<const int4*>(tiles);
  p.members = members;
  p.part_out = prefix_out;
  p.part_lse = prefix_lse;
  p.counters = counters;
  p.slabs = (B + sc::kSlabRows - 1) / sc::kSlabRows;
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
  m.rows = B * Hq;
  m.Hq = Hq;
  m.max_pages = max_pages;
  m.pre_pps = prefix_pages_per_split;
  m.pre_splits = prefix_splits;
  m.tail_pps = pages_per_split;
  m.tail_splits = num_splits;
  m.status = p.status;
  sc::TailArgs t;
  t.q = q;
  t.kv_pool = kv_pool;
  t.block_table = block_table;
  t.ctx_len = ctx_len;
  t.first_page = prefix_pages;
  t.part_out = part_out;
  t.part_lse = part_lse;
  t.counters = counters;
  t.num_pages = num_pages;
  t.scale_log2 = p.scale_log2;
  t.B = B;
  t.Hq = Hq;
  t.Hkv = Hkv;
  t.G = p.G;
  t.HG = (p.G + sc::kTailHeads - 1) / sc::kTailHeads;
  t.max_pages = max_pages;
  t.pages_per_split = pages_per_split;
  t.num_splits = num_splits;
  t.status = p.status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto launch = D == 64    ? sc::launch_shared<64>
                      : D == 128 ? sc::launch_shared<128>
                                 : sc::launch_shared<256>;
  return launch(maps, p, m, ntiles, t, s);
}
