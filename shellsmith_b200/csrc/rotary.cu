// Rotary positions with several axes, the q/k RMS norm and the KV append in one launch.
//
// Reference call site: studio_compute/mlx_decode.py:94-100, where mlx-vlm's
// `_prepare_projected_qkv` norms q and k per head, turns them by the token's
// absolute position (time, height, width for images and video) and appends k, v to
// the cache. Per token n and head, with x the head's D values:
//   y = x / sqrt(mean(x^2) + eps) * w          (where a weight is given)
//   t = pos[axis_i][n] * f_i,                  pair i < R / 2 of the R rotary dims
//   (y_i, y_{i + R/2}) <- (y_i cos t - y_{i+R/2} sin t, y_{i+R/2} cos t + y_i sin t)
// with every step in fp32 and one rounding to bf16 at the end (the norm's result is
// not rounded first: the turned value then carries one bf16 rounding, not two).
//
// The angle is reduced in double: at position 200,000 an fp32 product is off by up
// to 0.01 rad, more than a bf16 step of the result. f_i / (2 pi) is tabulated in
// double, so the reduction is one multiply and one subtraction of the nearest whole
// turn; sine and cosine of the remaining fraction are fp32.
//
// B200 mapping. HBM-bound: each value is read and written once. A CTA makes the (cos, sin)
// table of its tokens in shared memory, then each of its warps takes heads and walks the
// tokens of one, four rows loaded before the first is computed. D / 8 lanes hold a row, 8
// values each as two 4-value pieces: a lane of the rotary part holds both halves of four
// pairs, so that a turn needs no exchange, and the norm is a shuffle sum. Products go two
// at a time (fp32 pairs).
//
// Measured (B200, 16 + 2 + 2 heads of 256, three axes, 64 rotary dims): 16,381 tokens
// (336 MB) 64 us, 5.2 TB/s, 79 % of a plain copy's rate: half of the issue slots are busy
// and the writes to the pool's pages leave in pieces of a row; 85 us before the rows of a
// head were walked by one warp and products paired. 8 tokens 3.0 us, 256 tokens of 24 + 8 +
// 8 heads of 128 4.0 us: a launch, the table and one row. Operands off a 16-byte boundary (or strides that are)
// are read by the element: 256 tokens 5.5 us against 5.0 beside it, 16,381 85 against 63.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace sc {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 32;     // most tokens of one CTA

struct RotaryArgs {
  const uint16_t *q, *k, *v;
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head;  // strides in elements
  const int32_t* positions;
  long long pos_axis;                                     // stride between axes
  const double* turns;                                    // f_i / (2 pi)
  const int32_t* axis;
  const uint16_t *q_weight, *k_weight;
  uint16_t *q_out, *k_out, *pool;
  const int64_t* slots;
  long long num_pages;
  float eps;
  int ntok, Hq, Hkv, half, axes, P, page_shift;
  unsigned int* status;
};

// 4 consecutive bf16 of a row; without kVec the address has 2-byte alignment only.
template <bool kVec>
__device__ __forceinline__ uint2 load4(const uint16_t* p) {
  if constexpr (kVec)
    return *reinterpret_cast<const uint2*>(p);
  else
    return make_uint2((uint32_t)p[0] | ((uint32_t)p[1] << 16),
                      (uint32_t)p[2] | ((uint32_t)p[3] << 16));
}

__device__ __forceinline__ void unpack4(const uint2& u, float* x) {
  x[0] = bf16_lo(u.x);
  x[1] = bf16_hi(u.x);
  x[2] = bf16_lo(u.y);
  x[3] = bf16_hi(u.y);
}

// Two fp32 values in one register pair: one instruction for two products.
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
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

template <int D, bool kVec>
__global__ void __launch_bounds__(kRotThreads, 4)
    rotary_kernel(const __grid_constant__ RotaryArgs a, int tokens) {
  constexpr int kLanes = D / 8;              // lanes of one row
  constexpr int kRows = 32 / kLanes;         // rows of one warp
  constexpr int kStep = kRotThreads / 32 * kRows;
  constexpr int kAhead = 4;                  // rows in flight per lane
  extern __shared__ float4 table[];          // [tokens][half / 4] x (4 cos, 4 sin)
  __shared__ long long pool_row[kRotTokens]; // where a token's rows start in the pool, or -1
  __shared__ int pool_flip[kRotTokens];      // and how its 16-byte chunks are permuted
  pdl_wait();
  pdl_trigger();
  const int t0 = blockIdx.x * tokens;
  const int nt = min(tokens, a.ntok - t0);
  for (int i = threadIdx.x; i < nt * a.half; i += kRotThreads) {
    const int t = i / a.half, p = i - t * a.half;
    const int ax = min(max(a.axis[p], 0), a.axes - 1);
    const double turn = (double)a.positions[ax * a.pos_axis + t0 + t] * a.turns[p];
    float s, c;
    sincospif(2.f * (float)(turn - rint(turn)), &s, &c);
    float* at = reinterpret_cast<float*>(table) + 2 * (i - (p & 3)) + (p & 3);
    at[0] = c;
    at[4] = s;
  }
  if (a.pool != nullptr && threadIdx.x < nt) {
    const int64_t slot = a.slots[t0 + threadIdx.x];
    const int64_t page = slot >> a.page_shift;
    const int off = (int)slot & (a.P - 1);
    const bool in = slot >= 0 && page < a.num_pages;
    if (slot >= 0 && !in) flag_device(a.status, DEV_BAD_INDEX);
    pool_row[threadIdx.x] = in ? (page * a.Hkv * 2 * a.P + off) * D : -1;
    pool_flip[threadIdx.x] = 8 * (off & 7);
  }

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = lane % kLanes;
  // This lane's pieces: of the rotary part the c-th of each half, of the rest two
  // neighbours. lo / hi are their first elements.
  const int turning = a.half / 4;            // lanes of the rotary part
  const bool turns = c < turning;
  const int lo = turns ? 4 * c : 8 * c;      // 2 half + 8 (c - half / 4)
  const int hi = turns ? lo + a.half : lo + 4;
  // Heads of one operand, a head (kRows of them) to a warp, its tokens one after the
  // other; kKind: 0 q, 1 k, 2 v. All lanes of a warp go around alike: the shuffles want
  // the whole warp. Operands start on different warps (skew).
  const auto walk = [&](auto kind, int nheads, int skew, const uint16_t* in, long long in_tok,
                        long long in_head, const uint16_t* weight) {
    constexpr int kKind = decltype(kind)::value;
    const int step = kStep * gridDim.y;
    int h = ((blockIdx.y * (kRotThreads / 32) + warp) * kRows + lane / kLanes + step - skew) % step;
    if (!__any_sync(0xffffffffu, h < nheads)) return;
    uint64_t w[4];
    if (weight != nullptr) {
      float f[8];
      unpack4(*reinterpret_cast<const uint2*>(weight + lo), f);
      unpack4(*reinterpret_cast<const uint2*>(weight + hi), f + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = pair(f[2 * e], f[2 * e + 1]);
    }
    for (; __any_sync(0xffffffffu, h < nheads); h += step) {
      const bool live = h < nheads;
      const uint16_t* src = in + t0 * in_tok + (live ? h : 0) * in_head;
      uint16_t* out = kKind == 0 ? a.q_out + ((size_t)t0 * nheads + h) * D
                                 : (kKind == 1 && a.pool == nullptr
                                        ? a.k_out + ((size_t)t0 * nheads + h) * D
                                        : a.pool + (size_t)(2 * h + (kKind == 2)) * a.P * D);
      for (int tb = 0; tb < nt; tb += kAhead) {
        uint2 u[kAhead][2];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          u[i][0] = u[i][1] = make_uint2(0u, 0u);
          if (live && tb + i < nt) {
            u[i][0] = load4<kVec>(src + lo);
            u[i][1] = load4<kVec>(src + hi);
          }
          src += in_tok;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int t = tb + i;
          if (t >= nt) break;  // uniform
          if constexpr (kKind != 2) {
            float f[8];
            unpack4(u[i][0], f);
            unpack4(u[i][1], f + 4);
            uint64_t x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = pair(f[2 * e], f[2 * e + 1]);
            if (weight != nullptr) {
              uint64_t sq = mul2(x[0], x[0]);
#pragma unroll
              for (int e = 1; e < 4; ++e) sq = fma2(x[e], x[e], sq);
              float s0, s1;
              unpair(sq, s0, s1);
              float sum = s0 + s1;
#pragma unroll
              for (int off = kLanes / 2; off >= 1; off >>= 1)
                sum += __shfl_xor_sync(0xffffffffu, sum, off);
              const float inv = rsqrtf(sum * (1.f / D) + a.eps);
              const uint64_t both = pair(inv, inv);
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = mul2(mul2(x[e], both), w[e]);
            }
            if (turns) {
              const float4 co = table[2 * (t * turning + c)], si = table[2 * (t * turning + c) + 1];
              const uint64_t c0 = pair(co.x, co.y), c1 = pair(co.z, co.w);
              const uint64_t s0 = pair(si.x, si.y), s1 = pair(si.z, si.w);
              const uint64_t n0 = pair(-si.x, -si.y), n1 = pair(-si.z, -si.w);
              const uint64_t y0 = x[0], y1 = x[1], z0 = x[2], z1 = x[3];
              x[0] = fma2(y0, c0, mul2(z0, n0));
              x[1] = fma2(y1, c1, mul2(z1, n1));
              x[2] = fma2(z0, c0, mul2(y0, s0));
              x[3] = fma2(z1, c1, mul2(y1, s1));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) unpair(x[e], f[2 * e], f[2 * e + 1]);
            u[i][0] = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
            u[i][1] = make_uint2(pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
          }
          if constexpr (kKind == 0) {
            if (live) {
              *reinterpret_cast<uint2*>(out + lo) = u[i][0];
              *reinterpret_cast<uint2*>(out + hi) = u[i][1];
            }
            out += (size_t)nheads * D;
          } else if (a.pool != nullptr) {
            const long long row = pool_row[t];
            if (live && row >= 0) {  // 16-byte chunks move, halves of one stay
              const int flip = pool_flip[t];
              *reinterpret_cast<uint2*>(out + row + (lo ^ flip)) = u[i][0];
              *reinterpret_cast<uint2*>(out + row + (hi ^ flip)) = u[i][1];
            }
          } else {
            if (live) {
              *reinterpret_cast<uint2*>(out + lo) = u[i][0];
              *reinterpret_cast<uint2*>(out + hi) = u[i][1];
            }
            out += (size_t)nheads * D;
          }
        }
      }
    }
  };
  __syncthreads();
  const int step = kStep * gridDim.y;
  walk(std::integral_constant<int, 0>{}, a.Hq, 0, a.q, a.q_tok, a.q_head, a.q_weight);
  walk(std::integral_constant<int, 1>{}, a.Hkv, a.Hq % step, a.k, a.k_tok, a.k_head, a.k_weight);
  if (a.pool != nullptr)
    walk(std::integral_constant<int, 2>{}, a.Hkv, (a.Hq + a.Hkv) % step, a.v, a.v_tok, a.v_head,
         static_cast<const uint16_t*>(nullptr));
}

template <int D>
cudaError_t launch_rotary(const RotaryArgs& a, bool vec, cudaStream_t s) {
  // Tokens of a CTA: as few as fill the GPU (four CTAs an SM), in whole waves of CTAs; few
  // tokens spread their heads over CTAs, so that a warp has about one row.
  constexpr long long kFit = 148 * 4;
  const int rows_per_cta = kRotThreads / 32 * (32 / (D / 8));
  const int heads = a.Hq + 2 * a.Hkv;
  const long long waves = (a.ntok + kFit * kRotTokens - 1) / (kFit * kRotTokens);
  const int tokens = (int)((a.ntok + kFit * waves - 1) / (kFit * waves));
  const int ctas = (a.ntok + tokens - 1) / tokens;
  const int spread = (heads + rows_per_cta - 1) / rows_per_cta;
  const dim3 grid(ctas, (int)std::max(1ll, std::min<long long>(spread, kFit / ctas)));
  const size_t smem = (size_t)tokens * a.half * sizeof(float2);
  return launch_pdl(vec ? rotary_kernel<D, true> : rotary_kernel<D, false>, grid,
                    dim3(kRotThreads), smem, s, a, tokens);
}

}  // namespace
}  // namespace sc

extern "C" int sc_rotary_append(const sc_bf16* q, const sc_bf16* k, const sc_bf16* v,
                                const int64_t* strides, const int32_t* positions,
                                int64_t pos_axis_stride, int axes, const double* turns,
                                const int32_t* axis, const sc_bf16* q_weight,
                                const sc_bf16* k_weight, float eps, sc_bf16* q_out,
                                sc_bf16* k_out, sc_bf16* kv_pool, const int64_t* slot_mapping,
                                int ntok, int Hq, int Hkv, int D, int rotary_dim, int P,
                                int64_t num_pages, void* stream) {
  const char* name = "sc_rotary_append";
  SC_REQUIRE(ntok >= 0 && Hq > 0 && Hkv > 0 && axes > 0, SC_ERR_INVALID,
             "%s: bad ntok=%d Hq=%d Hkv=%d axes=%d", name, ntok, Hq, Hkv, axes);
  SC_REQUIRE(D == 64 || D == 128 || D == 256, SC_ERR_UNSUPPORTED, "%s: D=%d not in {64,128,256}",
             name, D);
  SC_REQUIRE(rotary_dim > 0 && rotary_dim % 16 == 0 && rotary_dim <= D, SC_ERR_UNSUPPORTED,
             "%s: rotary_dim=%d must be a multiple of 16 in [16, D]", name, rotary_dim);
  if (ntok == 0) return SC_OK;
  SC_REQUIRE(q && k && strides && positions && turns && axis && q_out, SC_ERR_INVALID,
             "%s: null pointer", name);
  SC_REQUIRE((kv_pool != nullptr) != (k_out != nullptr), SC_ERR_INVALID,
             "%s: exactly one of kv_pool and k_out", name);
  if (kv_pool != nullptr) {
    SC_REQUIRE(v && slot_mapping && num_pages > 0, SC_ERR_INVALID,
               "%s: a pool needs v, slot_mapping and num_pages", name);
    SC_REQUIRE(P == 8 || P == 16 || P == 32, SC_ERR_UNSUPPORTED, "%s: P=%d not in {8,16,32}",
               name, P);
  }
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  SC_REQUIRE(aligned(q_out) && aligned(k_out) && aligned(kv_pool) && aligned(q_weight) &&
                 aligned(k_weight),
             SC_ERR_INVALID, "%s: outputs, pool and weights must be 16-byte aligned", name);
  bool vec = aligned(q) && aligned(k) && aligned(v);
  for (int i = 0; i < 6; ++i) vec = vec && strides[i] % 8 == 0;
  sc::RotaryArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_tok = strides[0];
  a.q_head = strides[1];
  a.k_tok = strides[2];
  a.k_head = strides[3];
  a.v_tok = strides[4];
  a.v_head = strides[5];
  a.positions = positions;
  a.pos_axis = pos_axis_stride;
  a.turns = turns;
  a.axis = axis;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.q_out = q_out;
  a.k_out = k_out;
  a.pool = kv_pool;
  a.slots = slot_mapping;
  a.num_pages = num_pages;
  a.eps = eps;
  a.ntok = ntok;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.half = rotary_dim / 2;
  a.axes = axes;
  a.P = kv_pool != nullptr ? P : 16;
  a.page_shift = a.P == 8 ? 3 : a.P == 16 ? 4 : 5;
  a.status = sc::device_status_word();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = D == 64    ? sc::launch_rotary<64>(a, vec, s)
                          : D == 128 ? sc::launch_rotary<128>(a, vec, s)
                                     : sc::launch_rotary<256>(a, vec, s);
  if (err != cudaSuccess)
    return sc::set_error(SC_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
  return sc::check_launch(name);
}
