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
// B200 mapping. HBM-bound: each value is read and written once. A CTA makes the
// (cos, sin) table of its tokens in shared memory, then its warps walk the tokens'
// head rows (q, k, v); D / 8 lanes hold a row, 8 values each, so a row moves as
// 16-byte accesses, the norm is a shuffle sum and the partner of a pair is a
// shuffle away (R / 2 is a multiple of 8).
#include "common.cuh"

namespace sc {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 4;      // tokens of one CTA on long inputs

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
  int ntok, Hq, Hkv, half, axes, P;
  unsigned int* status;
};

// 8 consecutive bf16 of a row; without kVec the address has 2-byte alignment only.
template <bool kVec>
__device__ __forceinline__ uint4 load8(const uint16_t* p) {
  if constexpr (kVec) {
    return *reinterpret_cast<const uint4*>(p);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ void unpack8(const uint4& u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(w[i]);
    x[2 * i + 1] = bf16_hi(w[i]);
  }
}

template <int D, bool kVec>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs a, int tokens) {
  constexpr int kLanes = D / 8;              // lanes of one row
  constexpr int kRows = 32 / kLanes;         // rows of one warp
  extern __shared__ float2 table[];          // [tokens][half] (cos, sin)
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
    table[i] = make_float2(c, s);
  }
  __syncthreads();

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = lane % kLanes;               // this lane's 16-byte chunk of its row
  const int heads = a.Hq + 2 * a.Hkv;
  const int nrows = nt * heads;
  const int step = kRotThreads / 32 * kRows * gridDim.y;
  const int hc = a.half / 8;                 // chunks of half the rotary dims
  // The partner of a rotary chunk holds the other halves of its pairs.
  const int partner = (c < hc ? c + hc : (c < 2 * hc ? c - hc : c)) + (lane - c);
  for (int r0 = (blockIdx.y * (kRotThreads / 32) + warp) * kRows; r0 < nrows; r0 += step) {
    const int r = r0 + lane / kLanes;
    const bool live = r < nrows;
    const int t = live ? r / heads : 0;
    const int h = live ? r - t * heads : 0;
    const long long tok = t0 + t;
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
    const int kvh = is_q ? 0 : (is_v ? h - a.Hq - a.Hkv : h - a.Hq);
    uint16_t* dst = nullptr;
    const uint16_t* src;
    if (is_q) {
      src = a.q + tok * a.q_tok + h * a.q_head;
      dst = a.q_out + ((size_t)tok * a.Hq + h) * D + 8 * c;
    } else {
      src = is_v ? a.v + tok * a.v_tok + kvh * a.v_head : a.k + tok * a.k_tok + kvh * a.k_head;
      if (a.pool != nullptr) {
        const int64_t slot = a.slots[tok];
        const int64_t page = slot / a.P;
        if (slot >= 0 && page < a.num_pages) {
          const int off = (int)(slot - page * a.P);
          dst = a.pool + ((((size_t)page * a.Hkv + kvh) * 2 + is_v) * a.P + off) * D +
                8 * (c ^ (off & 7));
        } else if (slot >= 0 && c == 0 && live) {
          flag_device(a.status, DEV_BAD_INDEX);
        }
      } else if (!is_v) {
        dst = a.k_out + ((size_t)tok * a.Hkv + kvh) * D + 8 * c;
      }
    }
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (live && dst != nullptr) u = load8<kVec>(src + 8 * c);
    float x[8];
    unpack8(u, x);
    const uint16_t* w = is_q ? a.q_weight : a.k_weight;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
    for (int off = kLanes / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (w != nullptr && !is_v) {
      const float inv = rsqrtf(sum * (1.f / D) + a.eps);
      float wf[8];
      unpack8(*reinterpret_cast<const uint4*>(w + 8 * c), wf);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * wf[i];
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], partner);
    if (!is_v && c < 2 * hc) {
      const float2* cs = table + t * a.half + 8 * (c < hc ? c : c - hc);
      const float sign = c < hc ? -1.f : 1.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * cs[i].x + sign * (y[i] * cs[i].y);
    }
    if (live && dst != nullptr) {
      if (!is_v)
        u = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                       pack_bf16x2(x[6], x[7]));
      *reinterpret_cast<uint4*>(dst) = u;
    }
  }
}

template <int D>
cudaError_t launch_rotary(const RotaryArgs& a, bool vec, cudaStream_t s) {
  // Few tokens: one token a CTA and its heads spread over CTAs, so that every warp has
  // about one row; many: kRotTokens tokens a CTA.
  const int rows_per_cta = kRotThreads / 32 * (32 / (D / 8));
  const int heads = a.Hq + 2 * a.Hkv;
  const bool few = a.ntok <= 1024;
  const int tokens = few ? 1 : kRotTokens;
  const dim3 grid((a.ntok + tokens - 1) / tokens, few ? (heads + rows_per_cta - 1) / rows_per_cta : 1);
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
  a.status = sc::device_status_word();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t err = D == 64    ? sc::launch_rotary<64>(a, vec, s)
                          : D == 128 ? sc::launch_rotary<128>(a, vec, s)
                                     : sc::launch_rotary<256>(a, vec, s);
  if (err != cudaSuccess)
    return sc::set_error(SC_ERR_CUDA, "%s: launch: %s", name, cudaGetErrorString(err));
  return sc::check_launch(name);
}
