// What happens to a new token's q, k and v between the projection and the cache, in one pass:
// per-head RMS norm of q and k, rotary positions, and the store of k and v into the page slot
// that the slot mapping names (16-bit, int8 or e4m3 pools, on this GPU or on peers).
//
//   y = x / sqrt(mean(x^2) + eps) * w                                    (q and k, if weights are given)
//   (a, b) -> gain * (a cos t - b sin t, b cos t + a sin t), t = position * inv_freq[i]
//       half layout: a = y[i], b = y[i + rot/2];  interleaved: a = y[2i], b = y[2i+1];  i < rot/2
//
// Bytes bound it: each row is read once and written once.  Sixteen lanes hold a row of 128 values,
// 16 bytes each; norm sums, absmax and rotation partners travel by shuffle.  Norm and rotation are
// fp32 with one rounding at the end.  The angle is reduced in fp64 (a position near 2^20 times an
// fp32 frequency keeps only four bits behind the point in fp32), once per token and block.
// A quantised pool gets what quantize_kv_kernel makes of the 16-bit row, bit for bit: so the
// values are rounded to 16 bits first, and a cache filled token by token equals one that
// was quantised whole.
#pragma once
#include "layer_kernels.cuh"
#include "merge_kernel.cuh"

namespace pkv {

constexpr int kNraThreads = 256;                       // 16 rows at a time
constexpr int kNraRows = kNraThreads / 16;

struct NormRopeParams {
  const void* qkv;             // [n_tokens] rows of (Hq + 2 Hkv) heads of 128
  int64_t qkv_stride;
  const int64_t* positions;
  const float* inv_freq;       // [rot / 2]
  const void* q_weight;        // [128] or null
  const void* k_weight;
  void* q_out;
  int64_t q_stride;
  const int64_t* slot_mapping; // null: no append
  int n_tokens, n_q_heads, n_kv_heads;
  int rot, interleaved;
  float eps, gain;
  int n_dev, page_size, fmt;   // fmt: PKV_F16 / PKV_BF16 / PKV_INT8 / PKV_FP8_E4M3
  int64_t bases[kMaxWorld], n_pages[kMaxWorld];
  uint8_t* k_pool[kMaxWorld];
  uint8_t* v_pool[kMaxWorld];
  __half* k_scale[kMaxWorld];
  __half* v_scale[kMaxWorld];
  int64_t page_stride[kMaxWorld], token_stride[kMaxWorld], head_stride[kMaxWorld];   // elements
  uint32_t* status;
};

// grid (tokens, blocks of 16 rows); rows of a token: q heads, k heads, v heads
template <bool BF16>
__global__ void __launch_bounds__(kNraThreads) norm_rope_append_kernel(const NormRopeParams p) {
  using E = Elem16<BF16>;
  __shared__ __align__(16) float s_cos[64], s_sin[64];
  const int tok = blockIdx.x, l = threadIdx.x & 15;
  const int rows = p.n_q_heads + (p.slot_mapping ? 2 * p.n_kv_heads : 0);
  const int row = blockIdx.y * kNraRows + (threadIdx.x >> 4);
  const bool live = row < rows;
  const bool is_q = row < p.n_q_heads, is_v = row >= p.n_q_heads + p.n_kv_heads;
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (live)
    raw = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.qkv) + (int64_t)tok * p.qkv_stride +
                                         (int64_t)row * kHeadDim)[l];
  const int half = p.rot >> 1;
  if (threadIdx.x < half) {
    // turns = position * f / 2 pi, reduced to [-1/2, 1/2] before it is rounded to fp32
    const double turns = (double)p.positions[tok] * (double)p.inv_freq[threadIdx.x] * 0.15915494309189533577;
    float sn, cs;
    sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
    s_cos[threadIdx.x] = cs * p.gain;
    s_sin[threadIdx.x] = sn * p.gain;
  }
  __syncthreads();
  // every lane of a warp stays in for the shuffles; lanes without a row work on zeros
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 f = E::up(w[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
  const void* weight = is_q ? p.q_weight : is_v ? nullptr : p.k_weight;
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (live && weight) {
    const float r = rsqrtf(ss * (1.f / kHeadDim) + p.eps);
    const uint4 wv = reinterpret_cast<const uint4*>(weight)[l];
    const uint32_t* pw = reinterpret_cast<const uint32_t*>(&wv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = E::up(pw[i]);
      x[2 * i] *= r * f.x;
      x[2 * i + 1] *= r * f.y;
    }
  }
  const int e0 = l * 8;
  if (p.interleaved) {
    if (!is_v && e0 < p.rot) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float cs = s_cos[e0 / 2 + i], sn = s_sin[e0 / 2 + i];
        const float a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = a * cs - b * sn;
        x[2 * i + 1] = b * cs + a * sn;
      }
    }
  } else {
    // rot is a multiple of 16, so a lane's eight values have their partners in one other lane
    const bool low = e0 < half;
    const int step = half >> 3;
    const int from = (threadIdx.x & 16) | ((low ? l + step : l - step) & 15);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], from);
    if (!is_v && e0 < p.rot) {
      const int f0 = low ? e0 : e0 - half;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float cs = s_cos[f0 + i], sn = s_sin[f0 + i];
        x[i] = low ? x[i] * cs - y[i] * sn : x[i] * cs + y[i] * sn;
      }
    }
  }
  uint4 packed;
  packed.x = E::down(x[0], x[1]); packed.y = E::down(x[2], x[3]);
  packed.z = E::down(x[4], x[5]); packed.w = E::down(x[6], x[7]);
  if (is_v) packed = raw;
  if (live && is_q)
    reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.q_out) + (int64_t)tok * p.q_stride +
                             (int64_t)row * kHeadDim)[l] = packed;
  if (!p.slot_mapping) return;

  // ---- the owner of the slot ----
  const int64_t slot = p.slot_mapping[tok];
  const int64_t gid = slot < 0 ? -1 : slot / p.page_size;
  int d = 0;
  for (int k = 1; k < p.n_dev; ++k) if (gid >= p.bases[k]) d = k;
  const int64_t page = gid - p.bases[d];
  const bool inside = slot >= 0 && page >= 0 && page < p.n_pages[d];
  if (slot >= 0 && !inside && p.status && blockIdx.y == 0 && threadIdx.x == 0) atomicOr(p.status, kStBadPage);
  const bool store = live && !is_q && inside;
  const int h = row - p.n_q_heads - (is_v ? p.n_kv_heads : 0);
  const int64_t off = slot - gid * p.page_size;
  const int64_t at = page * p.page_stride[d] + off * p.token_stride[d] + (int64_t)h * p.head_stride[d] + e0;
  if (p.fmt == 0 || p.fmt == 1) {
    if (store) *reinterpret_cast<uint4*>((is_v ? p.v_pool[d] : p.k_pool[d]) + at * 2) = packed;
    return;
  }
  const uint32_t* pk = reinterpret_cast<const uint32_t*>(&packed);
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = E::up(pk[i]);
    x[2 * i] = f.x; x[2 * i + 1] = f.y;
    a = fmaxf(a, fmaxf(fabsf(f.x), fabsf(f.y)));
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  const __half sc = kv_row_scale(a, p.fmt);
  const float sf = __half2float(sc);
  uint2 codes = make_uint2(0u, 0u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    codes.x |= kv_code(x[i], sf, p.fmt) << (8 * i);
    codes.y |= kv_code(x[4 + i], sf, p.fmt) << (8 * i);
  }
  if (store) {
    *reinterpret_cast<uint2*>((is_v ? p.v_pool[d] : p.k_pool[d]) + at) = codes;
    if (l == 0) (is_v ? p.v_scale[d] : p.k_scale[d])[(page * p.page_size + off) * p.n_kv_heads + h] = sc;
  }
}

}  // namespace pkv
