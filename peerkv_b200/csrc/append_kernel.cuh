// What happens to a new token's q, k and v between the projection and the cache, in one pass:
// per-head RMS norm of q and k, rotary positions, and the store of k and v into the page slot
// that the slot mapping names (16-bit, int8 or e4m3 pools, on this GPU or on peers).
//
//   y = x / sqrt(mean(x^2) + eps) * w                                    (q and k, if weights are given)
//   (a, b) -> gain * (a cos t - b sin t, b cos t + a sin t), t = position * inv_freq[i]
//       half layout: a = y[i], b = y[i + rot/2];  interleaved: a = y[2i], b = y[2i+1];  i < rot/2
//
// Bytes bound it: each row is read once and written once; the instructions are what keeps a kernel from
// that.  A warp takes a token (or, where there are few tokens, some of its rows) and works alone:
// sixteen lanes hold a row of 128 values, 16 bytes each, two rows at a time, eight in flight; norm
// sums, absmax and rotation partners travel by shuffle.  A row is y = r (x C + partner S), with
// the weights folded into the cosines C and the signed sines S once per token and lane, in packed
// fp32 pairs, and the partners exchanged as the 16-bit words they came as.  (A block per token with
// a barrier behind the angles took 240 instructions per two rows and 76 us for 8192 tokens of
// 32 + 16 heads.)
// Norm and rotation are fp32 with one rounding at the end.  The angle is reduced in fp64 (a position
// near 2^20 times an fp32 frequency keeps only four bits behind the point in fp32).
// A quantised pool gets what quantize_kv_kernel makes of the 16-bit row, bit for bit: so the
// values are rounded to 16 bits first, and a cache filled token by token equals one that
// was quantised whole.
#pragma once
#include "layer_kernels.cuh"
#include "merge_kernel.cuh"
#include "tcgen05.cuh"

namespace pkv {

constexpr int kNraWarps = 4;                           // of a block; each on its own

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

constexpr int kNraBatch = 4;                           // pairs of rows a warp has in flight

// One warp per (token, split of its rows).  The rows of a token are taken in pairs, q heads, then k
// heads, then v heads (an odd last head has a pair to itself); split s takes the pairs s, s +
// splits, ...  Each kind has a loop of its own: v rows are copied.
template <bool BF16, bool INTERLEAVED, bool QUANT>
__global__ void __launch_bounds__(kNraWarps * 32) norm_rope_append_kernel(const NormRopeParams p, int splits) {
  using E = Elem16<BF16>;
  __shared__ __align__(16) float s_cs[kNraWarps][2][64];
  const int lane = threadIdx.x & 31, l = lane & 15, e0 = l * 8, hi = lane >> 4;
  const int64_t unit = (int64_t)blockIdx.x * kNraWarps + (threadIdx.x >> 5);
  const int tok = (int)(unit / splits), split = (int)(unit - (int64_t)tok * splits);
  if (tok >= p.n_tokens) return;
  float* s_cos = s_cs[threadIdx.x >> 5][0];
  float* s_sin = s_cs[threadIdx.x >> 5][1];
  const int q_pairs = (p.n_q_heads + 1) >> 1, kv_pairs = p.slot_mapping ? (p.n_kv_heads + 1) >> 1 : 0;
  const uint16_t* src = reinterpret_cast<const uint16_t*>(p.qkv) + (int64_t)tok * p.qkv_stride + e0;
  // this lane's 16 bytes of the batch of pairs that starts at pair i of the `heads` heads from src0 on
  auto fetch = [&](uint4 (&raw)[kNraBatch], const uint16_t* src0, int i, int heads) {
#pragma unroll
    for (int k = 0; k < kNraBatch; ++k) {
      const int row = 2 * (i + k * splits) + hi;
      raw[k] = row < heads ? *reinterpret_cast<const uint4*>(src0 + row * kHeadDim) : make_uint4(0, 0, 0, 0);
    }
  };
  // first pair of a kind that is this split's, the kind's pairs counting from `before`
  auto first_pair = [&](int before) { const int r = (split - before) % splits; return r < 0 ? r + splits : r; };
  uint4 raw[kNraBatch];
  fetch(raw, src, split, p.n_q_heads);                   // on their way while the angles are made

  const int half = p.rot >> 1;
#pragma unroll
  for (int f = lane; f < 64; f += 32) {
    if (f < half) {
      // turns = position * f / 2 pi, reduced to [-1/2, 1/2] before it is rounded to fp32
      const double turns = (double)p.positions[tok] * (double)p.inv_freq[f] * 0.15915494309189533577;
      float sn, cs;
      sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
      s_cos[f] = cs * p.gain;
      s_sin[f] = sn * p.gain;
    }
  }
  int64_t at = -1, scale_at = 0;                         // where the token's rows lie in pool d; -1: nowhere
  int d = 0;
  if (p.slot_mapping) {
    const int64_t slot = p.slot_mapping[tok];
    if (slot >= 0) {
      const int64_t gid = slot <= 0x7fffffff ? (int64_t)((uint32_t)slot / (uint32_t)p.page_size) : slot / p.page_size;
      const int64_t off = slot - gid * p.page_size;
      for (int k = 1; k < p.n_dev; ++k) if (gid >= p.bases[k]) d = k;
      const int64_t page = gid - p.bases[d];
      if (page >= 0 && page < p.n_pages[d]) {
        at = page * p.page_stride[d] + off * p.token_stride[d];
        scale_at = (page * p.page_size + off) * p.n_kv_heads;
      } else if (p.status && split == 0 && lane == 0) {
        atomicOr(p.status, kStBadPage);
      }
    }
  }
  __syncwarp();

  // rot is a multiple of 16, so a lane's eight values have their partners in one other lane
  const bool low = e0 < half, in = e0 < p.rot;
  const int partner = INTERLEAVED ? l : (low ? l + (half >> 3) : l - (half >> 3)) & 15;
  const int from = (lane & 16) | partner;
  uint64_t c2[4], s2[4];                                 // C and S of this lane's eight values, as pairs
  auto tables = [&](const void* weight) {
    float w[8], pw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = pw[i] = 1.f;
    if (weight) {
      const uint4 a = reinterpret_cast<const uint4*>(weight)[l], b = reinterpret_cast<const uint4*>(weight)[partner];
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = E::up(aw[i]), g = E::up(bw[i]);
        w[2 * i] = f.x; w[2 * i + 1] = f.y;
        pw[2 * i] = INTERLEAVED ? f.y : g.x; pw[2 * i + 1] = INTERLEAVED ? f.x : g.y;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float c[2], sn[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int e = e0 + 2 * i + k, f = INTERLEAVED ? e >> 1 : low ? e : e - half;
        const bool first = INTERLEAVED ? k == 0 : low;           // the a of (a, b): its sine counts negative
        c[k] = in ? w[2 * i + k] * s_cos[f] : w[2 * i + k];
        sn[k] = in ? pw[2 * i + k] * (first ? -s_sin[f] : s_sin[f]) : 0.f;
      }
      c2[i] = pack_f32x2(c[0], c[1]);
      s2[i] = pack_f32x2(sn[0], sn[1]);
    }
  };
  // norm and rotation of a row; every lane stays in for the shuffles
  auto turn = [&](const uint4& v, bool norm) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint64_t x2[4], r2 = pack_f32x2(1.f, 1.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = E::up(w[i]);
      x2[i] = pack_f32x2(f.x, f.y);
    }
    if (norm) {
      uint64_t sa = mul_f32x2(x2[0], x2[0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) sa = fma_f32x2(x2[i], x2[i], sa);
      const float2 sp = unpack_f32x2(sa);
      float ss = sp.x + sp.y;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss * (1.f / kHeadDim) + p.eps);
      r2 = pack_f32x2(r, r);
    }
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t pv = INTERLEAVED ? __byte_perm(w[i], 0, 0x1032) : __shfl_sync(0xffffffffu, w[i], from);
      if (!in) pv = 0u;
      const float2 f = E::up(pv);
      const float2 y = unpack_f32x2(mul_f32x2(fma_f32x2(pack_f32x2(f.x, f.y), s2[i], mul_f32x2(x2[i], c2[i])), r2));
      o[i] = E::down(y.x, y.y);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
  };

  uint16_t* q_row = reinterpret_cast<uint16_t*>(p.q_out) + (int64_t)tok * p.q_stride + e0;
  if (split < q_pairs) tables(p.q_weight);
  for (int i = split; i < q_pairs; i += kNraBatch * splits) {
    if (i != split) fetch(raw, src, i, p.n_q_heads);
#pragma unroll
    for (int k = 0; k < kNraBatch; ++k) {
      if (i + k * splits >= q_pairs) break;
      const int row = 2 * (i + k * splits) + hi;
      const uint4 v = turn(raw[k], p.q_weight != nullptr);
      if (row < p.n_q_heads) *reinterpret_cast<uint4*>(q_row + row * kHeadDim) = v;
    }
  }
  if (at < 0) return;

  const int64_t hs = p.head_stride[d];
  auto store = [&](uint8_t* pool, __half* scales, int h, const uint4& v) {       // all lanes
    const bool live = h < p.n_kv_heads;
    const int64_t to = at + (int64_t)h * hs + e0;
    if constexpr (!QUANT) {
      if (live) *reinterpret_cast<uint4*>(pool + to * 2) = v;
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      float x[8], a = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = E::up(w[i]);
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
      if (live) {
        *reinterpret_cast<uint2*>(pool + to) = codes;
        if (l == 0) scales[scale_at + h] = sc;
      }
    }
  };
  const int k0 = first_pair(q_pairs), v0 = first_pair(q_pairs + kv_pairs);
  if (k0 < kv_pairs) {
    const uint16_t* ks = src + (int64_t)p.n_q_heads * kHeadDim;
    fetch(raw, ks, k0, p.n_kv_heads);
    tables(p.k_weight);
    for (int i = k0; i < kv_pairs; i += kNraBatch * splits) {
      if (i != k0) fetch(raw, ks, i, p.n_kv_heads);
#pragma unroll
      for (int k = 0; k < kNraBatch; ++k) {
        if (i + k * splits >= kv_pairs) break;
        store(p.k_pool[d], p.k_scale[d], 2 * (i + k * splits) + hi, turn(raw[k], p.k_weight != nullptr));
      }
    }
  }
  const uint16_t* vs = src + (int64_t)(p.n_q_heads + p.n_kv_heads) * kHeadDim;
  for (int i = v0; i < kv_pairs; i += kNraBatch * splits) {
    fetch(raw, vs, i, p.n_kv_heads);
#pragma unroll
    for (int k = 0; k < kNraBatch; ++k) {
      if (i + k * splits >= kv_pairs) break;
      store(p.v_pool[d], p.v_scale[d], 2 * (i + k * splits) + hi, raw[k]);
    }
  }
}

}  // namespace pkv
