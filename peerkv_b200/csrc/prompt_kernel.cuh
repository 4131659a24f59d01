// Prompt attention: many query rows per sequence, packed sequences of different lengths, K/V
// in the paged pool (or packed like the queries), on the fifth-generation tensor cores.  The
// same kernel attends a group of decoding sequences to the prefix they share: the group is
// one "sequence" whose query rows all see every key.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - m_i),  lse_i = m_i + log sum_j p_ij
//   causal: query row i of n sees keys j <= L - n + i (the n rows are the last of L tokens).
//
// Tile.  128 rows = 128 / G tokens x the G query heads of one kv-head, so one K/V tile serves
// the whole group and the causal diagonal of a tile is 128 / G tokens wide instead of 128.  A CTA
// works on two row tiles at once (an "item" = 2 row tiles of one sequence and kv-head): while
// one softmax warpgroup exponentiates, the tensor cores run the other's products.  An item
// with a single row tile (few rows: a shared prefix, a chunk's end) gives the two warpgroups
// alternate KV tiles instead and joins their accumulators at the end.
//
// Warps (384 threads, one CTA per SM): 0-3 and 4-7 the two softmax warpgroups, one thread per
// row; 8 walks the work list and loads Q and K, 11 loads V (TMA); 9 and 10 issue the tcgen05
// instructions of the two row tiles.
// TMEM: S0 S1 O0 O1, 128 columns each; the 16-bit P overwrites the first half of its S.
// Shared memory: Q 2 x 32 KB; K and V tiles of 128 keys in rings of two and three 32 KB slots.
//
// Sums.  Scores, maxima, sums and O are fp32.  P is rounded to the 16-bit type of V, as the
// matrix instruction wants both operands alike; the row sum adds the unrounded values.  The
// rounding costs an output as much as its own last rounding does (2^-9 relative per weight in bf16, 2^-12
// in fp16 on average, independent signs), half of the error budget of a 16-bit output.  (The kernel for dense
// tensors, prefill_kernel.cuh, sends a bf16 P as two terms: its result is an fp32 partial.  Here that
// would be half as many products again on the pipe that bounds a step, for an output that is
// rounded to 16 bits itself.)  The reference of the exponentials moves only when a row's maximum has grown
// by more than 2^8: until then O need not be touched; l and lse use the same reference, so nothing
// is lost.  fp16 ends at 2^-24, and behind one dominant key the many small weights can be the output: there
// the reference is lifted by 2^7, so that the row's largest weight stands between 2^7 and 2^15 and a small one
// keeps its 11 bits down to 2^-21 of it and is off by at most 2^-32 of it below.  bf16 has fp32's range.
//
// Work split.  The KV tiles of all items form one list that is cut into equal pieces, one per
// CTA, wherever the cut falls: ragged batches, causal triangles and a handful of rows over a
// long cache are all balanced the same way.  An item that is cut leaves unnormalised (O, m, l)
// pieces in a workspace which prompt_join_kernel adds up in a fixed order.
//
// What bounds it (B200, bf16, 32 q and 8 kv heads).  A step, 256 rows x 128 keys, takes the tensor
// cores 2048 cycles and the special-function unit as many (32768 exponentials at 16 a cycle); it
// measures 2900: a stream's scores, exponentials and product follow one another, and two streams
// half a step apart hide most but not all of that (the tensor pipe is busy 54 % of the active cycles, the
// special-function unit 57 %).  8192-token prompt: 532 us call behind call (1.03 PFLOP/s, 0.75 of the
// sustained rate of the library's large products; the power cap takes the clock down), 475 us from
// idle (1.16 PFLOP/s, 0.72 of their burst rate).  Short prompts and short prefixes are bound by
// latency: 6 us from launch to the first scores (lengths, block table, first tiles, each a trip to
// memory behind the other), 2 us an item's epilogue, 5 us the join.  A prefix of 32768 tokens for 64
// sequences streams at 3 TB/s: its steps are compute, then the same latencies.
// Tried and dropped: exponentials on the FMA pipe (1/16 to 1/4 of them: 4 to 25 % more cycles),
// one S buffer for both streams with P beside it (same cycles, more code, ragged batches 10 % slower),
// one warp issuing both streams' products (waits and issue between them took as long as they did).
#pragma once
#include "decode_kernel.cuh"
#include "tcgen05.cuh"

namespace pkv {

constexpr int kPaRows = 128;       // rows of a row tile (TMEM lanes)
constexpr int kPaKeys = 128;       // keys of a KV tile
constexpr int kPaThreads = 384;
constexpr int kPaKSlots = 2, kPaVSlots = 3, kPaSlots = kPaKSlots + kPaVSlots;
constexpr int kPaTileBytes = kPaKeys * kHeadDim * 2;     // 32 KB
constexpr int kPaHalfBytes = kPaTileBytes / 2;           // 128 rows x 64 values, 128-byte swizzle
constexpr int kPaRingOff = 2 * kPaTileBytes;
constexpr int kPaMiscOff = kPaRingOff + kPaSlots * kPaTileBytes;
constexpr int kPaMiscBytes = 640 + 128 * 8;
constexpr int kPaSmem = kPaMiscOff + kPaMiscBytes + 1024;  // 1 KB to align the base
static_assert(kPaSmem <= 232448, "shared memory of a CTA");
constexpr int kPaMaxCtas = 256;
// 384 threads x 168 registers at launch = 64512; 256 x 208 + 128 x 80 = 63488 after the split.
constexpr int kPaSoftmaxRegs = 208;
constexpr int kPaOtherRegs = 80;
// What the largest weight of a row is at least, as a power of two (see Sums).
template <bool BF16> constexpr float kPaLift = BF16 ? 0.f : 7.f;
constexpr uint32_t kPaColO = 256;                        // TMEM columns: S0 0, S1 128, O0 256, O1 384
// The cost axis counts thirds of a key of a step with two row tiles.  A step with one row
// tile takes two thirds of that; what an item takes besides its steps (first scores, epilogue) is
// weighted like three steps (with 192 keys instead of 384 a ragged batch of prompts takes 370 us instead of 349, a chunk
// that rides with single tokens 73 instead of 66).
constexpr int kPaItemCost = 1152;  // per item, = 3 x 384 keys
constexpr int kPaMinPiece = 1024;  // no CTA gets less (4 sequences behind 2048 tokens: 24.9 us in a graph; 25.6 with 768, 26.1 with 1536)

// Which CTA found which item cut (one per CTA, for the join).
struct PromptRec {
  int64_t a;             // start of the CTA's first item on the cost axis: the item's name
  int mid;               // the CTA's piece starts inside that item
  int kt0, kt1, n;       // the KV tiles of the item this CTA did, of n
  int q0, n_tok, h;      // first packed row, tokens and kv-head of the item
  int pad;
};

struct PromptParams {
  const int32_t* cu_q;         // [n_seq + 1]
  const int32_t* seq_lens;     // [n_seq] tokens in the cache; null: packed K/V, cu_k
  const int32_t* cu_k;         // [n_seq + 1]
  const int32_t* block_table;  // [n_seq][bt_stride]
  int64_t bt_stride;
  int64_t n_pages;
  int table_cols;              // usable entries of a block-table row
  int page_size, box_tok;      // tokens one TMA box brings (divides page_size and 128)
  int head_major;
  int n_seq, total_q, total_k;
  int n_kv_heads, n_q_heads, group, tok_tile;   // tok_tile = 128 / group tokens per row tile
  int causal;
  float scale_log2;
  void* out;                   // [total_q][n_q_heads][128]
  int out_dtype;               // PKV_F16 / PKV_BF16 / PKV_F32
  float* lse;                  // [total_q][n_q_heads] or null
  const float* o_more;         // one more partial of the same rows to fold in, or null
  const float* lse_more;
  int more_late;               // o_more, lse_more come from the kernel before this one, which may still run
  float4* part_o;              // workspace: [2 * CTAs][32][256]
  float2* part_ml;             // [2 * CTAs][256]
  PromptRec* rec;              // [CTAs + 1]; rec[CTAs].kt0 = CTAs in use
  uint32_t* status;            // or null
};

// ---- the cost axis -------------------------------------------------------------------- //
struct PromptSeq {
  int q0, n, len, k0;          // packed first row, new tokens, cached tokens, first packed key
  int tiles;                   // items per kv-head
  int64_t step, add;           // item t costs add + step * (t + 1), in thirds of a key
};

__device__ __forceinline__ PromptSeq prompt_seq(const PromptParams& p, int s) {
  PromptSeq r;
  const int lo = min(max(p.cu_q[s], 0), p.total_q), hi = min(max(p.cu_q[s + 1], lo), p.total_q);
  r.q0 = lo;
  r.n = hi - lo;
  if (p.seq_lens) {
    r.k0 = 0;
    r.len = (int)min((int64_t)max(p.seq_lens[s], 0), (int64_t)p.table_cols * p.page_size);
  } else {
    r.k0 = min(max(p.cu_k[s], 0), p.total_k);
    r.len = min(max(p.cu_k[s + 1], r.k0), p.total_k) - r.k0;
  }
  const int tt = 2 * p.tok_tile;
  r.tiles = (r.n + tt - 1) / tt;
  const int w = r.n > p.tok_tile ? 3 : 2;
  r.step = p.causal ? w * tt : 0;
  r.add = (int64_t)w * (p.causal ? max(r.len - r.n, 0) : r.len) + kPaItemCost;
  return r;
}
__device__ __forceinline__ int64_t prompt_items_cost(const PromptSeq& s, int64_t t) {   // of items 0 .. t-1
  return t * s.add + s.step * (t * (t + 1) / 2);
}

// Length of a CTA's piece of the cost axis: total / n_cta, a little more where the single-precision
// quotient needs it so that n_cta pieces cover the axis.  No piece is empty: one is at least 512
// long (kPaMinPiece), and what it is too long by, times n_cta, stays below that.  (A 64-bit or
// double-precision division costs the start of every CTA some hundred cycles.)
__device__ __forceinline__ int64_t prompt_piece(int64_t total, int n_cta) {
  return (int64_t)((float)total * __fdividef(1.f, (float)n_cta)) + (total >> 20) + 1;
}

struct PromptItem {
  int s, h, t;                 // sequence, kv-head, item of the sequence
  int64_t a, x0, x1;           // item's start on the cost axis; this CTA's piece of the axis
  PromptSeq seq;
  int q0, n_tok;               // first packed row, tokens of this item
  int vis;                     // keys its last row sees
  int n, kt0, kt1;             // KV tiles: of the item, and this CTA's share

  // piece of a CTA -> tile index: monotone, 0 at the item's start, n at its end
  __device__ __forceinline__ int cut(int64_t y, int64_t cost) const {
    if (y <= 0 || n == 0) return 0;
    return y >= cost ? n : min(n, (int)((float)y * __fdividef((float)n, (float)cost)));
  }
  __device__ __forceinline__ void fill(const PromptParams& p) {
    const int tt = 2 * p.tok_tile;
    q0 = seq.q0 + t * tt;
    n_tok = min(tt, seq.n - t * tt);
    vis = p.causal ? max(0, min(seq.len, seq.len - seq.n + t * tt + n_tok)) : seq.len;
    n = (vis + kPaKeys - 1) / kPaKeys;
    const int64_t cost = seq.add + seq.step * (t + 1);
    kt0 = cut(x0 - a, cost);
    kt1 = cut(x1 - a, cost);
  }
  // first item of the piece (fill() follows): s, seq and `base`, the cost before s, are known
  __device__ __forceinline__ void start(const PromptParams& p, int64_t base) {
    const int64_t per = prompt_items_cost(seq, seq.tiles);
    h = (int)__fdividef((float)(x0 - base), (float)per);  // about; the next lines make it exact
    h = min(max(h, 0), p.n_kv_heads - 1);
    while (h > 0 && h * per > x0 - base) --h;
    while (h + 1 < p.n_kv_heads && (h + 1) * per <= x0 - base) ++h;
    const int64_t y = x0 - base - h * per;
    int lo = 0, hi = seq.tiles - 1;                      // largest t with cost(0 .. t-1) <= y
    while (lo < hi) {
      const int m = (lo + hi + 1) >> 1;
      if (prompt_items_cost(seq, m) <= y) lo = m; else hi = m - 1;
    }
    t = lo;
    a = base + h * per + prompt_items_cost(seq, t);
  }
  // the next item (fill() follows); false when the piece is done
  __device__ __forceinline__ bool next(const PromptParams& p) {
    a += seq.add + seq.step * (t + 1);
    if (a >= x1) return false;
    if (++t == seq.tiles) {
      t = 0;
      if (++h == p.n_kv_heads) {
        h = 0;
        do {
          if (++s >= p.n_seq) return false;
          seq = prompt_seq(p, s);
        } while (seq.tiles == 0);
      }
    }
    return true;
  }
  // this CTA has tiles of the item, or the item has none and starts here
  __device__ __forceinline__ bool mine() const { return kt1 > kt0 || (n == 0 && x0 <= a); }
  __device__ __forceinline__ bool whole() const { return kt0 == 0 && kt1 == n; }
  __device__ __forceinline__ bool two(const PromptParams& p) const { return n_tok > p.tok_tile; }
};

// What the other warps need of an item: the scheduling warp hands it to them through shared
// memory, so that the cost axis and its 64-bit arithmetic live in one warp's registers.
struct __align__(16) PromptWork {
  int n_tiles;                 // KV tiles of this CTA's share; -1: no more items
  int kt0, vis, len;           // first tile; keys the item's last row sees; the sequence's keys
  int lim0;                    // keys token 0 of the item sees (causal), or len
  int q0, n_tok, h;            // first packed row, tokens, kv-head
  int s, k0;                   // sequence; first packed key
  int two, slot;               // two row tiles; workspace slot, or -1: written directly
};
constexpr int kPaWorkRing = 4;

// ---- bounded waits -------------------------------------------------------------------- //
// A step of the pipeline takes microseconds; a wait that has not ended after two seconds sets
// the abort flag, every later wait returns at once, and the CTA runs out.
__device__ __forceinline__ bool pa_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {   // whole warp
  unsigned long long t0 = 0;
#pragma unroll 1
  for (uint32_t w = 1; !__all_sync(0xffffffffu, mbar_try_wait(bar, parity)); ++w) {   // all lanes leave together
    if (w & 63u) continue;                            // the clock is slow to read
    const unsigned long long now = global_ns();
    if (t0 == 0) t0 = now;
    if (__any_sync(0xffffffffu, *abort_flag || now - t0 > 2000000000ull)) {
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}

// The same value in every lane, in a form in which the compiler knows it.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// The K tiles have a ring of two slots, the V tiles one of three: slot and phase parity of the
// i-th tile a CTA loads.  (Two rings, each filled by one warp, which has waited for a slot's
// last release before it fills it: so no wait can mistake one round of a slot for another.)
__device__ __forceinline__ uint32_t pa_slot(int kv, uint32_t i) { return kv ? kPaKSlots + i % kPaVSlots : i % kPaKSlots; }
__device__ __forceinline__ uint32_t pa_phase(int kv, uint32_t i) { return (kv ? i / kPaVSlots : i / kPaKSlots) & 1; }

__device__ __forceinline__ void store_row16(void* row, int out_dtype, int chunk, const float (&v)[8]) {
  // eight values of a row at column 8 * chunk
  if (out_dtype == 4) {
    float4* d = reinterpret_cast<float4*>(row) + chunk * 2;
    d[0] = make_float4(v[0], v[1], v[2], v[3]);
    d[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint4 w;
    if (out_dtype == 1) { w.x = pack2<true>(v[0], v[1]); w.y = pack2<true>(v[2], v[3]); w.z = pack2<true>(v[4], v[5]); w.w = pack2<true>(v[6], v[7]); }
    else { w.x = pack2<false>(v[0], v[1]); w.y = pack2<false>(v[2], v[3]); w.z = pack2<false>(v[4], v[5]); w.w = pack2<false>(v[6], v[7]); }
    reinterpret_cast<uint4*>(row)[chunk] = w;
  }
}

// Four neighbouring lanes, each with four pieces of its row: afterwards lane q of them holds piece q
// of all four rows.  Two rounds of swaps.
template <int N>
__device__ __forceinline__ void quad_transpose(uint32_t (&pc)[4][N], int quad) {
#pragma unroll
  for (int d = 1; d <= 2; d <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j & d) continue;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint32_t a = pc[j][e], b = pc[j | d][e];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, quad & d ? a : b, d);
        pc[j][e] = quad & d ? got : a;
        pc[j | d][e] = quad & d ? b : got;
      }
    }
}

template <bool BF16>
__global__ void __launch_bounds__(kPaThreads, 1)
prompt_attn_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PromptParams p) {
  extern __shared__ uint8_t pa_raw[];
  uint8_t* sgen = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pa_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t smem = smem_u32(sgen);
  uint8_t* misc = sgen + kPaMiscOff;
  const uint32_t bars = smem + kPaMiscOff;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  auto full = [&](int i) { return bars + 8u * i; };
  auto empty = [&](int i) { return bars + 8u * (kPaSlots + i); };
  const uint32_t q_full = bars + 8u * 10, q_empty = bars + 8u * 11, done = bars + 8u * 12;
  auto s_full = [&](int w) { return bars + 8u * (13 + w); };
  auto o_full = [&](int w) { return bars + 8u * (15 + w); };
  const uint32_t x_ready = bars + 8u * 17, x_done = bars + 8u * 18;
  auto p_full = [&](int i) { return bars + 8u * (19 + i); };           // 2 * stream + half of the keys
  auto turn = [&](int w) { return bars + 8u * (23 + w); };
  auto w_full = [&](uint32_t i) { return bars + 8u * (25 + i % kPaWorkRing); };
  auto w_empty = [&](uint32_t i) { return bars + 8u * (25 + kPaWorkRing + i % kPaWorkRing); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 272);
  uint32_t* tmem_word = reinterpret_cast<uint32_t*>(misc + 276);
  volatile int64_t* first = reinterpret_cast<volatile int64_t*>(misc + 280);   // s, base
  int64_t* wsum = reinterpret_cast<int64_t*>(misc + 296);                      // 12 warp sums
  PromptWork* ring = reinterpret_cast<PromptWork*>(misc + 400);                // 4 x 48 bytes
  float2* xml = reinterpret_cast<float2*>(misc + 640);                         // behind the first sequence at 592
  static_assert(sizeof(PromptSeq) <= 48, "first sequence");

  if (threadIdx.x == 0) {
    for (int i = 0; i < kPaSlots; ++i) { mbar_init(full(i), 1); mbar_init(empty(i), 2); }
    mbar_init(q_full, 1); mbar_init(q_empty, 2); mbar_init(done, 2);
    for (int w = 0; w < 2; ++w) { mbar_init(s_full(w), 1); mbar_init(o_full(w), 1); mbar_init(turn(w), 1); }
    for (int i = 0; i < 4; ++i) mbar_init(p_full(i), 4);
    mbar_init(x_ready, 4); mbar_init(x_done, 4);
    for (int i = 0; i < kPaWorkRing; ++i) { mbar_init(w_full(i), 1); mbar_init(w_empty(i), 11); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 8) tmem_alloc(smem_u32(tmem_word), 512);
  if (warp == 9 && lane == 0) { prefetch_tensormap(&qmap); prefetch_tensormap(&kmap); prefetch_tensormap(&vmap); }
  // Launched with programmatic stream serialisation: nothing of global memory is read above.  With
  // more_late only the other partial of the rows is still in the making: the kernel starts on SMs
  // that its maker has left, and waits where it needs that partial or writes a result.
  if (!p.more_late) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's piece of the cost axis ----
  const int per_thread = (p.n_seq + kPaThreads - 1) / kPaThreads;
  const int sb = min((int)threadIdx.x * per_thread, p.n_seq), se = min(sb + per_thread, p.n_seq);
  int64_t mine = 0;
  PromptSeq seq;
  for (int s = sb; s < se; ++s) {
    seq = prompt_seq(p, s);
    mine += p.n_kv_heads * prompt_items_cost(seq, seq.tiles);
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) wsum[warp] = incl;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int64_t before = incl - mine, total = 0;
#pragma unroll 1
  for (int w = 0; w < kPaThreads / 32; ++w) {
    if (w < warp) before += wsum[w];
    total += wsum[w];
  }
  const int n_cta = (int)min((int64_t)gridDim.x, (total + kPaMinPiece - 1) / kPaMinPiece);
  const bool active = (int)blockIdx.x < n_cta;
  const int64_t piece = active ? prompt_piece(total, n_cta) : 0;
  const int64_t x0 = blockIdx.x * piece, x1 = min(total, x0 + piece);
  if (active && before <= x0 && x0 < before + mine) {
    int64_t base = before;
    for (int s = sb; s < se; ++s) {
      if (se - sb > 1) seq = prompt_seq(p, s);
      const int64_t c = p.n_kv_heads * prompt_items_cost(seq, seq.tiles);
      if (x0 < base + c) {
        first[0] = s;
        first[1] = base;
        *reinterpret_cast<PromptSeq*>(misc + 592) = seq;
        break;
      }
      base += c;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.rec[gridDim.x].kt0 = n_cta;
  __syncthreads();
  const uint32_t tmem = *tmem_word;

  // Every reader warp (softmax 8, matrix 2, V loads 1) takes the items in turn: wait, copy, give the place back.
  uint32_t n_work = 0;
  PromptWork wk;
  auto take = [&]() {
    if (!pa_wait(w_full(n_work), (n_work / kPaWorkRing) & 1, abort_flag)) return false;
    wk = ring[n_work % kPaWorkRing];
    __syncwarp();
    if (lane == 0) mbar_arrive(w_empty(n_work));
    ++n_work;
    return wk.n_tiles >= 0;
  };
  if (warp < 8) {
    // ------------------------------ softmax warpgroups ------------------------------ //
    setmaxnreg_inc<kPaSoftmaxRegs>();
    const int w = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lane_base = tmem + ((uint32_t)(warp & 3) << 21);      // lane 32 * (warp % 4)
    const uint32_t ts = lane_base + w * 128, to = lane_base + kPaColO + w * 128;
    const int tok_in = row / p.group;
    uint32_t n_s = 0, n_o = 0, n_x = 0;                                   // barrier phases used
    while (active && take()) {
      const bool two = wk.two;
      const int tok = (two ? w * p.tok_tile : 0) + tok_in;               // token of this row in the item
      const int steps = two ? wk.n_tiles : (wk.n_tiles + 1 - w) >> 1;    // one row tile: alternate KV tiles
      // The row is a query of this item.  The others hold the queries behind it or, where the group does not
      // divide 128, what the last call left in shared memory: scaled by 0 they run along and never move their
      // warp's reference (which would round the rows beside them otherwise from call to call).  Costs 1 % on
      // long prompts; a test in the condition cost 3 to 6 %.
      const bool valid = tok < wk.n_tok && row < p.tok_tile * p.group;
      const float sl = valid ? p.scale_log2 : 0.f;
      // keys [0, lim) are visible to this row
      const int lim = p.causal ? min(wk.len, wk.lim0 + tok) : wk.len;
      int left = lim - (wk.kt0 + (two ? 0 : w)) * kPaKeys;               // of them, in and behind this tile
      const int stride = two ? kPaKeys : 2 * kPaKeys;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < steps; ++j, left -= stride) {
        if (!(ok = pa_wait(s_full(w), n_s & 1, abort_flag))) break;
        ++n_s;
        tc_fence_after();
        uint32_t sreg[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(sreg[c], ts + c * 32);
        tmem_wait_ld();
        if (__any_sync(0xffffffffu, left < kPaKeys)) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i >= left) sreg[c][i] = 0xff800000u;           // -inf
        }
        const uint64_t sl2 = pack_f32x2(sl, sl);
        uint64_t ref2, sums;                                               // two fp32 sums
        // a row that has seen no key yet has m = -inf: 0 as the reference keeps exp2(-inf) = 0
        auto set_ref = [&]() { const float ref = m == -INFINITY ? 0.f : kPaLift<BF16> - m * sl; ref2 = pack_f32x2(ref, ref); };
        auto hand_over = [&](int half) {                                   // its product can start
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_full(2 * w + half));
        };
        float mx0 = -INFINITY, mx1 = -INFINITY;
        auto exps = [&](int half, bool with_max) {                         // 64 keys: P and its sums
          if (half == 0) sums = 0;
#pragma unroll
          for (int c = 2 * half; c < 2 * half + 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const uint64_t x2 = fma_f32x2(pack_u32x2(sreg[c][i], sreg[c][i + 1]), sl2, ref2);
              const float2 x = unpack_f32x2(x2);
              const uint64_t e2 = pack_f32x2(fast_exp2(x.x), fast_exp2(x.y));
              if (with_max) {      // of this half and of the other one, where the exponentials leave room
                mx0 = max3(mx0, __uint_as_float(sreg[c][i]), __uint_as_float(sreg[c][i + 1]));
                mx1 = max3(mx1, __uint_as_float(sreg[c ^ 2][i]), __uint_as_float(sreg[c ^ 2][i + 1]));
              }
              sums = add_f32x2(sums, e2);
              const float2 e = unpack_f32x2(e2);
              pk[i / 2] = pack2<BF16>(e.x, e.y);
            }
            // the first half goes when its stores have long arrived: waiting for them right away held the
            // warp up (5 % of the loop)
            if (c == 2) hand_over(0);
            tmem_st16(ts + c * 16, pk);
          }
        };
        // The exponentials start with the reference of the tiles before, beside the search for this
        // tile's maximum; only if that lies more than 2^8 above are they done again (as they are
        // for an item's first tile, which has no reference yet).
#pragma unroll 1
        for (;;) {
          set_ref();
          mx0 = mx1 = -INFINITY;
          exps(0, true);
          const float tile_max = fmaxf(mx0, mx1);
          if (!__any_sync(0xffffffffu, (tile_max - m) * sl > 8.f)) break;
          // The product that wrote O last is complete: the scores just waited for were issued
          // behind it, and the next one waits for this warpgroup.
          const float mn = fmaxf(m, tile_max);
          const float alpha = m == -INFINITY ? 0.f : fast_exp2((m - mn) * sl);
          l *= alpha;
          m = mn;
          if (j == 0) continue;
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t o[16];
            tmem_ld16(o, to + c * 16);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st16(to + c * 16, o);
          }
        }
        exps(1, false);
        hand_over(1);
        const float2 sa = unpack_f32x2(sums);
        l += sa.x + sa.y;
      }
      if (!ok) break;

      // ---- epilogue ----
      float a0 = 1.f, a1 = 0.f;                 // weights of O_w and (one row tile) of the other stream's O
      bool join = false;
      if (steps > 0) {
        if (!pa_wait(o_full(w), n_o & 1, abort_flag)) break;
        ++n_o;
        tc_fence_after();
      }
      if (!two && wk.n_tiles > 1) {
        if (w == 1) {
          xml[row] = make_float2(m, l);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(x_ready);
          if (!pa_wait(x_done, n_x & 1, abort_flag)) break;          // O1 and xml are free again
          ++n_x;
        } else {
          if (!pa_wait(x_ready, n_x & 1, abort_flag)) break;
          ++n_x;
          tc_fence_after();
          const float2 other = xml[row];
          const float mn = fmaxf(m, other.x);
          a0 = m == -INFINITY ? 0.f : fast_exp2((m - mn) * sl);
          a1 = other.x == -INFINITY ? 0.f : fast_exp2((other.x - mn) * sl);
          l = l * a0 + other.y * a1;
          m = mn;
          join = true;
        }
      }
      if (two || w == 0) {
        const bool whole = wk.slot < 0;
        const int64_t orow = (int64_t)(wk.q0 + tok) * p.n_q_heads + wk.h * p.group + (row - tok_in * p.group);
        const float m2 = m == -INFINITY ? -INFINITY : m * sl - kPaLift<BF16>;   // base-2 units, what l counts in
        float wa = l > 0.f ? 1.f / l : 0.f, wb = 0.f;
        if (l != l) wa = l;                                            // NaN scores stay NaN
        if (p.more_late) asm volatile("griddepcontrol.wait;" ::: "memory");
        if (whole && valid) {
          float lse2 = l > 0.f ? m2 + log2f(l) : (l != l ? l : -INFINITY);
          if (p.o_more) {
            const float b2 = p.lse_more[orow] * 1.4426950408889634f;
            const float top = fmaxf(lse2, b2);
            const float ea = lse2 == -INFINITY ? 0.f : exp2f(lse2 - top), eb = b2 == -INFINITY ? 0.f : exp2f(b2 - top);
            const float s = ea + eb, inv = s > 0.f ? 1.f / s : (s != s ? s : 0.f);     // a NaN on either side stays one
            wa *= ea * inv;
            wb = eb * inv;
            lse2 = s > 0.f ? top + log2f(s) : (s != s ? s : -INFINITY);
          }
          if (p.lse) p.lse[orow] = lse2 * 0.6931471805599453f;
        }
        const int prow = (two ? w * kPaRows : 0) + row;
        if (!whole) p.part_ml[(size_t)wk.slot * 256 + prow] = make_float2(m2, l);
        float4* po = p.part_o + (size_t)max(wk.slot, 0) * 32 * 256 + prow;
        // 16 columns of this row's O, of both streams where they share the row tile
        auto columns = [&](uint32_t (&o)[16], int col) {
          tmem_ld16(o, to + col);
          if (join) {
            uint32_t o1[16];
            tmem_ld16(o1, to + 128 + col);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i)
              o[i] = __float_as_uint(__uint_as_float(o[i]) * a0 + __uint_as_float(o1[i]) * a1);
          }
          tmem_wait_ld();
          if (steps == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = 0u;
          }
        };
        if (!whole) {
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t o[16];
            columns(o, c * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              po[(c * 4 + i) * 256] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                  __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
          }
        } else {
          // Written directly, a row is 256 bytes of its own: 32 lanes that store 16 bytes each of their
          // rows touch 32 cache lines per instruction, and the store path takes about three
          // cycles a line (an item's epilogue took 5000 to 10000 cycles).  Four lanes swap pieces
          // first, so that a line is touched for 64 bytes at a time.
          const int quad = lane & 3;
          int64_t qrow[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) qrow[i] = __shfl_sync(0xffffffffu, valid ? orow : (int64_t)-1, (lane & 28) + i);
          if (!p.o_more && p.out_dtype != 4) {
            uint4* dst[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[i] = static_cast<uint4*>(p.out) + qrow[i] * (kHeadDim / 8) + quad;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t pc[4][4];                                 // [piece of 8 columns][2 values each]
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                uint32_t o[16];
                columns(o, c * 32 + k * 16);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float u = __uint_as_float(o[2 * i]) * wa, v = __uint_as_float(o[2 * i + 1]) * wa;
                  pc[2 * k + (i >> 2)][i & 3] = p.out_dtype == 1 ? pack2<true>(u, v) : pack2<false>(u, v);
                }
              }
              quad_transpose(pc, quad);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (qrow[i] >= 0) *dst[i] = make_uint4(pc[i][0], pc[i][1], pc[i][2], pc[i][3]);
                dst[i] += 4;
              }
            }
          } else {
            float qwb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) qwb[i] = __shfl_sync(0xffffffffu, wb, (lane & 28) + i);
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t pc[4][4];                                 // [piece of 4 columns]
              columns(reinterpret_cast<uint32_t(&)[16]>(pc), c * 16);
#pragma unroll
              for (int i = 0; i < 16; ++i) pc[i >> 2][i & 3] = __float_as_uint(__uint_as_float(pc[i >> 2][i & 3]) * wa);
              quad_transpose(pc, quad);
              float4 x[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (qwb[i] != 0.f && qrow[i] >= 0)
                  x[i] = *reinterpret_cast<const float4*>(p.o_more + qrow[i] * kHeadDim + c * 16 + quad * 4);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (qrow[i] < 0) continue;
                const int64_t at = qrow[i] * kHeadDim + c * 16 + quad * 4;
                const float4 v = make_float4(fmaf(x[i].x, qwb[i], __uint_as_float(pc[i][0])),
                                             fmaf(x[i].y, qwb[i], __uint_as_float(pc[i][1])),
                                             fmaf(x[i].z, qwb[i], __uint_as_float(pc[i][2])),
                                             fmaf(x[i].w, qwb[i], __uint_as_float(pc[i][3])));
                const bool bf = p.out_dtype == 1;
                if (p.out_dtype == 4)
                  *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = v;
                else
                  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
                      make_uint2(bf ? pack2<true>(v.x, v.y) : pack2<false>(v.x, v.y),
                                 bf ? pack2<true>(v.z, v.w) : pack2<false>(v.z, v.w));
              }
            }
          }
        }
        tc_fence_before();
        if (join) {
          __syncwarp();
          if (lane == 0) mbar_arrive(x_done);
        }
      }
    }
  } else {
    setmaxnreg_dec<kPaOtherRegs>();
    if (warp == 8 || warp == 11) {
      // ------------ work list, Q and K tiles: warp 8; V tiles: warp 11 ------------ //
      // Every operand of a TMA instruction is made uniform first: with per-lane operands (a lane
      // per box) the instructions of a tile go out one by one at 100 cycles each, 1600 for 128
      // keys in pages of 16, as long as the tile's products.
      const int kv = warp == 11 ? 1 : 0;
      const CUtensorMap* map = kv ? &vmap : &kmap;
      const int boxes = kPaKeys / p.box_tok;              // of one half tile
      const uint32_t box_bytes = (uint32_t)p.box_tok * 128u;
      const bool paged = p.seq_lens != nullptr;
      uint32_t n_tile = 0, n_q = 0;                       // tiles and Q loads issued
      bool ok = active;
      PromptItem it;
      it.s = -1;
      it.x0 = x0;
      it.x1 = x1;
      bool recorded = false;
      uint32_t n_given = 0;
      // the work list: what this warp puts into the ring the other warps take out
      auto give = [&](const PromptWork& v) {
        if (!pa_wait(w_empty(n_given), ((n_given / kPaWorkRing) & 1) ^ 1, abort_flag)) return false;
        if (lane == 0) {
          ring[n_given % kPaWorkRing] = v;
          mbar_arrive(w_full(n_given));
        }
        __syncwarp();
        ++n_given;
        return v.n_tiles >= 0;
      };
      auto make = [&]() {
        bool have = true;
        do {
          if (it.s < 0) {
            it.s = (int)first[0];
            it.seq = *reinterpret_cast<const PromptSeq*>(misc + 592);
            it.start(p, first[1]);
          } else {
            have = it.next(p);
          }
          if (have) it.fill(p);
        } while (have && !it.mine() && recorded);
        if (!recorded) {                             // what the join needs of the first item
          recorded = true;
          if (lane == 0) {
            PromptRec r;
            r.a = it.a; r.mid = it.x0 > it.a ? 1 : 0; r.kt0 = it.kt0; r.kt1 = it.kt1; r.n = it.n;
            r.q0 = it.q0; r.n_tok = it.n_tok; r.h = it.h; r.pad = 0;
            p.rec[blockIdx.x] = r;
          }
        }
        wk.n_tiles = have ? it.kt1 - it.kt0 : -1;
        wk.kt0 = it.kt0; wk.vis = it.vis; wk.len = it.seq.len;
        wk.lim0 = it.seq.len - it.seq.n + (it.q0 - it.seq.q0) + 1;
        wk.q0 = it.q0; wk.n_tok = it.n_tok; wk.h = it.h; wk.s = it.s; wk.k0 = it.seq.k0;
        wk.two = it.two(p) ? 1 : 0;
        wk.slot = it.whole() ? -1 : 2 * (int)blockIdx.x + (it.x0 > it.a ? 0 : 1);
        return give(wk);
      };
      while (ok && (kv == 0 ? make() : take())) {
        const int n_tiles = uniform(wk.n_tiles), h = uniform(wk.h), two = uniform(wk.two);
        if (n_tiles == 0) continue;
        const int kt0 = uniform(wk.kt0), vis = uniform(wk.vis), k0 = uniform(wk.k0);
        const int32_t* row = paged ? p.block_table + (int64_t)wk.s * p.bt_stride : nullptr;
        // lane b: the page of box b of tile i, read a few tiles ahead of its use
        auto fetch = [&](int i) {
          const int key = (kt0 + i) * kPaKeys + lane * p.box_tok;
          if (!paged || i >= n_tiles || lane >= boxes || key >= vis) return 0;
          const int page = __ldg(row + key / p.page_size);
          if (page >= 0 && page < p.n_pages) return page;
          if (p.status) atomicOr(p.status, kStBadPage);
          return 0;
        };
        auto load = [&](int i, int page) {
          const uint32_t slot = pa_slot(kv, n_tile);
          if (!pa_wait(empty(slot), pa_phase(kv, n_tile) ^ 1, abort_flag)) return false;
          ++n_tile;
          const int key0 = (kt0 + i) * kPaKeys;
          const int n_box = min(boxes, (vis - key0 + p.box_tok - 1) / p.box_tok);   // >= 1
          const uint32_t dst = smem + kPaRingOff + slot * kPaTileBytes, bar = full(slot);
          if (elect_one()) mbar_arrive_expect_tx(bar, n_box * 2 * box_bytes);
          __syncwarp();
          if (!paged) {
            if (elect_one()) {
              const int c1 = p.head_major ? k0 + key0 : h, c2 = p.head_major ? h : k0 + key0;
              tma_load_4d_keep(dst, map, bar, 0, c1, c2, 0);
              tma_load_4d_keep(dst + kPaHalfBytes, map, bar, 64, c1, c2, 0);
            }
          } else {
            int pg[8];                                     // at most 128 / 16 boxes of a half tile
#pragma unroll
            for (int b = 0; b < 8; ++b) pg[b] = __shfl_sync(0xffffffffu, page, b);
            int tok = key0 % p.page_size;
            if (elect_one()) {
#pragma unroll
              for (int b = 0; b < 8; ++b) {
                if (b >= n_box) break;
                const int c1 = p.head_major ? tok : h, c2 = p.head_major ? h : tok;
                tma_load_4d_keep(dst + b * box_bytes, map, bar, 0, c1, c2, pg[b]);
                tma_load_4d_keep(dst + kPaHalfBytes + b * box_bytes, map, bar, 64, c1, c2, pg[b]);
                tok += p.box_tok;
                if (tok >= p.page_size) tok = 0;
              }
            }
          }
          __syncwarp();
          return true;
        };
        int p0 = fetch(0), p1 = fetch(1), p2 = fetch(2);
        // Q: the group's heads of up to 2 * tok_tile tokens, in two halves of 64 values
        if (kv == 0) {
          if (!(ok = pa_wait(q_empty, (n_q & 1) ^ 1, abort_flag))) break;
          ++n_q;
          const int q0 = uniform(wk.q0);
          if (elect_one()) {
            const uint32_t half = (uint32_t)p.tok_tile * p.group * 128u;
            mbar_arrive_expect_tx(q_full, half * (two ? 4u : 2u));
#pragma unroll 1
            for (int w = 0; w < (two ? 2 : 1); ++w)
              for (int d = 0; d < 2; ++d)
                tma_load_3d(smem + w * kPaTileBytes + d * kPaHalfBytes, &qmap, q_full, d * 64, h * p.group,
                            q0 + w * p.tok_tile);
          }
          __syncwarp();
        }
#pragma unroll 1
        for (int i = 0; i < n_tiles && ok; ++i) {
          ok = load(i, p0);
          p0 = p1;
          p1 = p2;
          p2 = fetch(i + 3);
        }
      }
      if (*abort_flag) {   // give the copies in flight a bounded chance to land before the CTA goes away
        for (uint32_t back = 1; back <= (uint32_t)(kv ? kPaVSlots : kPaKSlots) && back <= n_tile; ++back)
          mbar_wait_bounded(full(pa_slot(kv, n_tile - back)), pa_phase(kv, n_tile - back), kPollLimit);
        if (n_q) mbar_wait_bounded(q_full, (n_q - 1) & 1, kPollLimit);
      }
    } else {
      // ------------------------------- matrix instructions ----------------------------- //
      // Warp 9 issues stream 0's, warp 10 stream 1's: one warp for both spent as long on waits and
      // issue between the products as the products took.  The warp stays together; one elected
      // lane issues.  Every ring slot is given back by both streams.
      constexpr uint32_t idesc_qk = umma_idesc(BF16, false, kPaRows, kPaKeys);
      constexpr uint32_t idesc_pv = umma_idesc(BF16, true, kPaRows, kHeadDim);
      const int w = warp - 9;
      uint32_t n_tile = 0, n_q = 0, n_p = 0, n_turn = 0;
      bool ok = true;
      auto wait_tile = [&](int kv, uint32_t i) { return pa_wait(full(pa_slot(kv, i)), pa_phase(kv, i), abort_flag); };
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t q_lo = umma_desc_lo(smem, 16), ring_k = umma_desc_lo(smem + kPaRingOff, 16),
                     ring_v = umma_desc_lo(smem + kPaRingOff, kPaHalfBytes);
      constexpr uint32_t hi = umma_desc_hi(1024), tile16 = kPaTileBytes / 16, half16 = kPaHalfBytes / 16;
      auto qk = [&](int qtile, uint32_t i) {         // S_w = Q K^T
        const uint32_t qa = q_lo + qtile * tile16, ka = ring_k + pa_slot(0, i) * tile16;
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint32_t off = (ks >> 2) * half16 + (ks & 3) * 2;
            umma_ss(tm + w * 128, qa + off, hi, ka + off, hi, idesc_qk, ks > 0 ? 1u : 0u);
          }
          umma_commit(s_full(w));
        }
        __syncwarp();
      };
      // O_w (+)= P_w V, in two halves of the keys as P arrives
      auto pv = [&](uint32_t i, int ksteps, bool first_tile, bool in_turn) {
        const uint32_t va = ring_v + pa_slot(1, i) * tile16, keep = first_tile ? 0u : 1u;
        const uint32_t phase = n_p++;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!pa_wait(p_full(2 * w + half), phase & 1, abort_flag)) return false;
          if (in_turn && half == 0 && !pa_wait(turn(w), (n_turn++ & 1) ^ (w == 0 ? 1u : 0u), abort_flag)) return false;
          tc_fence_after();
          if (elect_one()) {
            if (ksteps == 8) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int ks = 4 * half + k;
                umma_ts(tm + kPaColO + w * 128, tm + w * 128 + ks * 8, va + ks * 128, hi, idesc_pv, ks > 0 ? 1u : keep);
              }
            } else {
#pragma unroll 1
              for (int ks = 4 * half; ks < min(4 * half + 4, ksteps); ++ks)
                umma_ts(tm + kPaColO + w * 128, tm + w * 128 + ks * 8, va + ks * 128, hi, idesc_pv, ks > 0 ? 1u : keep);
            }
          }
          __syncwarp();
        }
        return true;
      };
      // V rows of the last 16-key step that lie behind the sequence hold whatever the page holds:
      // their weights are 0, but 0 * NaN is not, so they are cleared in shared memory.
      auto clean = [&](uint32_t i, int kt, int ksteps) {
        const int from = wk.len - kt * kPaKeys, to = ksteps * 16;
        uint8_t* v = sgen + kPaRingOff + pa_slot(1, i) * kPaTileBytes;
#pragma unroll 1
        for (int r = max(from, 0); r < to; ++r) {
          *reinterpret_cast<uint32_t*>(v + r * 128 + lane * 4) = 0u;
          *reinterpret_cast<uint32_t*>(v + kPaHalfBytes + r * 128 + lane * 4) = 0u;
        }
        fence_proxy_async();
        __syncwarp();
      };
      // (all commits from one thread: elect_one picks the same lane every time)
      auto commit = [&](uint32_t bar) { if (elect_one()) umma_commit(bar); __syncwarp(); };
      auto give_back = [&](int kv, uint32_t i) { commit(empty(pa_slot(kv, i))); };
      while (ok && active && take()) {
        const int n_tiles = uniform(wk.n_tiles);
        if (n_tiles == 0) continue;
        if (!(ok = pa_wait(q_full, n_q & 1, abort_flag))) break;
        ++n_q;
        const uint32_t base = n_tile;
        n_tile += n_tiles;
        // V tile i of the item: product and release
        auto values = [&](int i, bool first_tile, bool in_turn) {
          const int kt = wk.kt0 + i, ks = min(8, (wk.vis - kt * kPaKeys + 15) >> 4);
          if (!wait_tile(1, base + i)) return false;
          if (ks * 16 > wk.len - kt * kPaKeys) clean(base + i, kt, ks);
          if (!pv(base + i, ks, first_tile, in_turn)) return false;
          give_back(1, base + i);
          return true;
        };
        auto pass = [&](int kv, int i) {
          if (!wait_tile(kv, base + i)) return false;
          if (elect_one()) mbar_arrive(empty(pa_slot(kv, base + i)));
          __syncwarp();
          return true;
        };
        auto scores = [&](int i, int qtile) {
          if (!wait_tile(0, base + i)) return false;
          qk(qtile, base + i);
          give_back(0, base + i);
          return true;
        };
        // Two row tiles: both streams take every tile, and they issue in turn: O_0 (+)= P_0 V and the
        // next S_0, then the same of stream 1.  Left alone they fall into step, and the
        // exponentials of both wait for the tensor cores and then compete (4300 cycles a step
        // instead of 3100 when this was put in).  One row tile: stream w takes tiles w, w + 2, ..., and lets the
        // others pass, so that no slot is filled again before both have seen it.
        const bool two = uniform(wk.two);
        const int ahead = two ? 1 : 2;                  // scores a stream is ahead of its values
#pragma unroll 1
        for (int t = 0; t < n_tiles + ahead; ++t) {
          const int i = t - ahead;
          const bool mine = two || (t & 1) == w;        // of tile t and, ahead being 1 or 2, of tile i
          if (i >= 0) {
            if (mine) {
              if (!(ok = values(i, i < (two ? 1 : 2), two))) break;
              if (i + (two ? 1 : 2) >= n_tiles) commit(o_full(w));
            } else if (!(ok = pass(1, i))) {
              break;
            }
          }
          if (t < n_tiles) {
            if (!(ok = mine ? scores(t, two ? w : 0) : pass(0, t))) break;
            if (t + 1 == n_tiles) commit(q_empty);
          }
          if (two && i >= 0) {
            if (elect_one()) mbar_arrive(turn(w ^ 1));
            __syncwarp();
          }
        }
      }
      // everything issued is complete, and its arrivals have landed, before the CTA goes away
      commit(done);
      mbar_wait_bounded(done, 0, kPollLimit);
    }
  }
  // (the join takes the end of this kernel for the end of the one before)
  if (p.more_late) asm volatile("griddepcontrol.wait;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag && p.status) atomicOr(p.status, kStPipeTimeout);
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds up the pieces of the items that were cut, in the order of their keys.  Every block reads
// what each CTA did first (one record a thread), lists the items that were cut, and takes
// tasks of (item, 8 of the 128 values); one thread per row, so a piece's values come in
// 4 KB runs.  The pieces are a few MB that were written a moment ago: L2.
constexpr int kPjTasks = 16;
// Pieces in flight per thread: a join is a few trips to the L2, not one per piece.  (4: packed short prompts
// 28.8 us instead of 29.6, but 64 sequences behind 32768 tokens, 18 pieces an item, 2.4 us more.)
constexpr int kPjBatch = 8;
__global__ void __launch_bounds__(256) prompt_join_kernel(const PromptParams p, int n_grid) {
  __shared__ int64_t s_a[kPaMaxCtas];
  __shared__ int s_kt0[kPaMaxCtas], s_kt1[kPaMaxCtas], s_n[kPaMaxCtas];
  __shared__ int4 s_item[kPaMaxCtas];                      // first row, tokens, kv-head, first entry of its list
  __shared__ int s_count[kPaMaxCtas], s_slot[2 * kPaMaxCtas], s_cnt[8];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, row = tid;
  PromptRec r;
  if (tid < n_grid) r = p.rec[tid];                        // (only those of the first n_cta are this launch's)
  const int n_cta = p.rec[n_grid].kt0;
  if (n_cta <= 1) return;
  if (tid < n_cta) {
    s_a[tid] = r.mid ? r.a : -1;                           // -1: starts with an item of its own
    s_kt0[tid] = r.kt0; s_kt1[tid] = r.kt1; s_n[tid] = r.n;
  }
  __syncthreads();
  // CTA c is the first to start inside an item that several CTAs share
  bool head = false;
  int last = tid;
  if (tid > 0 && tid < n_cta && s_a[tid] >= 0 && s_a[tid - 1] != s_a[tid] && s_kt0[tid] < s_n[tid]) {
    head = true;
    for (int c = tid; c < n_cta && s_a[c] == s_a[tid]; ++c) {
      if (s_kt0[c] == 0 && s_kt1[c] == s_n[c]) head = false;   // one CTA did all of it, and wrote it
      last = c;
    }
  }
  const unsigned mask = __ballot_sync(0xffffffffu, head);
  if ((tid & 31) == 0) s_cnt[tid >> 5] = __popc(mask);
  __syncthreads();
  int at = __popc(mask & ((1u << (tid & 31)) - 1)), n_items = 0;
  for (int w = 0; w < 8; ++w) {
    if (w < (tid >> 5)) at += s_cnt[w];
    n_items += s_cnt[w];
  }
  if (head) {
    // the item's pieces in order: the last item of CTA tid - 1, the first items of tid .. last,
    // those that are not empty.  Lists cannot overlap: an item has at most last - tid + 2 entries
    int e = tid + at;
    s_item[at] = make_int4(r.q0, r.n_tok, r.h, e);
    if (s_kt0[tid] > 0) s_slot[e++] = 2 * (tid - 1) + 1;
    for (int c = tid; c <= last; ++c)
      if (s_kt1[c] > s_kt0[c]) s_slot[e++] = 2 * c;
    s_count[at] = e - (tid + at);
  }
  __syncthreads();

  for (int task = blockIdx.x; task < n_items * kPjTasks; task += gridDim.x) {
    const int4 item = s_item[task / kPjTasks];
    const int col = task % kPjTasks, n = s_count[task / kPjTasks];
    const int* slots = s_slot + item.w;
    const int w = row >> 7, lr = row & 127;
    const int tok_in = lr / p.group, tok = w * p.tok_tile + tok_in;
    if ((w && item.y <= p.tok_tile) || lr >= p.tok_tile * p.group || tok >= item.y) continue;
    const int64_t orow = (int64_t)(item.x + tok) * p.n_q_heads + item.z * p.group + (lr - tok_in * p.group);
    // one pass with a running maximum, a batch of pieces at a time
    float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    if (p.o_more) {
      m = p.lse_more[orow] * 1.4426950408889634f;
      if (m != -INFINITY) {
        const float4* more = reinterpret_cast<const float4*>(p.o_more + orow * kHeadDim + col * 8);
        const float4 x = more[0], y = more[1];
        l = 1.f;
        acc[0] = x.x; acc[1] = x.y; acc[2] = x.z; acc[3] = x.w; acc[4] = y.x; acc[5] = y.y; acc[6] = y.z; acc[7] = y.w;
      }
    }
    for (int i0 = 0; i0 < n; i0 += kPjBatch) {
      float2 ml[kPjBatch];
      float4 x[kPjBatch], y[kPjBatch];
#pragma unroll
      for (int k = 0; k < kPjBatch; ++k) {
        ml[k] = make_float2(-INFINITY, 0.f);
        x[k] = y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i0 + k < n) {
          const size_t slot = slots[i0 + k];
          ml[k] = p.part_ml[slot * 256 + row];
          const float4* po = p.part_o + slot * 32 * 256 + (size_t)col * 2 * 256 + row;
          x[k] = po[0];
          y[k] = po[256];
        }
      }
      float mn = m;
#pragma unroll
      for (int k = 0; k < kPjBatch; ++k) mn = fmaxf(mn, ml[k].x);
      const float keep = m == -INFINITY ? 0.f : fast_exp2(m - mn);
      m = mn;
      l *= keep;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] *= keep;
#pragma unroll
      for (int k = 0; k < kPjBatch; ++k) {
        const float f = ml[k].x == -INFINITY ? (ml[k].y == ml[k].y ? 0.f : ml[k].y) : fast_exp2(ml[k].x - m);
        l += ml[k].y * f;
        acc[0] += x[k].x * f; acc[1] += x[k].y * f; acc[2] += x[k].z * f; acc[3] += x[k].w * f;
        acc[4] += y[k].x * f; acc[5] += y[k].y * f; acc[6] += y[k].z * f; acc[7] += y[k].w * f;
      }
    }
    const float inv = l > 0.f ? 1.f / l : (l != l ? l : 0.f);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= inv;
    uint8_t* dst = reinterpret_cast<uint8_t*>(p.out) + orow * kHeadDim * (p.out_dtype == 4 ? 4 : 2);
    store_row16(dst, p.out_dtype, col, acc);
    if (p.lse && col == 0)
      p.lse[orow] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : (l != l ? l : -INFINITY);
  }
}

}  // namespace pkv
