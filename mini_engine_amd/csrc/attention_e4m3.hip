// Attention over the 8-bit paged cache (e4m3.h) on the CDNA4 matrix cores, compiled once per head size with -DME_HEAD_DIM=<D>
// (a multiple of 16 up to 256): queries and results bfloat16, keys and values e4m3 under a power of two per 16 tokens and head.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j),  over the keys j that the query sees; a sink adds exp(sink) to
//   the denominator.
//
// Everything is computed transposed, as S^T = K Q^T and O^T += V^T P^T; a "column" is one (query token, query head) pair of a key head.
// Maxima, sums and accumulators are float32 and per column; probabilities are rounded to bfloat16 for the second product, as they are
// over a bfloat16 cache. A result's distance from the formula's is so 1.2 to 1.4 times that of one rounding to bfloat16 at the end. The
// denominator sums them unrounded for single tokens, and as rounded for prompts, whose sum takes two of them at a time so.
//
// The stored numbers times their power are bfloat16 numbers: what the products take turned into such is turned exactly
// (v_cvt_scalef32_pk_bf16_fp8, two numbers and the power in one instruction). So it is for single tokens, where both products run on
// v_mfma_f32_16x16x32_bf16 over blocks of 64 keys. With n = lane & 15, g = lane >> 4:
//   * the four tiles of S^T let row m of tile tt stand for key 16 (m / 4) + 4 tt + m % 4, so lane (n, g) ends with the 16 keys
//     16 g .. 16 g + 15 of column n in order: the operand of the second product, without a movement of data;
//   * a lane reads 16 bytes of keys (16 channels 64 j + 16 g ..) and of values (16 keys 16 g .. of channel 16 dt + n) at a time: two
//     products' operands each. Which channel lies in which slot of the first product is free as long as the queries follow;
//   * every lane's keys of a block lie under one power, and so do its values: one byte and a shift per lane.
// Prompts are described at their kernel.
//
// Keys that a column does not see are replaced, never multiplied by zero: scores by "none", stored values by zero bytes where no
// column sees them; and where some columns of a prompt's tile see a key whose value is NaN and others do not, the tile's columns are done
// once more one by one.
#include "kv_e4m3.h"
#include <type_traits>

#ifndef ME_HEAD_DIM
#error "compile with -DME_HEAD_DIM=<multiple of 16>"
#endif
constexpr int HD = ME_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size");
constexpr int DT = HD / 16;              // 16-channel tiles of the output
constexpr int KL = (HD + 63) / 64;       // 16-byte loads of a key row per lane
constexpr int BK = 64;                   // keys of a block
constexpr float NONE = -1e30f;           // "no key yet": finite, so that differences never give NaN
constexpr float LOG2E = 1.4426950408889634f;
// log2 units by which a column's maximum must rise before its sums are rescaled: probabilities then reach 2^8 instead of 1, which
// neither float32 sums nor bfloat16's relative rounding minds, and blocks after a tile's first hardly ever rescale.
constexpr float RESCALE_STEP = 8.f;
constexpr float MOST_WEIGHT = 4096.f;          // ... and, of prompts, the sum of a lane's weights of a block up to which it stays

struct Attn8Args {
  const bf16_t* q;
  int64_t q_stride;
  bf16_t* out;
  int64_t out_stride;
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* k_powers;
  const uint8_t* v_powers;
  int num_pages;
  const int32_t* tables;         // [num_seqs, table_stride] page ids; entries that hold no page: below 0 or beyond num_pages
  int table_stride, table_cols;
  const int32_t* contexts;       // [num_seqs] keys after this step's write
  const int32_t* cu;             // prompts: [num_seqs + 1] prefix sums of new tokens
  int num_seqs;
  int Hq, Hkv, G, page_shift;
  float scale;
  int window, chunk;             // > 0: the last `window` keys, or the keys of the query's own block of `chunk` positions
  int part_keys, num_parts;      // keys of a partition (a multiple of 64) and how many of them a launch has
  float* part_o;                 // [rows, Hq, num_parts, HD] unnormalised
  float* part_ml;                // [rows, Hq, num_parts, 2] maximum (log2 domain) and sum
  const float* sinks;            // [Hq] or nullptr
  int64_t rows;                  // prompts: their tokens
};

__device__ __forceinline__ int first_seen(const Attn8Args& a, int pos) {
  if (a.chunk > 0) return pos - pos % a.chunk;
  return a.window > 0 ? max(0, pos - a.window + 1) : 0;
}
__device__ __forceinline__ int context_of(const Attn8Args& a, int b) {
  return (int)min((int64_t)max(a.contexts[b], 0), (int64_t)a.table_cols << a.page_shift);
}

__device__ __forceinline__ float max_of_column(float v) {      // over the four lanes of a column, left in all of them
  unsigned u = __float_as_uint(v);
  auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  u = __float_as_uint(v);
  auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float sum_of_column(float v) {
  unsigned u = __float_as_uint(v);
  auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  u = __float_as_uint(v);
  auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Eight stored numbers (two words) times a power of two, as the operand of a product.
__device__ __forceinline__ bf16x8 operand(uint32_t w0, uint32_t w1, float power) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, power, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, power, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, power, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, power, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// (a byte that no append has written may be anything)
__device__ __forceinline__ uint32_t code_of(uint32_t byte) { return min(max(byte, (uint32_t)(E4_LEAST + E4_BIAS)), (uint32_t)(E4_MOST + E4_BIAS)); }
__device__ __forceinline__ float power_of(uint32_t byte) { return __uint_as_float(code_of(byte) << 23); }

// A block's keys and values as they lie in memory. Loads are unconditional: a lane whose keys are not to be read (at or past the
// context, in front of what anybody sees, in a table entry without a page) reads page 0, which is always there.
struct Pages {
  int k, v;            // table entries as loaded
};
// Keys and values of single tokens are read once: marked as not to be kept by the caches, which the memory system answers with a higher rate.
__device__ __forceinline__ u32x4v stream16(const uint8_t* p) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4v*>(p)); }
struct Block {
  u32x4v k[4][KL], v[DT];
  uint32_t kcode, vcode;
  bool there;          // this lane's 16 keys (of the scores and of the values) lie in a page
};
__device__ __forceinline__ bool group_in(int key, int lo, int L) { return key < L && key + E4_BLOCK > lo; }

__device__ __forceinline__ Pages find_pages(const Attn8Args& a, const int32_t* __restrict__ table, int t0, int lo, int L, int n, int g) {
  const int kk = t0 + 16 * (n >> 2), vk = t0 + 16 * g;
  Pages p;
  p.k = table[group_in(kk, lo, L) ? kk >> a.page_shift : 0];
  p.v = table[group_in(vk, lo, L) ? vk >> a.page_shift : 0];
  return p;
}
__device__ __forceinline__ void load_keys(const Attn8Args& a, const Pages& p, int kvh, int t0, int lo, int L, int n, int g, Block& b) {
  const int kk = t0 + 16 * (n >> 2), off = kk & ((1 << a.page_shift) - 1);
  const bool ok = group_in(kk, lo, L) && (unsigned)p.k < (unsigned)a.num_pages;
  const int64_t at = (int64_t)(ok ? p.k : 0) * a.Hkv + kvh;
  const uint8_t* from = a.k + ((at << a.page_shift) + off + (n & 3)) * HD + 16 * g;
#pragma unroll
  for (int tt = 0; tt < 4; ++tt)
#pragma unroll
    for (int j = 0; j < KL; ++j)
      b.k[tt][j] = stream16(from + tt * 4 * HD + ((HD % 64 == 0 || 64 * j + 16 * g < HD) ? 64 * j : -16 * g));
  b.kcode = a.k_powers[(at << (a.page_shift - 4)) + (off >> 4)];
}
__device__ __forceinline__ void load_values(const Attn8Args& a, const Pages& p, int kvh, int t0, int lo, int L, int n, int g, Block& b) {
  const int vk = t0 + 16 * g, off = vk & ((1 << a.page_shift) - 1);
  b.there = group_in(vk, lo, L) && (unsigned)p.v < (unsigned)a.num_pages;
  const int64_t at = (int64_t)(b.there ? p.v : 0) * a.Hkv + kvh;
  const uint8_t* from = a.v + ((at * HD + n) << a.page_shift) + off;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) b.v[dt] = stream16(from + ((int64_t)(16 * dt) << a.page_shift));
  b.vcode = a.v_powers[(at << (a.page_shift - 4)) + (off >> 4)];
}

// The queries of one column, in the order of the channels that load_keys gives a lane.
__device__ __forceinline__ void load_q(const bf16_t* row, bool valid, int g, bf16x8 (&q)[2 * KL]) {
#pragma unroll
  for (int j = 0; j < KL; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in = HD % 64 == 0 || 64 * j + 16 * g < HD;
      bf16x8 x = *reinterpret_cast<const bf16x8*>(row + (in ? 64 * j + 16 * g + 8 * h : 0));
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = valid && in ? x[e] : static_cast<bf16_t>(0.f);
      q[2 * j + h] = x;
    }
}

// Zero bytes where none of the tile's columns sees the key: at and past L, in front of lo, in no page.
__device__ __forceinline__ void hide_values(Block& b, int t0, int lo, int L, int g) {
  const int from = b.there ? max(lo - (t0 + 16 * g), 0) : 16, to = L - (t0 + 16 * g);      // keys [from, to) of this lane's 16 stay
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int x = min(max(from - 4 * w, 0), 4), y = min(max(to - 4 * w, 0), 4);
    const uint32_t upto = y == 4 ? 0xffffffffu : (1u << (8 * y)) - 1u, below = x == 4 ? 0xffffffffu : (1u << (8 * x)) - 1u;
    const uint32_t keep = upto & ~below;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) b.v[dt][w] &= keep;
  }
}

struct Column {
  int lo, hi;                    // keys [lo, hi] that the column sees (hi < lo: none)
  float m, l;                    // reference point of the exponentials (log2 domain), this lane's share of the sum
  f32x4 acc[DT];
};

// The softmax of a block's scores (16 keys of a lane, from `first` on): under the column's reference point, which rises where it must (the
// column's sums with it), their probabilities are added to the sum and rounded to bfloat16 as the second product's operand (the sum
// takes them unrounded). FULL: the column sees all keys. there: they lie in a page.
template <bool FULL>
__device__ __forceinline__ void softmax(const f32x4 (&st)[4], float sc, int first, bool there, Column& c, bf16x8 (&pb)[2]) {
  float s[16];
  float top = NONE;
  uint32_t seen = 0;
  if constexpr (!FULL) {
    const int from = max(c.lo - first, 0), to = min(c.hi - first, 15);
    seen = there && to >= from && from < 16 ? (2u << to) - (1u << from) : 0u;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i] = st[i >> 2][i & 3] * sc;
    if constexpr (!FULL) s[i] = (seen >> i) & 1 ? s[i] : NONE;
    top = fmaxf(top, s[i]);
  }
  if (__any(top > c.m + RESCALE_STEP)) {
    const float next = max_of_column(top);
    if (next > c.m + RESCALE_STEP) {
      const float f = __builtin_amdgcn_exp2f(c.m - next);
      c.l *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) c.acc[dt][i] *= f;
      c.m = next;
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float p = __builtin_amdgcn_exp2f(s[i] - c.m);
    if constexpr (!FULL) p = (seen >> i) & 1 ? p : 0.f;      // while a column has seen no key, its reference point is NONE too
    sum += p;
    pb[i >> 3][i & 7] = static_cast<bf16_t>(p);
  }
  c.l += sum;
}

// One block out of registers, for a wave's single column tile; more_keys and more_values ask for the next one's, each as soon as this one's
// have been used, into the same registers. FULL: every column sees every key of it, and all of them lie in pages. (Otherwise all columns
// see the same keys: what none of them sees is zeroed, and a NaN among the others is everybody's.)
template <bool FULL, typename K, typename V>
__device__ __forceinline__ void attend(const Attn8Args& a, Block& b, int t0, int lo, int L, int g, const bf16x8 (&q)[2 * KL], Column& c, K more_keys,
                                       V more_values) {
  const float kpow = power_of(b.kcode), vpow = power_of(b.vcode);
  f32x4 st[4];
#pragma unroll
  for (int tt = 0; tt < 4; ++tt) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KL; ++j) {
      const bool in = HD % 64 == 0 || 64 * j + 16 * g < HD;
      u32x4v w = b.k[tt][j];
      if (!in) w = u32x4v{0, 0, 0, 0};
      s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(w[0], w[1], kpow), q[2 * j], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(w[2], w[3], kpow), q[2 * j + 1], s, 0, 0, 0);
    }
    st[tt] = s;
  }
  more_keys();
  bf16x8 pb[2];
  softmax<FULL>(st, a.scale * LOG2E, t0 + 16 * g, b.there, c, pb);
  if constexpr (!FULL) hide_values(b, t0, lo, L, g);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      c.acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(b.v[dt][2 * h], b.v[dt][2 * h + 1], vpow), pb[h], c.acc[dt], 0, 0, 0);
  more_values();
}

// A softmax's denominator with its head's sink; a column that saw no key stays at zero.
__device__ __forceinline__ float with_sink(const Attn8Args& a, int head, float m, float l) {
  return a.sinks != nullptr && !(l <= 0.f) ? l + exp2f(fmaf(a.sinks[head], LOG2E, -m)) : l;
}
__device__ __forceinline__ float inverse(float d) { return d == 0.f ? 0.f : 1.f / d; }       // NaN stays NaN

// =====================================================================================
// Single tokens. Grid (key heads x column tiles, requests, partitions): the 4 waves of a workgroup take the 64-key blocks of a
// partition in turn and are merged through LDS. A request has as many partitions as its keys need; the workgroups of others leave at once
// and write nothing. The last partitions come first: only long requests have them. A block's keys are asked for when its predecessor's
// have been multiplied, its values when the predecessor's have been: into the same registers (two blocks in registers of their own left
// no room for the sums, 8 requests of 32,768 keys 110 us for 98).
// =====================================================================================
__device__ __forceinline__ int parts_of(const Attn8Args& a, int L) {      // of a request with L keys: 1 at least
  const int base = L > 0 ? first_seen(a, L - 1) & ~(BK - 1) : 0;
  return a.num_parts == 1 ? 1 : min(a.num_parts, max(1, (L - base + a.part_keys - 1) / a.part_keys));
}

constexpr int HEAD_LANES = HD <= 16 ? 1 : HD <= 32 ? 2 : HD <= 64 ? 4 : HD <= 128 ? 8 : 16;      // lanes of a head in norm and rotation

// FUSED: the rows are the packed products of tokens that are not in the cache yet: every workgroup norms and rotates its heads' queries, and
// the one that has a request's last partition writes the token's key and value first (nobody else reads their block of 16). A launch
// fewer, 4-6 us of a layer's 16: 28 layers, one request of 2,048 keys 1.07 -> 0.95 ms, 8 of them 1.30 -> 1.12.
template <bool FUSED>
__global__ void __launch_bounds__(256, HD <= 128 ? 2 : 1) attn8_decode_kernel(Attn8Args a, AppendArgs w) {
  extern __shared__ __align__(16) float lds[];      // [4 waves][columns][HD + 2], FUSED: behind them queries [columns][HD] in bfloat16
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int b = blockIdx.y, part = a.num_parts - 1 - blockIdx.z;
  const int L = context_of(a, b), pos = L - 1;
  if (part >= parts_of(a, L)) return;
  const int col_tiles = (a.G + 15) / 16;
  const int kvh = blockIdx.x / col_tiles, ctile = blockIdx.x - kvh * col_tiles;
  const int lo = L > 0 ? first_seen(a, pos) : 0;
  const int base = lo & ~(BK - 1);
  const int p_lo = base + part * a.part_keys, p_hi = part + 1 < a.num_parts ? min(p_lo + a.part_keys, L) : L;      // (the last one takes what the host did not know of)
  const int ncols = min(16, a.G - ctile * 16);
  const bool valid = n < ncols;
  const int head = kvh * a.G + ctile * 16 + (valid ? n : 0);
  const int32_t* __restrict__ table = a.tables + (int64_t)b * a.table_stride;
  Column c;
  c.m = NONE; c.l = 0.f;
  c.lo = lo; c.hi = valid ? pos : -1;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) c.acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  bf16_t* queries = reinterpret_cast<bf16_t*>(lds + ((4 * ncols * (HD + 2) + 3) & ~3));
  if constexpr (FUSED) {
    const int position = w.table ? min(max(pos, 0), w.table_positions - 1) : 0;      // (beyond the table only past the host's largest context)
    constexpr int HEADS = 64 / HEAD_LANES;
    for (int i = wave * HEADS + lane / HEAD_LANES; i - lane / HEAD_LANES < ncols; i += 4 * HEADS) {
      const int l = lane % HEAD_LANES;
      const bool there = 16 * l < HD;
      const bf16_t* row = w.rows + b * w.row_stride + (int64_t)(kvh * a.G + ctile * 16 + min(i, ncols - 1)) * HD + (there ? 8 * l : 0);
      Weights weights;
      Turn turn;
      load_weights(w, w.q_w, there ? 8 * l : 0, weights);
      load_turn(w, there ? 8 * l : 0, position, turn);
      float x1[8], x2[8];
      norm_rotate<HEAD_LANES>(w, w.q_w != nullptr, weights, turn, load8(row, w.wide), load8(row + HD / 2, w.wide), there, x1, x2);
      if (!there || i >= ncols) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) { queries[i * HD + 8 * l + j] = static_cast<bf16_t>(x1[j]); queries[i * HD + HD / 2 + 8 * l + j] = static_cast<bf16_t>(x2[j]); }
    }
    if (L > 0 && part == parts_of(a, L) - 1 && wave >= 2) {
      const int page = table[pos >> a.page_shift];
      if ((unsigned)page < (unsigned)a.num_pages) {
        const int slot = page << a.page_shift | (pos & ((1 << a.page_shift) - 1));
        if (wave == 2) store_keys<HEAD_LANES>(w, b, 1, kvh, lane, slot, position);
        else store_values(w, b, 1, kvh, lane, slot);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // there before anybody of the workgroup reads it
    }
    __syncthreads();
  }
  int t0 = p_lo + BK * wave;
  if (t0 < p_hi) {
    constexpr int STEP = 4 * BK;
    Block blk;
    Pages pages = find_pages(a, table, t0, lo, L, n, g);
    bf16x8 q[2 * KL];
    load_q(FUSED ? queries + (valid ? n : 0) * HD : a.q + b * a.q_stride + (int64_t)head * HD, valid, g, q);
    load_keys(a, pages, kvh, t0, lo, L, n, g, blk);
    load_values(a, pages, kvh, t0, lo, L, n, g, blk);
    while (true) {
      // the next block's table entries, looked up while this one's keys are on their way
      const bool more = t0 + STEP < p_hi;
      if (more) pages = find_pages(a, table, t0 + STEP, lo, L, n, g);
      auto more_keys = [&]() { if (more) load_keys(a, pages, kvh, t0 + STEP, lo, L, n, g, blk); };
      auto more_values = [&]() { if (more) load_values(a, pages, kvh, t0 + STEP, lo, L, n, g, blk); };
      // a block whose pages are all there and whose keys the token sees: whole-wave test
      if (t0 >= lo && t0 + BK <= p_hi && __all(blk.there)) attend<true>(a, blk, t0, lo, L, g, q, c, more_keys, more_values);
      else attend<false>(a, blk, t0, lo, L, g, q, c, more_keys, more_values);
      if (!more) break;
      t0 += STEP;
    }
  }
  const float l = sum_of_column(c.l);
  const int stride = HD + 2;
  if (valid) {
    float* mine = lds + (wave * ncols + n) * stride;
    if (g == 0) { mine[HD] = c.m; mine[HD + 1] = l; }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[16 * dt + 4 * g + i] = c.acc[dt][i];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < ncols * HD; e += 256) {
    const int col = e / HD, d = e - col * HD;
    float M = NONE, o = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, lds[(w * ncols + col) * stride + HD]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float* theirs = lds + (w * ncols + col) * stride;
      const float f = exp2f(theirs[HD] - M);
      o += f * theirs[d];
      sum += f * theirs[HD + 1];
    }
    const int hq = kvh * a.G + ctile * 16 + col;
    if (a.num_parts == 1) {
      a.out[b * a.out_stride + (int64_t)hq * HD + d] = static_cast<bf16_t>(o * inverse(with_sink(a, hq, M, sum)));
    } else {
      const int64_t row = ((int64_t)b * a.Hq + hq) * a.num_parts + part;
      a.part_o[row * HD + d] = o;
      if (d == 0) { a.part_ml[2 * row] = M; a.part_ml[2 * row + 1] = sum; }
    }
  }
}

// =====================================================================================
// Portions of prompts. A tile is 128 columns of one request and key head; each of the 4 waves of its workgroup has 32 of them, a column to
// two lanes (l and l ^ 32). The workgroup walks the keys that its columns see in blocks of 32, which half as many instructions take as
// tiles of 16 x 16, with one column's state to a lane instead of two. Row r of a tile of scores stands for the key whose bits 2 and 3 are
// exchanged: lane l then holds keys 8 h .. 8 h + 7 and 16 + 8 h .. of its column (h = l / 32), the values' operand as it is.
//   scores  v_mfma_scale_f32_32x32x64_f8f6f4 takes the cached bytes as they are and a block's power as the product's own. The query is two
//           e4m3 numbers (below), so a tile takes as long as in bfloat16 (twice the products at twice the rate), without turning keys
//           into anything, and half the bytes of keys out of LDS: 8,192 tokens, 32 heads over 8 of 128, 554 -> 518 us.
//   values  are turned into bfloat16 once, two blocks ahead, from which every wave reads its operands of v_mfma_f32_32x32x16_bf16.
// A block's bytes go to LDS by themselves (global_load_lds_dwordx4), five and six blocks ahead (bytes held in registers could be asked for one
// step ahead only, less than a trip to memory). What a wave brings of a block lies in one page under one power, so pages, powers and
// addresses are scalars, found for 32 blocks at a time, and a lane turns into bfloat16 what it has brought itself.
//   keys    [4 waves' 8 keys][16 channels][8 keys] of 16 bytes, the second 16 keys 128 bytes further on: a read of 16 bytes a lane is
//           worked off for lanes 0-3, 12-15 and 20-27 together, then for the others of 32, which so lie in 16 different groups of banks.
//   values  [8 keys][channel] of 16 bytes.
// Step k of the walk is a pipeline: beside the numbers of block k's softmax the products of block k + 1's scores, beside the products of
// its values the conversion of block k + 2's values and the reads of its keys. One barrier a step. LDS: bytes of keys of eight blocks, of
// values of four, values of three. Weights are taken under the reference point as it is, and only where their sum says that the maximum has
// risen by much once more: the maximum of every block (11 instructions a step of 80, and exponentials that wait for it) and a sum of
// single weights instead of pairs cost 6%; registers of scores that change their meaning every second step instead of being copied, 2%.
//
// Bound by the matrix cores' and the vector units' shared issue: of 930 cycles a step and wave at 8,192 tokens 512 are products (55% of the
// time; two waves to a unit) and 45% of a wave's time is issue. 478 us there are 1,150 TF/s, against 1,430 of a large bfloat16 product.
// A workgroup alone on its unit takes 0.5 us a step, two of them 0.9, so a short prompt takes what its last tile takes: 2,048 tokens (16
// heads over 8) 44 us, of which 5.5 until the first step. Two sets of 4 waves that share a tile's keys came to 41 us there and
// cost portions of few tokens 3 us; 64 columns to a wave left one wave to a unit: 657 us for 590.
// Grid (tiles x key heads, segments): surplus tiles (the grid is made for the most there can be) exit.
// =====================================================================================
typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int COLS = 128;                    // columns of a tile
constexpr int PB = 32;                       // keys of a block
constexpr int CB = (HD + 31) / 32;           // products of a tile of scores: 64 numbers of a column's query against as many of the keys
constexpr int KC = (CB + 1) / 2;             // operands of keys
constexpr int DC = (HD + 31) / 32;           // channel tiles of the values
constexpr int VBUF = 4 * DC * 32 * 16;
constexpr int PIECES = (HD + 127) / 128;     // 16-byte pieces of keys (and of values) of a block that a lane brings
constexpr int RAW = 4 * 1024 * PIECES;       // bytes of a block's keys (and of its values) as they come
constexpr int KRAW = RAW + 256;              // the second 16 keys 128 bytes further on
constexpr int AT_K = 0, AT_RAW = 8 * KRAW, AT_V = AT_RAW + 4 * RAW, AT_FLAGS = AT_V + 3 * VBUF, LDS_BYTES = AT_FLAGS + 16;
typedef int i32x8 __attribute__((ext_vector_type(8)));
static_assert(LDS_BYTES <= 160 * 1024 && (HD > 128 || 2 * LDS_BYTES <= 160 * 1024), "one workgroup to a compute unit, two up to head size 128");

// 64 x 16 bytes from base + voff (bytes, per lane) to LDS at lds_addr + 16 * lane. The write to m0 needs one wait state before an
// instruction that reads it for an LDS address. base and lds_addr are the same in every lane.
__device__ __forceinline__ void bring16(const uint8_t* base, uint32_t voff, uint32_t lds_addr) {
  const uint64_t g = reinterpret_cast<uint64_t>(base);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(g >> 32)), lo = __builtin_amdgcn_readfirstlane((uint32_t)g);
  const uint64_t from = (uint64_t)hi << 32 | lo;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(voff), "s"(from) : "memory");
}
// All but the last N requests of this wave have landed.
template <int N>
__device__ __forceinline__ void brought() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// The LDS writes of this wave done, every wave at the same point; requests to memory stay on their way.
__device__ __forceinline__ void step_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// One column over the keys [lo, hi) that it sees, without a product of zero anywhere, key by key in plain float32: what a wave does with
// its columns where a block that some of them see and others do not holds a value that is NaN. A lane scores every 64th key and has every
// 64th channel.
__device__ void one_column(const Attn8Args& a, const int32_t* table, int64_t row, int kvh, int head, int lo, int hi, int seg, int lane) {
  const int mask = (1 << a.page_shift) - 1;
  const bf16_t* q = a.q + row * a.q_stride + (int64_t)head * HD;
  float m = NONE, l = 0.f, o[(HD + 63) / 64];
#pragma unroll
  for (int j = 0; j < (HD + 63) / 64; ++j) o[j] = 0.f;
  for (int t0 = lo; t0 < hi; t0 += 64) {
    const int key = t0 + lane;
    const int page = key < hi ? table[key >> a.page_shift] : -1;
    const bool sees = (unsigned)page < (unsigned)a.num_pages;
    const int64_t at = (int64_t)(sees ? page : 0) * a.Hkv + kvh;
    const int off = sees ? key & mask : 0;
    const int64_t code = (at << (a.page_shift - 4)) + (off >> 4);
    const float kp = power_of(a.k_powers[code]), vp = power_of(a.v_powers[code]);
    float s = 0.f;
    for (int d = 0; d < HD; ++d) s = fmaf(static_cast<float>(q[d]), __builtin_amdgcn_cvt_f32_fp8((int)a.k[((at << a.page_shift) + off) * HD + d], 0) * kp, s);
    s = sees ? s * (a.scale * LOG2E) : NONE;
    const float next = fmaxf(m, wave_max(s)), f = exp2f(m - next);
    const float p = sees ? exp2f(s - next) : 0.f;
    m = next;
    l = l * f + wave_sum(p);
#pragma unroll
    for (int j = 0; j < (HD + 63) / 64; ++j) o[j] *= f;
    for (int i = 0; i < 64; ++i) {
      if (!__shfl((int)sees, i)) continue;
      const float pi = __shfl(p, i), vpi = __shfl(vp, i);
      const int64_t head_of = (int64_t)__shfl(page, i) * a.Hkv + kvh;
      const int place = (t0 + i) & mask;
#pragma unroll
      for (int j = 0; j < (HD + 63) / 64; ++j)
        if (lane + 64 * j < HD)
          o[j] = fmaf(pi, __builtin_amdgcn_cvt_f32_fp8((int)a.v[((head_of * HD + lane + 64 * j) << a.page_shift) + place], 0) * vpi, o[j]);
    }
  }
  const int64_t to = (row * a.Hq + head) * a.num_parts + seg;
  const float inv = inverse(with_sink(a, head, m, l));
#pragma unroll
  for (int j = 0; j < (HD + 63) / 64; ++j)
    if (lane + 64 * j < HD) {
      if (a.num_parts > 1) a.part_o[to * HD + lane + 64 * j] = o[j];
      else a.out[row * a.out_stride + (int64_t)head * HD + lane + 64 * j] = static_cast<bf16_t>(o[j] * inv);
    }
  if (a.num_parts > 1 && lane == 0) { a.part_ml[2 * to] = m; a.part_ml[2 * to + 1] = l; }
}

__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD <= 128 ? 2 : 1, HD <= 128 ? 2 : 1))) attn8_prompt_kernel(Attn8Args a, int tiles) {
  extern __shared__ __align__(16) char lds_bytes[];
  int* nan_flag = reinterpret_cast<int*>(lds_bytes + AT_FLAGS);      // a block that not every column sees whole holds a value that is NaN
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int kvh = blockIdx.x % a.Hkv, tile = tiles - 1 - (int)(blockIdx.x / a.Hkv), seg = blockIdx.y;
  // request b has the tiles from cu[b] * G / COLS + b on
  int b = 0, end = a.num_seqs;
  while (end - b > 1) {
    const int mid = (b + end) >> 1;
    if ((int)((int64_t)a.cu[mid] * a.G / COLS) + mid <= tile) b = mid; else end = mid;
  }
  const int q0 = a.cu[b], q_len = a.cu[b + 1] - q0;
  const int col0 = (tile - (int)((int64_t)q0 * a.G / COLS) - b) * COLS;
  const int L = context_of(a, b), start = L - q_len;
  asm volatile("" ::"s"(L));                  // (asked for together with the counts)
  if (col0 >= q_len * a.G) return;
  const int32_t* __restrict__ table = a.tables + (int64_t)b * a.table_stride;
  // the keys that the tile's columns see, and this segment's share of them
  const int last_tok = min(col0 + COLS, q_len * a.G) - 1;
  const int tile_lo = first_seen(a, max(start + col0 / a.G, 0)), tile_hi = start + last_tok / a.G + 1;
  const int seg_lo = (tile_lo & ~(BK - 1)) + seg * a.part_keys, seg_hi = seg + 1 < a.num_parts ? min(tile_hi, seg_lo + a.part_keys) : tile_hi;
  const int nblk = (seg_hi - seg_lo + PB - 1) / PB;           // (none: not above 0)
  // keys that every column of the tile sees
  const int tile_from = first_seen(a, max(start + last_tok / a.G, 0)), tile_upto = start + col0 / a.G;

  const int col = col0 + 32 * wave + n;
  const bool valid = col < q_len * a.G;
  const int tok = valid ? col / a.G : 0, head = kvh * a.G + (valid ? col - tok * a.G : 0);
  const int64_t row = q0 + tok;
  float m = NONE, l = 0.f;
  const int lo = valid ? first_seen(a, max(start + tok, 0)) : 0, hi = valid ? start + tok : -1;      // the keys that the column sees
  uint4 raw[KC][4];                           // the column's query: channels 64 j + 32 h ..: a lane's 32; of an odd last 32 a lane has 16
  {
    const bf16_t* from = a.q + row * a.q_stride + (int64_t)head * HD;
#pragma unroll
    for (int j = 0; j < KC; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (2 * j + 1 == CB && e >= 2) break;
        const int c = 64 * j + (2 * j + 1 < CB ? 32 : 16) * h + 8 * e;
        raw[j][e] = *reinterpret_cast<const uint4*>(from + (c < HD ? c : 0));
        if (!valid || c >= HD) raw[j][e] = make_uint4(0, 0, 0, 0);
      }
  }
  f32x16 acc[DC];
#pragma unroll
  for (int dt = 0; dt < DC; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;
  // the keys that every column of the wave sees: columns are in order, and who is not there sees what the others see
  const int all_lo = __builtin_amdgcn_readlane(valid ? lo : tile_from, 31), all_hi = __builtin_amdgcn_readlane(valid ? hi : 1 << 30, 0);
  bool again = false;

  if (nblk > 0) {
    const int group = wave >> 1, part = wave & 1;             // this wave brings half of a block's 16 keys `group`: 8 keys, HD / 2 channels of values
    const int page_mask = (1 << a.page_shift) - 1;
    if (threadIdx.x == 0) *nan_flag = 0;
    // What 32 blocks need is held by the wave's lanes, one for every 16 keys, and a block's read from there: where its bytes lie (page 0 where
    // no page is), behind the wave's own pieces of keys and of values, and the powers (asked for when the pages are known).
    const uint32_t page_bytes = (uint32_t)(a.Hkv * HD) << a.page_shift;
    auto ask_pages = [&](int t0) { const int key = t0 + 16 * lane; return table[group_in(key, tile_lo, L) ? key >> a.page_shift : 0]; };
    auto settle_pages = [&](int t0, int raw) { return group_in(t0 + 16 * lane, tile_lo, L) && (unsigned)raw < (unsigned)a.num_pages ? raw : -1; };
    struct Where { uint32_t k_lo, k_hi, v_lo, v_hi; };
    auto find = [&](int t0, int ids) {
      const uint64_t page = (uint64_t)(uint32_t)max(ids, 0) * page_bytes;
      const int off = (t0 + 16 * lane) & page_mask;
      const uint64_t k = page + off * HD, v = page + off;
      return Where{(uint32_t)k, (uint32_t)(k >> 32), (uint32_t)v, (uint32_t)(v >> 32)};
    };
    auto ask_codes = [&](int t0, int ids) -> uint32_t {
      const int off = (t0 + 16 * lane) & page_mask;
      const int64_t at = (((int64_t)max(ids, 0) * a.Hkv + kvh) << (a.page_shift - 4)) + (off >> 4);
      return code_of(a.k_powers[at]) | code_of(a.v_powers[at]) << 23;      // as the products take it, and the power itself
    };
    int more_pages = settle_pages(seg_lo, ask_pages(seg_lo));
    Where at = find(seg_lo, more_pages);
    uint32_t codes = ask_codes(seg_lo, more_pages), more_codes = 0;
    // bits 2 k and 2 k + 1: block k's groups lie in pages; of the last 32 blocks looked up and of the 32 before
    uint64_t held = __ballot(more_pages >= 0), held_before = 0;
    // first_steady, first_whole: the first block that the wave, that every column of the tile sees whole; steady steps begin where their own
    // block is the wave's and the one two on, whose values they convert, the tile's. clear: the first block from there on that does not wholly
    // lie in pages, as far as is known.
    const int first_steady = max(all_lo - seg_lo + PB - 1, 0) / PB, first_whole = max(tile_from - seg_lo + PB - 1, 0) / PB;
    const int begin_steady = max(first_steady, first_whole - 2);
    auto clear_upto = [&](int k0) {
      const int skip = begin_steady - k0;
      const uint64_t missing = skip >= 32 ? 0 : ~held & (~0ull << (2 * max(skip, 0)));
      return k0 + (missing ? __builtin_ctzll(missing) / 2 : 32);
    };
    int clear = clear_upto(0);
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds_bytes;
    const uint32_t mine = 16 * lane + 1024 * PIECES * wave;     // where this lane's values lie in a block's bytes
    // Block k's keys to slot k % 8, its values to slot k % 4 (beyond the last block: page 0's, which is always there). A lane's keys: row
    // lane % 8 of the wave's 8, 16 channels; its values: a channel.
    const uint8_t* k_head = a.k + (((int64_t)kvh << a.page_shift) + 8 * part) * HD;
    const uint8_t* v_head = a.v + (((int64_t)kvh * HD + part * (HD / 2)) << a.page_shift);
    const uint32_t k_lane = (lane & 7) * HD + (lane >> 3) * 16, v_lane = (uint32_t)lane << a.page_shift;
    const uint32_t my_keys = lds0 + AT_K + 1024 * PIECES * wave + 128 * group, my_values = lds0 + AT_RAW + 1024 * PIECES * wave;
    auto held_at = [&](uint32_t x, int k) { return (uint32_t)__builtin_amdgcn_readlane(x, (2 * k + group) & 63); };
    auto keys_of = [&](int k) { return (uint64_t)held_at(at.k_hi, k) << 32 | held_at(at.k_lo, k); };
    auto values_of = [&](int k) { return (uint64_t)held_at(at.v_hi, k) << 32 | held_at(at.v_lo, k); };
    auto bring_keys = [&](int k, uint64_t from) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        if (HD % 128 == 0 || lane + 64 * i < HD / 2) bring16(k_head + from + 128 * i, k_lane, my_keys + (k & 7) * KRAW + 1024 * i);
    };
    auto bring_values = [&](int k, uint64_t from) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        if (HD % 128 == 0 || lane + 64 * i < HD / 2)
          bring16(v_head + from + ((int64_t)(64 * i) << a.page_shift), v_lane, my_values + (k & 3) * RAW + 1024 * i);
    };
    u32x4v raw_v[PIECES];
    auto read_raw_values = [&](int k) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) raw_v[i] = *reinterpret_cast<const u32x4v*>(lds_bytes + AT_RAW + (k & 3) * RAW + mine + 1024 * i);
    };
    // Half j of block k's values. Keys in front of tile_lo, or from seg_hi on (up to two blocks more are turned than walked), or in no page
    // become zeros; a NaN among the others is reported: one that some column of the tile sees.
    // WHOLE: every column of the tile sees all of the block, and it lies in pages.
    auto store_values = [&](auto whole_tag, int j, int k, uint32_t code, uint32_t there, char* vbuf) {
      constexpr bool WHOLE = decltype(whole_tag)::value;
      const float power = __uint_as_float(code & 0x7f800000u);
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int p = lane + 64 * i;
        uint32_t w0 = raw_v[i][2 * j], w1 = raw_v[i][2 * j + 1];
        if constexpr (!WHOLE) {
          const int first = seg_lo + PB * k + 16 * group;
          if (!((there >> group) & 1) || first < tile_lo || first + 16 > seg_hi) {
            const int from = ((there >> group) & 1) ? tile_lo - first - 8 * j : 8, to = seg_hi - first - 8 * j;
            const uint64_t upto = to >= 8 ? ~0ull : to <= 0 ? 0ull : (1ull << (8 * to)) - 1, below = from >= 8 ? ~0ull : from <= 0 ? 0ull : (1ull << (8 * from)) - 1;
            const uint64_t keep = upto & ~below;
            w0 &= (uint32_t)keep; w1 &= (uint32_t)(keep >> 32);
          }
        }
        if (HD % 128 == 0 || p < HD / 2) {
          if constexpr (!WHOLE) {
            // all seven lower bits of a byte
            const uint32_t nan = (((w0 & 0x7f7f7f7fu) + 0x01010101u) | ((w1 & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u;
            if (__builtin_expect(nan != 0, 0)) *nan_flag = 1;
          }
          *reinterpret_cast<bf16x8*>(vbuf + ((2 * group + j) * (32 * DC) + part * (HD / 2) + p) * 16) = operand(w0, w1, power);
        }
      }
    };

    const float sc = a.scale * LOG2E;
    const uint32_t rd_v = AT_V + (32 * DC * h + n) * 16;
    // A lane's row stands for key 16 (n / 16) + 8 (n / 4 % 2) + 4 (n / 8 % 2) + n % 4; its channels are 64 j + 32 h .. + 31, of an odd last 32
    // the 16 h-th 16, twice (zeros beyond the head's)
    const uint32_t rd_k = AT_K + 1024 * PIECES * (2 * (n >> 4) + ((n >> 2) & 1)) + 128 * (n >> 4) + 16 * ((n & 3) + 4 * ((n >> 3) & 1));
    union Keys { i32x8 all; u32x4v half[2]; };
    Keys ka[KC];
    auto read_keys = [&](int k) {
#pragma unroll
      for (int j = 0; j < KC; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool odd = 2 * j + 1 == CB;
          if (odd && e) { ka[j].half[1] = ka[j].half[0]; break; }
          const int piece = 4 * j + (odd ? h : 2 * h + e), last = 4 * j + (odd ? 1 : 2 + e);      // (of the upper lanes)
          const u32x4v w = *reinterpret_cast<const u32x4v*>(lds_bytes + (k & 7) * KRAW + rd_k + 1024 * (j / 2) + 128 * (piece & 7));
          ka[j].half[e] = 16 * last < HD || 16 * piece < HD ? w : u32x4v{0, 0, 0, 0};
        }
    };
    // The column's query as two e4m3 numbers each under one power, x = (high + low / 16) 2^p with |high| <= 256: what rounding to high leaves of
    // a bfloat16 has 4 bits, so the two are exact for numbers down to 2^-13 of the largest and off by 2^-21 of the largest at most below.
    i32x8 q[CB];
    uint32_t q_powers;                          // of high, of low; in the third byte, of high in the lower lanes and of low in the upper ones
    // product i of a tile of scores: high and low of 64 channels in turn, or both of 32 (a lane's power is for 32 of the 64 numbers: those in
    // the first four registers of both halves of the lanes, or those in the last four)
    uint32_t k_powers = 0;
    auto score = [&](int i, const f32x16& c) {
      if (i / 2 * 2 + 1 >= CB) return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(ka[i / 2].all, q[i], c, 0, 0, 0, (int)k_powers, 2, (int)q_powers);
      if (i % 2 == 0) return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(ka[i / 2].all, q[i], c, 0, 0, 0, (int)k_powers, 0, (int)q_powers);
      return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(ka[i / 2].all, q[i], c, 0, 0, 0, (int)k_powers, 1, (int)q_powers);
    };
    const int power_lane = 4 * (n >> 4);
    auto powers_of_block = [&](int k) { return (uint32_t)__builtin_amdgcn_ds_bpermute(power_lane + ((8 * k) & 255), (int)codes); };      // of the lane's key
    const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    f32x16 scores, scores_next;               // of the block whose softmax comes next, of the one after

    // What the first step finds: block 0's scores, block 1's keys in registers and block 2's in LDS, the values of 0 and 1 in LDS, and on their
    // way, in this order, the keys and values of (3, 2), (4, 3), (5, 4).
    bring_keys(0, keys_of(0)); bring_keys(1, keys_of(1)); bring_values(0, values_of(0)); bring_values(1, values_of(1)); bring_keys(2, keys_of(2));
    bring_keys(3, keys_of(3)); bring_values(2, values_of(2)); bring_values(3, values_of(3));
    {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < KC; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (2 * j + 1 == CB && e >= 2) break;
#pragma unroll
          for (int i = 0; i < 4; ++i) { const uint32_t w = (&raw[j][e].x)[i]; top = max(top, max(w & 0x7fffu, (w >> 16) & 0x7fffu)); }
        }
      const auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);
      const int power = min(max((int)(max(both[0], both[1]) >> 7) - 7, 4), 247);      // the largest number between 128 and 256 of it
      const float down = __uint_as_float((uint32_t)(254 - power) << 23);
      q_powers = (uint32_t)power | (uint32_t)(power - 4) << 8 | (uint32_t)(power - (h ? 4 : 0)) << 16;
#pragma unroll
      for (int j = 0; j < KC; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {           // four channels at a time
          if (2 * j + 1 == CB && e >= 4) break;
          const uint32_t w[2] = {(&raw[j][e >> 1].x)[2 * (e & 1)], (&raw[j][e >> 1].x)[2 * (e & 1) + 1]};
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16) * down;
          int high = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
          high = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], high, true);
          float r[4];
          r[0] = (x[0] - __builtin_amdgcn_cvt_f32_fp8(high, 0)) * 16.f; r[1] = (x[1] - __builtin_amdgcn_cvt_f32_fp8(high, 1)) * 16.f;
          r[2] = (x[2] - __builtin_amdgcn_cvt_f32_fp8(high, 2)) * 16.f; r[3] = (x[3] - __builtin_amdgcn_cvt_f32_fp8(high, 3)) * 16.f;
          int low = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
          low = __builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], low, true);
          if (2 * j + 1 < CB) { q[2 * j][e] = high; q[(2 * j + 1) % CB][e] = low; }
          else { q[2 * j][e] = high; q[2 * j][(4 + e) & 7] = low; }
        }
    }
    step_barrier();                           // (the flag)
    brought<3 * PIECES>();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      read_raw_values(k);
#pragma unroll
      for (int j = 0; j < 2; ++j) store_values(std::false_type{}, j, k, held_at(codes, k), (uint32_t)(held >> (2 * k)), lds_bytes + AT_V + k * VBUF);
    }
    step_barrier();
    bring_keys(4, keys_of(4)); bring_keys(5, keys_of(5)); bring_values(4, values_of(4));
    read_keys(0);
    k_powers = powers_of_block(0);
#pragma unroll
    for (int i = 0; i < CB; ++i) scores = score(i, i ? scores : zero);
    read_keys(1);
    k_powers = powers_of_block(1);
    uint64_t values_at = values_of(5);        // of the block whose values are asked for next

    uint32_t cur = 0, nxt = VBUF, to = 2 * VBUF;        // the values of blocks k, k + 1, k + 2
    auto there_of = [&](int b, int k) { return (uint32_t)(((b >> 5) == ((k + 5) >> 5) ? held : held_before) >> ((2 * b) & 63)) & 3u; };      // block b's groups, in step k
    // STEADY: every column of the wave sees every key of block k, every one of the tile those of block k + 2, and both lie in pages; such a
    // step has no branch but for a maximum that rises and for what is held for the next 32 blocks.
    auto step = [&](auto steady_tag, int k, const f32x16& st, f32x16& sn) {
      constexpr bool STEADY = decltype(steady_tag)::value, FULL = STEADY;
      const int t0 = seg_lo + PB * k;
      brought<4 * PIECES>();                  // keys of block k + 3, values of k + 2; the two steps' after them are still on their way
      read_raw_values(k + 2);
      const uint32_t code_v = held_at(codes, k + 2), next_powers = powers_of_block(k + 2);
      bf16x8 va[2 * DC];                      // keys 16 j + 8 h .. of channel tile dt: DC j + dt
      auto read_values = [&](int from, int upto) {
#pragma unroll
        for (int i = 0; i < 2 * DC; ++i)
          if (i >= from && i < upto) va[i] = *reinterpret_cast<const bf16x8*>(lds_bytes + cur + rd_v + 512 * (i % DC) + 2 * 512 * DC * (i / DC));
      };
      // the lane's 16 keys: 8 h + i, and 16 + 8 h + i - 8 from i = 8 on
      uint32_t seen = 0;
      if constexpr (!FULL) {
        const int from = max(lo - t0, 0), upto = min(hi - t0, 31);
        const uint32_t range = upto >= from && from < 32 ? (uint32_t)((2ull << upto) - (1ull << from)) : 0u;
        const uint32_t there = there_of(k, k);
        seen = (range & ((there & 1 ? 0xffffu : 0u) | (there & 2 ? 0xffff0000u : 0u))) >> (8 * h);
      }
      auto sees = [&](int i) { return (seen >> (i < 8 ? i : i + 8)) & 1; };
      bf16x8 pb[2];
      auto weigh = [&](int i) {               // (while a column has seen no key, its reference point is NONE: infinite)
        const float p = __builtin_amdgcn_exp2f(fmaf(st[i], sc, -m));
        return FULL || sees(i) ? p : 0.f;
      };
      auto sum_up = [&]() {                   // of the weights as they are rounded
        float s[2] = {0.f, 0.f};
        const bf16x2 ones = {static_cast<bf16_t>(1.f), static_cast<bf16_t>(1.f)};
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i & 1] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{pb[i >> 2][2 * (i & 3)], pb[i >> 2][2 * (i & 3) + 1]}, ones, s[i & 1], false);
        return s[0] + s[1];
      };
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        // the values' operands take the registers of the keys' that have been used
        if (i == 8) { __builtin_amdgcn_sched_barrier(0); read_values(0, DC); }
        if (i == 12) { __builtin_amdgcn_sched_barrier(0); read_values(DC, 2 * DC); }
#pragma unroll
        for (int j = 0; j < CB; ++j)
          if (i == 16 * j / CB) {
            sn = score(j, j ? sn : zero);
            // (beyond 128 channels every product's sums would be moved between registers for it: 300 tokens over 2,800 keys 111 us for 85)
            if constexpr (HD <= 128) asm volatile("" : "+v"(sn));
            __builtin_amdgcn_sched_barrier(0);
          }
        pb[i >> 3][i & 7] = static_cast<bf16_t>(weigh(i));
      }
      asm volatile("" : "+v"(sn));            // (wanted in the next step only: the products would be moved behind everything that follows)
      float sum = sum_up();
      // The reference point is raised only when a weight got large, and the block's weights are taken again.
      if (__builtin_expect(__any(sum > MOST_WEIGHT), 0)) {
        float top = NONE;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, FULL || sees(i) ? st[i] * sc : NONE);
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        const float next = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
        // (a branch of the lanes, not of the wave: the sums are scaled in the registers that they are in)
        if (next > m) {
          const float f = __builtin_amdgcn_exp2f(m - next);
          l *= f;
#pragma unroll
          for (int dt = 0; dt < DC; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] *= f;
          m = next;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) pb[i >> 3][i & 7] = static_cast<bf16_t>(weigh(i));
        sum = sum_up();
      }
      __builtin_amdgcn_sched_barrier(0);
      l += sum;
      char* vbuf = lds_bytes + AT_V + to;
#pragma unroll
      for (int i = 0; i < 2 * DC; ++i) {
        if (i == DC) { __builtin_amdgcn_sched_barrier(0); read_keys(k + 2); }      // where half of the values' have been used
        acc[i % DC] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[i], pb[i / DC], acc[i % DC], 0, 0, 0);
        if constexpr (STEADY) {
#pragma unroll
          for (int j = i / DC; j < (i + 1) / DC; ++j) store_values(std::true_type{}, j, k + 2, code_v, 3, vbuf);
        }
      }
      if constexpr (!STEADY) {
#pragma unroll
        for (int j = 0; j < 2; ++j) store_values(std::false_type{}, j, k + 2, code_v, there_of(k + 2, k), vbuf);
      }
      // (what is held for 32 blocks is stored whether it has changed or not: a store in each branch would put it into scratch memory)
      const int next = k + 6;
      Where now = at;
      int later = more_pages;
      uint32_t now_codes = codes, later_codes = more_codes;
      if (__builtin_expect(((next + 1) & 31) < 5, 0)) {
        asm volatile("" ::: "memory");
        const int t_next = seg_lo + PB * next;
        if ((next & 31) == 31) later = ask_pages(t_next + PB);
        if ((next & 31) == 0) {
          later = settle_pages(t_next, later);
          now = find(t_next, later); later_codes = ask_codes(t_next, later);
          held_before = held; held = __ballot(later >= 0);
          if (clear == next) clear = clear_upto(next);
        }
        if ((next & 31) == 3) now_codes = later_codes;      // the next step looks up block k + 3's, the first of its 32
      }
      at = now; more_pages = later; codes = now_codes; more_codes = later_codes;
      bring_keys(next, keys_of(next));
      bring_values(next - 1, values_at);
      values_at = values_of(next); k_powers = next_powers;
      const uint32_t free = cur;
      cur = nxt; nxt = to; to = free;
      step_barrier();
    };
    // Blocks are walked in ascending order: in front of the window's first whole block, those that the wave sees whole (steady as long as every
    // group has its page), the rest. Loops of their own: where the ways through a step meet, the sums would change their registers.
    const int end_steady = __builtin_amdgcn_readfirstlane(all_hi >= seg_lo && tile_upto >= seg_lo ? min(min((all_hi + 1 - seg_lo) / PB, (tile_upto + 1 - seg_lo) / PB - 2), nblk) : 0);
    int k = 0;
    for (; k < min(begin_steady, nblk); ++k) { step(std::false_type{}, k, scores, scores_next); scores = scores_next; }
    for (; k + 1 < min(end_steady, clear - 2); k += 2) { step(std::true_type{}, k, scores, scores_next); step(std::true_type{}, k + 1, scores_next, scores); }
    for (; k < nblk; ++k) { step(std::false_type{}, k, scores, scores_next); scores = scores_next; }
    brought<0>();                             // (what was asked for beyond the last block lands before the LDS is another workgroup's)
    again = *nan_flag != 0;
  }
  if (__builtin_expect(again, 0)) {
    // (zero times NaN: what such a block has added is of no use to the columns that do not see it)
    for (int i = 0; i < 32; ++i) {
      const int c = col0 + 32 * wave + i;
      if (c >= q_len * a.G) break;
      const int t = c / a.G;
      one_column(a, table, q0 + t, kvh, kvh * a.G + c - t * a.G, max(seg_lo, first_seen(a, max(start + t, 0))), min(seg_hi, start + t + 1), seg, lane);
    }
    return;
  }
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
  l = __uint_as_float(both[0]) + __uint_as_float(both[1]);
  if (!valid) return;
  // the lane's channels: 32 dt + 8 i + 4 h .. + 3
  if (a.num_parts > 1) {
    const int64_t at = (row * a.Hq + head) * a.num_parts + seg;
#pragma unroll
    for (int dt = 0; dt < DC; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (32 * dt + 8 * i < HD)
          *reinterpret_cast<f32x4*>(a.part_o + at * HD + 32 * dt + 8 * i + 4 * h) = f32x4{acc[dt][4 * i], acc[dt][4 * i + 1], acc[dt][4 * i + 2], acc[dt][4 * i + 3]};
    if (h == 0) { a.part_ml[2 * at] = m; a.part_ml[2 * at + 1] = l; }
    return;
  }
  const float inv = inverse(with_sink(a, head, m, l));
  bf16_t* o = a.out + row * a.out_stride + (int64_t)head * HD + 4 * h;
#pragma unroll
  for (int dt = 0; dt < DC; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (32 * dt + 8 * i < HD) {
        bf16x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = static_cast<bf16_t>(acc[dt][4 * i + e] * inv);
        *reinterpret_cast<bf16x4*>(o + 32 * dt + 8 * i) = r;
      }
}

// Joins the partitions of a (row, head): out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p. A wave to a (row, head): a lane weighs a
// partition, then all of them sum the channels, eight partitions asked for at a time, the first eight before anything else is known.
// DECODE: row t is request t, which may have fewer partitions than there is room for; what lies behind them is read and not used.
template <bool DECODE>
__global__ void __launch_bounds__(256) attn8_join_kernel(Attn8Args a, int64_t rows) {
  const int lane = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= rows * a.Hq) return;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + at * a.num_parts;
  const float* po = a.part_o + at * a.num_parts * HD;
  constexpr int CH = (HD + 63) / 64;
  float v[8][CH];
  auto ask = [&](int p) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        const int d = lane + 64 * j;
        v[e][j] = po[(int64_t)min(p + e, a.num_parts - 1) * HD + (HD % 64 == 0 || d < HD ? d : 0)];
      }
  };
  ask(0);
  const float2 none = make_float2(NONE, 0.f);
  float2 mine = lane < a.num_parts ? ml[lane] : none;
  const int64_t t = at / a.Hq;
  const int head = (int)(at - t * a.Hq);
  const int parts = DECODE ? parts_of(a, context_of(a, (int)t)) : a.num_parts;
  if (lane >= parts) mine = none;
  float M = mine.x;
  for (int p = lane + 64; p < parts; p += 64) M = fmaxf(M, ml[p].x);
  M = wave_max(M);
  float sum = 0.f, o[CH];
#pragma unroll
  for (int j = 0; j < CH; ++j) o[j] = 0.f;
  for (int p0 = 0; p0 < parts; p0 += 64) {
    if (p0 > 0) mine = p0 + lane < parts ? ml[p0 + lane] : none;
    const float f = mine.y == 0.f ? 0.f : exp2f(mine.x - M);      // (no key: nothing, whatever the maxima)
    sum += wave_sum(f * mine.y);
    const int upto = min(64, parts - p0);
    for (int i = 0; i < upto; i += 8) {
      if (p0 + i > 0) ask(p0 + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float fe = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), i + e));
#pragma unroll
        for (int j = 0; j < CH; ++j) o[j] = i + e < upto ? fmaf(fe, v[e][j], o[j]) : o[j];
      }
    }
  }
  const float inv = inverse(with_sink(a, head, M, sum));
#pragma unroll
  for (int j = 0; j < CH; ++j)
    if (lane + 64 * j < HD) a.out[t * a.out_stride + (int64_t)head * HD + lane + 64 * j] = static_cast<bf16_t>(o[j] * inv);
}

// =====================================================================================
// Host side
// =====================================================================================
#include "errors.inc"

extern "C" int me_attn8_head_dim() { return HD; }

static int fill(Attn8Args& a, const void* q, int64_t q_stride, void* out, int64_t out_stride, const void* k, const void* v,
                const void* k_powers, const void* v_powers, int64_t num_pages, const int32_t* tables, int table_stride, int table_cols,
                const int32_t* contexts, int num_seqs, int Hq, int Hkv, int page, float scale, int window, int chunk, int part_keys,
                int num_parts, float* scratch, int64_t rows, const float* sinks) {
  ME_CHECK(Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0, "attention_e4m3: %d query heads are not a multiple of %d key heads", Hq, Hkv);
  ME_CHECK(page >= E4_BLOCK && (page & (page - 1)) == 0, "attention_e4m3: page size %d must be a power of two, 16 or more", page);
  ME_CHECK((int64_t)Hkv * page * HD < (1ll << 31), "attention_e4m3: a page of %d tokens and %d heads is beyond 2^31 bytes", page, Hkv);
  ME_CHECK(num_pages >= 1 && num_pages * page < (1ll << 31), "attention_e4m3: %lld pages of %d tokens are more places than a slot can name", (long long)num_pages, page);
  ME_CHECK(q_stride % 8 == 0 && out_stride % 4 == 0, "attention_e4m3: token strides must keep 16-byte alignment");
  ME_CHECK(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0 &&
               reinterpret_cast<uintptr_t>(v) % 16 == 0, "attention_e4m3: q, out and cache pointers must be 16-byte aligned");
  ME_CHECK(table_cols >= 1 && table_stride >= table_cols && num_seqs >= 1, "attention_e4m3: bad block tables");
  ME_CHECK(scale > 0.f, "attention_e4m3: the score scale must be positive");
  ME_CHECK(window >= 0 && chunk >= 0 && !(window && chunk), "attention_e4m3: a window and a block mask exclude each other");
  ME_CHECK(num_parts >= 1 && num_parts <= 65535 && (num_parts == 1 || (scratch != nullptr && part_keys >= BK && part_keys % BK == 0)), "attention_e4m3: bad partitions");
  a = Attn8Args{};
  a.q = (const bf16_t*)q; a.q_stride = q_stride; a.out = (bf16_t*)out; a.out_stride = out_stride;
  a.k = (const uint8_t*)k; a.v = (const uint8_t*)v; a.k_powers = (const uint8_t*)k_powers; a.v_powers = (const uint8_t*)v_powers;
  a.num_pages = (int)num_pages; a.tables = tables; a.table_stride = table_stride; a.table_cols = table_cols; a.contexts = contexts;
  a.num_seqs = num_seqs; a.Hq = Hq; a.Hkv = Hkv; a.G = Hq / Hkv; a.page_shift = __builtin_ctz(page); a.scale = scale;
  a.window = window; a.chunk = chunk; a.part_keys = num_parts > 1 ? part_keys : 0; a.num_parts = num_parts; a.sinks = sinks; a.rows = rows;
  a.part_o = scratch;
  a.part_ml = scratch ? scratch + rows * Hq * num_parts * HD : nullptr;
  return 0;
}

template <bool DECODE>
static int join(const Attn8Args& a, int64_t rows, hipStream_t stream) {
  if (a.num_parts == 1) return 0;
  attn8_join_kernel<DECODE><<<(unsigned)((rows * a.Hq + 3) / 4), 256, 0, stream>>>(a, rows);
  ME_LAUNCH_CHECK();
  return 0;
}

template <bool FUSED>
static int launch_decode(const Attn8Args& a, const AppendArgs& w, hipStream_t stream) {
  ME_CHECK(a.num_seqs <= 65535, "attention_e4m3: at most 65535 single tokens in a launch");
  const int cols = a.G < 16 ? a.G : 16;
  const size_t lds = (size_t)(4 * cols * (HD + 2) + 3) / 4 * 16 + (FUSED ? (size_t)cols * HD * 2 : 0);
  if (lds > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute((const void*)attn8_decode_kernel<FUSED>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    ME_CHECK(e == hipSuccess, "attention_e4m3: %zu bytes of shared memory: %s", lds, hipGetErrorString(e));
  }
  dim3 grid(a.Hkv * ((a.G + 15) / 16), a.num_seqs, a.num_parts);
  attn8_decode_kernel<FUSED><<<grid, 256, lds, stream>>>(a, w);
  ME_LAUNCH_CHECK();
  return join<true>(a, a.num_seqs, stream);
}

// q, out: the requests' rows. scratch: [rows, Hq, num_parts, HD + 2] floats, or null for one partition.
extern "C" int me_attn8_decode(const void* q, int64_t q_stride, void* out, int64_t out_stride, const void* k, const void* v,
                               const void* k_powers, const void* v_powers, int64_t num_pages, const int32_t* tables, int table_stride,
                               int table_cols, const int32_t* contexts, int num_seqs, int Hq, int Hkv, int page, float scale, int window,
                               int chunk, int part_keys, int num_parts, float* scratch, const float* sinks, hipStream_t stream) {
  Attn8Args a;
  if (int rc = fill(a, q, q_stride, out, out_stride, k, v, k_powers, v_powers, num_pages, tables, table_stride, table_cols, contexts,
                    num_seqs, Hq, Hkv, page, scale, window, chunk, part_keys, num_parts, scratch, num_seqs, sinks)) return rc;
  return launch_decode<false>(a, AppendArgs{}, stream);
}

// The same over rows [num_seqs, (Hq + 2 Hkv) HD] (values_are_keys: Hq + Hkv) of tokens at positions contexts[r] - 1, whose keys and values are
// written first. At most 16 query heads to a key head: one workgroup has all of a partition's columns.
extern "C" int me_attn8_decode_fused(const void* rows, int64_t row_stride, void* out, int64_t out_stride, const float* q_w, const float* k_w,
                                     float eps, const float* table, int64_t table_positions, void* k, void* v, void* k_powers,
                                     void* v_powers, int64_t num_pages, const int32_t* tables, int table_stride, int table_cols,
                                     const int32_t* contexts, int num_seqs, int Hq, int Hkv, int page, float scale, int window, int chunk,
                                     int part_keys, int num_parts, float* scratch, const float* sinks, int values_are_keys, hipStream_t stream) {
  Attn8Args a;
  if (int rc = fill(a, rows, row_stride, out, out_stride, k, v, k_powers, v_powers, num_pages, tables, table_stride, table_cols, contexts,
                    num_seqs, Hq, Hkv, page, scale, window, chunk, part_keys, num_parts, scratch, num_seqs, sinks)) return rc;
  ME_CHECK(a.G <= 16, "attention_e4m3: one launch for a token's write and attention takes up to 16 query heads to a key head, not %d", a.G);
  ME_CHECK((q_w == nullptr) == (k_w == nullptr), "attention_e4m3: give both norm weights or neither");
  ME_CHECK(table == nullptr || (table_positions >= 1 && table_positions < (1ll << 31)), "attention_e4m3: empty rotation table");
  AppendArgs w{};
  w.rows = (const bf16_t*)rows; w.row_stride = row_stride; w.q_w = q_w; w.k_w = k_w; w.eps = eps; w.table = table;
  w.table_positions = (int)table_positions; w.k = (uint8_t*)k; w.v = (uint8_t*)v; w.k_powers = (uint8_t*)k_powers; w.v_powers = (uint8_t*)v_powers;
  w.Hq = Hq; w.Hkv = Hkv; w.D = HD; w.page = page; w.page_shift = a.page_shift; w.v_head = values_are_keys ? Hq : Hq + Hkv; w.T = num_seqs;
  w.wide = reinterpret_cast<uintptr_t>(q_w) % 16 == 0 && reinterpret_cast<uintptr_t>(k_w) % 16 == 0 && reinterpret_cast<uintptr_t>(table) % 16 == 0;
  return launch_decode<true>(a, w, stream);
}

extern "C" int me_attn8_prompt(const void* q, int64_t q_stride, void* out, int64_t out_stride, const void* k, const void* v,
                               const void* k_powers, const void* v_powers, int64_t num_pages, const int32_t* tables, int table_stride,
                               int table_cols, const int32_t* contexts, const int32_t* cu, int64_t rows, int num_seqs, int Hq, int Hkv,
                               int page, float scale, int window, int chunk, int part_keys, int num_parts, float* scratch,
                               const float* sinks, hipStream_t stream) {
  Attn8Args a;
  if (int rc = fill(a, q, q_stride, out, out_stride, k, v, k_powers, v_powers, num_pages, tables, table_stride, table_cols, contexts,
                    num_seqs, Hq, Hkv, page, scale, window, chunk, part_keys, num_parts, scratch, rows, sinks)) return rc;
  a.cu = cu;
  const int64_t tiles = rows * a.G / COLS + num_seqs;
  ME_CHECK(rows >= 1 && rows * a.G < (1ll << 30) && tiles * Hkv < (1ll << 31), "attention_e4m3: too many tokens for one launch");
  if (LDS_BYTES > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute((const void*)attn8_prompt_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES);
    ME_CHECK(e == hipSuccess, "attention_e4m3: %d bytes of shared memory: %s", LDS_BYTES, hipGetErrorString(e));
  }
  attn8_prompt_kernel<<<dim3((unsigned)(tiles * Hkv), num_parts), 256, LDS_BYTES, stream>>>(a, (int)tiles);
  ME_LAUNCH_CHECK();
  return join<false>(a, rows, stream);
}
