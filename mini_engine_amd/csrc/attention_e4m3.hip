// Attention over the 8-bit paged cache (e4m3.h) on the CDNA4 matrix cores, compiled once per head size with -DME_HEAD_DIM=<D>
// (a multiple of 16 up to 256): queries and results bfloat16, keys and values e4m3 under a power of two per 16 tokens and head.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j),  over the keys j that the query sees; a sink adds exp(sink) to
//   the denominator.
//
// The stored numbers times their power are bfloat16 numbers, so they are turned into such (v_cvt_scalef32_pk_bf16_fp8: two numbers and
// the power in one instruction, exactly) and both products run on v_mfma_f32_16x16x32_bf16 without a rounding that a bfloat16 cache would not
// have. Everything is computed transposed, as S^T = K Q^T and O^T += V^T P^T, over blocks of 64 keys; a "column" is one (query
// token, query head) pair of a key head. With n = lane & 15, g = lane >> 4:
//   * the four tiles of S^T let row m of tile tt stand for key 16 (m / 4) + 4 tt + m % 4, so lane (n, g) ends with the 16 keys
//     16 g .. 16 g + 15 of column n in order: the operand of the second product, without a movement of data;
//   * a lane reads 16 bytes of keys (16 channels 64 j + 16 g ..) and of values (16 keys 16 g .. of channel 16 dt + n) at a time: two
//     products' operands each. Which channel lies in which slot of the first product is free as long as the queries follow;
//   * every lane's keys of a block lie under one power, and so do its values: one byte and a shift per lane.
// Maxima, sums and accumulators are float32 and per column.
//
// Keys that a column does not see are replaced, never multiplied by zero: scores by "none", stored values by zero bytes where no
// column sees them, and where some columns of a tile see a key whose value is NaN and others do not, only those that see it become NaN.
#include "e4m3.h"
#include <cstdlib>

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
__device__ __forceinline__ float power_of(uint32_t code) { return __uint_as_float(min(max(code, (uint32_t)(E4_LEAST + E4_BIAS)), (uint32_t)(E4_MOST + E4_BIAS)) << 23); }

// A block's keys and values as they lie in memory. Loads are unconditional: a lane whose keys are not to be read (at or past the
// context, in front of what anybody sees, in a table entry without a page) reads page 0, which is always there.
struct Pages {
  int k, v;            // table entries as loaded
};
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
__device__ __forceinline__ void load_block(const Attn8Args& a, const Pages& p, int kvh, int t0, int lo, int L, int n, int g, Block& b) {
  const int mask = (1 << a.page_shift) - 1;
  const int kk = t0 + 16 * (n >> 2), vk = t0 + 16 * g;
  const bool kok = group_in(kk, lo, L) && (unsigned)p.k < (unsigned)a.num_pages;
  b.there = group_in(vk, lo, L) && (unsigned)p.v < (unsigned)a.num_pages;
  const int64_t kh = (int64_t)(kok ? p.k : 0) * a.Hkv + kvh, vh = (int64_t)(b.there ? p.v : 0) * a.Hkv + kvh;
  const int koff = kk & mask, voff = vk & mask;
  const uint8_t* kp = a.k + ((kh << a.page_shift) + koff + (n & 3)) * HD + 16 * g;
#pragma unroll
  for (int tt = 0; tt < 4; ++tt)
#pragma unroll
    for (int j = 0; j < KL; ++j)
      b.k[tt][j] = *reinterpret_cast<const u32x4v*>(kp + tt * 4 * HD + ((HD % 64 == 0 || 64 * j + 16 * g < HD) ? 64 * j : -16 * g));
  const uint8_t* vp = a.v + ((vh * HD + n) << a.page_shift) + voff;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) b.v[dt] = *reinterpret_cast<const u32x4v*>(vp + ((int64_t)(16 * dt) << a.page_shift));
  b.kcode = a.k_powers[(kh << (a.page_shift - 4)) + (koff >> 4)];
  b.vcode = a.v_powers[(vh << (a.page_shift - 4)) + (voff >> 4)];
}

// The queries of one column, in the order of the channels that load_block gives a lane.
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

template <int CT>
struct Columns {
  bf16x8 q[CT][2 * KL];
  int lo[CT], hi[CT];            // keys [lo, hi] that the column sees (hi < lo: none)
  float m[CT], l[CT];            // reference point of the exponentials (log2 domain), this lane's share of the sum
  f32x4 acc[CT][DT];
};

// One block for all columns of a wave. FULL: every column sees every key of it, and all of them lie in pages.
template <int CT, bool FULL>
__device__ __forceinline__ void attend(const Attn8Args& a, Block& b, int t0, int lo, int L, int g, Columns<CT>& c) {
  const float kpow = power_of(b.kcode), vpow = power_of(b.vcode);
  const float sc = a.scale * LOG2E;
  f32x4 st[CT][4];
#pragma unroll
  for (int tt = 0; tt < 4; ++tt) {
    bf16x8 ka[2 * KL];
#pragma unroll
    for (int j = 0; j < KL; ++j) {
      const bool in = HD % 64 == 0 || 64 * j + 16 * g < HD;
      u32x4v w = b.k[tt][j];
      if (!in) w = u32x4v{0, 0, 0, 0};
      ka[2 * j] = operand(w[0], w[1], kpow);
      ka[2 * j + 1] = operand(w[2], w[3], kpow);
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 2 * KL; ++ks) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[ks], c.q[ct][ks], s, 0, 0, 0);
      st[ct][tt] = s;
    }
  }
  bf16x8 pb[CT][2];
  uint32_t seen[CT];             // bit i: the column sees this lane's key i
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    float s[16];
    float top = NONE;
    seen[ct] = 0xffffu;
    if constexpr (!FULL) {
      const int from = max(c.lo[ct] - (t0 + 16 * g), 0), to = min(c.hi[ct] - (t0 + 16 * g), 15);
      seen[ct] = b.there && to >= from && from < 16 ? (2u << to) - (1u << from) : 0u;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = st[ct][i >> 2][i & 3];
      if constexpr (!FULL) s[i] = (seen[ct] >> i) & 1 ? s[i] : NONE;
      top = fmaxf(top, s[i]);
    }
    if (__any(top > 0.5f * NONE && top * sc > c.m[ct] + RESCALE_STEP)) {
      top = max_of_column(top);
      const float next = top > 0.5f * NONE ? top * sc : NONE;
      if (next > c.m[ct] + RESCALE_STEP) {
        const float f = __builtin_amdgcn_exp2f(c.m[ct] - next);
        c.l[ct] *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) c.acc[ct][dt][i] *= f;
        c.m[ct] = next;
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float p = __builtin_amdgcn_exp2f(fmaf(s[i], sc, -c.m[ct]));
      if constexpr (!FULL) p = (seen[ct] >> i) & 1 ? p : 0.f;
      sum += p;
      pb[ct][i >> 3][i & 7] = static_cast<bf16_t>(p);      // the sum takes it unrounded
    }
    c.l[ct] += sum;
  }
  if constexpr (!FULL) {
    hide_values(b, t0, lo, L, g);
    uint32_t any = 0;            // a stored NaN: all seven lower bits of a byte
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int w = 0; w < 4; ++w) any |= (b.v[dt][w] & 0x7f7f7f7fu) + 0x01010101u;
    if (__any((any & 0x80808080u) != 0)) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        bf16x8 va[2], bad[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          va[h] = operand(b.v[dt][2 * h], b.v[dt][2 * h + 1], vpow);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool is = ((b.v[dt][2 * h + (e >> 2)] >> (8 * (e & 3))) & 0x7f) == 0x7f;
            bad[h][e] = static_cast<bf16_t>(is ? 1.f : 0.f);
            va[h][e] = is ? static_cast<bf16_t>(0.f) : va[h][e];
          }
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          f32x4 count = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            bf16x8 sees;
#pragma unroll
            for (int e = 0; e < 8; ++e) sees[e] = static_cast<bf16_t>((seen[ct] >> (8 * h + e)) & 1 ? 1.f : 0.f);
            count = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bad[h], sees, count, 0, 0, 0);
            c.acc[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[h], pb[ct][h], c.acc[ct][dt], 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) c.acc[ct][dt][i] = count[i] > 0.f ? __uint_as_float(0x7fc00000u) : c.acc[ct][dt][i];
        }
      }
      return;
    }
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bf16x8 va = operand(b.v[dt][2 * h], b.v[dt][2 * h + 1], vpow);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) c.acc[ct][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pb[ct][h], c.acc[ct][dt], 0, 0, 0);
    }
  }
}

// A softmax's denominator with its head's sink; a column that saw no key stays at zero.
__device__ __forceinline__ float with_sink(const Attn8Args& a, int head, float m, float l) {
  return a.sinks != nullptr && !(l <= 0.f) ? l + exp2f(fmaf(a.sinks[head], LOG2E, -m)) : l;
}
__device__ __forceinline__ float inverse(float d) { return d == 0.f ? 0.f : 1.f / d; }       // NaN stays NaN

// =====================================================================================
// Single tokens. Grid (key heads x column tiles, requests, partitions): the 4 waves of a workgroup take the 64-key blocks of a
// partition in turn and are merged through LDS.
// =====================================================================================
__global__ void __launch_bounds__(256) attn8_decode_kernel(Attn8Args a) {
  extern __shared__ float lds[];      // [4 waves][columns][HD + 2]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int b = blockIdx.y, part = blockIdx.z;
  const int col_tiles = (a.G + 15) / 16;
  const int kvh = blockIdx.x / col_tiles, ctile = blockIdx.x - kvh * col_tiles;
  const int L = context_of(a, b), pos = L - 1;
  const int lo = L > 0 ? first_seen(a, pos) : 0;
  const int base = lo & ~(BK - 1);
  const int p_lo = base + part * a.part_keys, p_hi = part + 1 < a.num_parts ? min(p_lo + a.part_keys, L) : L;      // (the last one takes what the host did not know of)
  const int ncols = min(16, a.G - ctile * 16);
  const bool valid = n < ncols;
  const int head = kvh * a.G + ctile * 16 + (valid ? n : 0);
  const int32_t* table = a.tables + (int64_t)b * a.table_stride;
  Columns<1> c;
  c.m[0] = NONE; c.l[0] = 0.f;
  c.lo[0] = lo; c.hi[0] = valid ? pos : -1;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) c.acc[0][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  int t0 = p_lo + BK * wave;
  if (t0 < p_hi) {
    load_q(a.q + b * a.q_stride + (int64_t)head * HD, valid, g, c.q[0]);
    Block blk;
    load_block(a, find_pages(a, table, t0, lo, L, n, g), kvh, t0, lo, L, n, g, blk);
    while (true) {
      // a block whose pages are all there and whose keys the token sees: whole-wave test
      const bool full = t0 >= lo && t0 + BK <= p_hi && __all(blk.there);
      if (full) attend<1, true>(a, blk, t0, lo, L, g, c);
      else attend<1, false>(a, blk, t0, lo, L, g, c);
      t0 += 4 * BK;
      if (t0 >= p_hi) break;
      load_block(a, find_pages(a, table, t0, lo, L, n, g), kvh, t0, lo, L, n, g, blk);
    }
  }
  const float l = sum_of_column(c.l[0]);
  const int stride = HD + 2;
  if (valid) {
    float* mine = lds + (wave * ncols + n) * stride;
    if (g == 0) { mine[HD] = c.m[0]; mine[HD + 1] = l; }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[16 * dt + 4 * g + i] = c.acc[0][dt][i];
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
// Portions of prompts. A tile is 64 CT columns of one request and key head; each of the 4 waves of its workgroup has 16 CT of
// them and walks the keys that they see. Grid (tiles x key heads, segments): surplus tiles (the grid is made for the most there can be) exit.
// =====================================================================================
template <int CT>
__global__ void __launch_bounds__(256) attn8_prompt_kernel(Attn8Args a, int tiles) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x % a.Hkv, tile = tiles - 1 - (int)(blockIdx.x / a.Hkv), seg = blockIdx.y;
  constexpr int COLS = 64 * CT;
  // request b has the tiles from cu[b] * G / COLS + b on
  int b = 0, end = a.num_seqs;
  while (end - b > 1) {
    const int mid = (b + end) >> 1;
    if ((int)((int64_t)a.cu[mid] * a.G / COLS) + mid <= tile) b = mid; else end = mid;
  }
  const int q0 = a.cu[b], q_len = a.cu[b + 1] - q0;
  const int col0 = (tile - (int)((int64_t)q0 * a.G / COLS) - b) * COLS;
  if (col0 >= q_len * a.G) return;
  const int L = context_of(a, b), start = L - q_len;
  const int32_t* table = a.tables + (int64_t)b * a.table_stride;
  // the keys that the tile's columns see, and this segment's share of them
  const int last_tok = min(col0 + COLS, q_len * a.G) - 1;
  const int tile_lo = first_seen(a, max(start + col0 / a.G, 0)), tile_hi = start + last_tok / a.G + 1;
  const int base = tile_lo & ~(BK - 1);
  const int seg_lo = base + seg * a.part_keys, seg_hi = seg + 1 < a.num_parts ? min(tile_hi, seg_lo + a.part_keys) : tile_hi;
  Columns<CT> c;
  int64_t row[CT];
  int head[CT];
  bool valid[CT];
  int wave_lo = 0x7fffffff, wave_hi = 0, all_lo = 0, all_hi = 0x7fffffff;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = col0 + (wave * CT + ct) * 16 + n;
    valid[ct] = col < q_len * a.G;
    const int tok = valid[ct] ? col / a.G : 0;
    head[ct] = kvh * a.G + (valid[ct] ? col - tok * a.G : 0);
    row[ct] = q0 + tok;
    c.m[ct] = NONE; c.l[ct] = 0.f;
    c.hi[ct] = valid[ct] ? start + tok : -1;
    c.lo[ct] = valid[ct] ? first_seen(a, max(start + tok, 0)) : 0;
    load_q(a.q + row[ct] * a.q_stride + (int64_t)head[ct] * HD, valid[ct], g, c.q[ct]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) c.acc[ct][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (valid[ct]) {
      wave_lo = min(wave_lo, c.lo[ct]); wave_hi = max(wave_hi, c.hi[ct] + 1);
      all_lo = max(all_lo, c.lo[ct]); all_hi = min(all_hi, c.hi[ct]);
    }
  }
  for (int off = 8; off > 0; off >>= 1) {
    wave_lo = min(wave_lo, __shfl_xor(wave_lo, off)); wave_hi = max(wave_hi, __shfl_xor(wave_hi, off));
    all_lo = max(all_lo, __shfl_xor(all_lo, off)); all_hi = min(all_hi, __shfl_xor(all_hi, off));
  }
  const bool whole = __all(valid[0] && valid[CT - 1]);
  int t0 = max(seg_lo, wave_lo & ~(BK - 1));
  const int upto = min(seg_hi, wave_hi);
  if (t0 < upto) {
    Block blk;
    for (; t0 < upto; t0 += BK) {
      load_block(a, find_pages(a, table, t0, tile_lo, L, n, g), kvh, t0, tile_lo, L, n, g, blk);
      const bool full = whole && t0 >= all_lo && t0 + BK - 1 <= all_hi && __all(blk.there);
      if (full) attend<CT, true>(a, blk, t0, tile_lo, L, g, c);
      else attend<CT, false>(a, blk, t0, tile_lo, L, g, c);
    }
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const float l = sum_of_column(c.l[ct]);
    if (!valid[ct]) continue;
    if (a.num_parts > 1) {
      const int64_t at = (row[ct] * a.Hq + head[ct]) * a.num_parts + seg;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(a.part_o + at * HD + 16 * dt + 4 * g) = c.acc[ct][dt];
      if (g == 0) { a.part_ml[2 * at] = c.m[ct]; a.part_ml[2 * at + 1] = l; }
      continue;
    }
    const float inv = inverse(with_sink(a, head[ct], c.m[ct], l));
    bf16_t* o = a.out + row[ct] * a.out_stride + (int64_t)head[ct] * HD + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      bf16x4 r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = static_cast<bf16_t>(c.acc[ct][dt][i] * inv);
      *reinterpret_cast<bf16x4*>(o + 16 * dt) = r;
    }
  }
}

// Joins the partitions of a (row, head): out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p. A wave to a (row, head); partitions
// without a key (l = 0) are not read.
__global__ void __launch_bounds__(256) attn8_join_kernel(Attn8Args a, int64_t rows) {
  const int lane = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= rows * a.Hq) return;
  const int64_t t = at / a.Hq;
  const int head = (int)(at - t * a.Hq);
  const float* ml = a.part_ml + 2 * at * a.num_parts;
  const float* po = a.part_o + at * a.num_parts * HD;
  float M = NONE;
  for (int p = lane; p < a.num_parts; p += 64) M = fmaxf(M, ml[2 * p]);
  M = wave_max(M);
  float sum = 0.f, o[(HD + 63) / 64];
#pragma unroll
  for (int j = 0; j < (HD + 63) / 64; ++j) o[j] = 0.f;
  for (int p = 0; p < a.num_parts; ++p) {
    const float l = ml[2 * p + 1];
    if (l == 0.f) continue;
    const float f = exp2f(ml[2 * p] - M);
    sum += f * l;
#pragma unroll
    for (int j = 0; j < (HD + 63) / 64; ++j)
      if (lane + 64 * j < HD) o[j] += f * po[(int64_t)p * HD + lane + 64 * j];
  }
  const float inv = inverse(with_sink(a, head, M, sum));
#pragma unroll
  for (int j = 0; j < (HD + 63) / 64; ++j)
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

static int join(const Attn8Args& a, int64_t rows, hipStream_t stream) {
  if (a.num_parts == 1) return 0;
  attn8_join_kernel<<<(unsigned)((rows * a.Hq + 3) / 4), 256, 0, stream>>>(a, rows);
  ME_LAUNCH_CHECK();
  return 0;
}

// q, out: the requests' rows. scratch: [rows, Hq, num_parts, HD + 2] floats, or null for one partition.
extern "C" int me_attn8_decode(const void* q, int64_t q_stride, void* out, int64_t out_stride, const void* k, const void* v,
                               const void* k_powers, const void* v_powers, int64_t num_pages, const int32_t* tables, int table_stride,
                               int table_cols, const int32_t* contexts, int num_seqs, int Hq, int Hkv, int page, float scale, int window,
                               int chunk, int part_keys, int num_parts, float* scratch, const float* sinks, hipStream_t stream) {
  Attn8Args a;
  if (int rc = fill(a, q, q_stride, out, out_stride, k, v, k_powers, v_powers, num_pages, tables, table_stride, table_cols, contexts,
                    num_seqs, Hq, Hkv, page, scale, window, chunk, part_keys, num_parts, scratch, num_seqs, sinks)) return rc;
  ME_CHECK(num_seqs <= 65535, "attention_e4m3: at most 65535 single tokens in a launch");
  const size_t lds = (size_t)4 * (a.G < 16 ? a.G : 16) * (HD + 2) * sizeof(float);
  if (lds > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute((const void*)attn8_decode_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    ME_CHECK(e == hipSuccess, "attention_e4m3: %zu bytes of shared memory: %s", lds, hipGetErrorString(e));
  }
  dim3 grid(a.Hkv * ((a.G + 15) / 16), num_seqs, num_parts);
  attn8_decode_kernel<<<grid, 256, lds, stream>>>(a);
  ME_LAUNCH_CHECK();
  return join(a, num_seqs, stream);
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
  constexpr int CT = 1;
  const int64_t tiles = rows * a.G / (64 * CT) + num_seqs;
  ME_CHECK(rows >= 1 && rows * a.G < (1ll << 30) && tiles * Hkv < (1ll << 31), "attention_e4m3: too many tokens for one launch");
  attn8_prompt_kernel<CT><<<dim3((unsigned)(tiles * Hkv), num_parts), 256, 0, stream>>>(a, (int)tiles);
  ME_LAUNCH_CHECK();
  return join(a, rows, stream);
}
