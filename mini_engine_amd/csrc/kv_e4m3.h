// Norm, rotation and the write of a block's keys and values into the 8-bit cache: what the append kernel and the single tokens' one
// launch share. kv_e4m3.hip says what is computed and why so.
#pragma once
#include "e4m3.h"

struct AppendArgs {
  const bf16_t* rows;
  int64_t row_stride;
  bf16_t* q_out;                 // [T, Hq * D]
  const float* q_w;              // [D] or both nullptr: no norm
  const float* k_w;
  float eps;
  const float* table;            // [table_positions, D / 2, 2] (cos, sin) or nullptr: no rotation
  int table_positions;
  const int32_t* positions;
  const int32_t* slots;          // below 0, or at and beyond slot_end: not stored
  int slot_end;
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_powers;
  uint8_t* v_powers;
  int Hq, Hkv, D, page, page_shift;
  int v_head;                    // a row's first value head
  int64_t T;
  int window, first_window;      // rows whose runs the waves of keys and values of kv_groups workgroups walk: of the first first_rows and of the others
  int first_rows;                // (a multiple of first_window)
  int kv_groups;
  int q_parts;                   // waves of queries to a row
  int64_t kv_grid;               // workgroups of keys and values in front of those of the queries
  int wide;                      // rows, weights and angles are read 16 bytes at a time
};

// Eight neighbouring numbers of a row.
__device__ __forceinline__ bf16x8 load8(const bf16_t* p, bool wide) {
  bf16x8 t;
  if (wide) {
    t = *reinterpret_cast<const bf16x8*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = p[i];
  }
  return t;
}
__device__ __forceinline__ void load8(const float* p, bool wide, float (&v)[8]) {
  if (wide) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[i];
  }
}

// A lane's norm weights and (cos, sin): its eight pairs (at + i, D / 2 + at + i).
struct Weights { float w1[8], w2[8]; };
struct Turn { float c0[8], c1[8]; };
__device__ __forceinline__ void load_weights(const AppendArgs& a, const float* w, int at, Weights& t) {
  if (w) { load8(w + at, a.wide, t.w1); load8(w + (a.D >> 1) + at, a.wide, t.w2); }
}
__device__ __forceinline__ void load_turn(const AppendArgs& a, int at, int position, Turn& t) {
  if (a.table) {
    const float* cs = a.table + ((int64_t)position * (a.D >> 1) + at) * 2;
    load8(cs, a.wide, t.c0); load8(cs + 8, a.wide, t.c1);
  }
}
// Norm and rotation of a head that L2 lanes share; lanes that have no channels hold zeros. Which products are fused with a sum is written
// out, not left to the compiler: every kernel gives the same bits.
template <int L2>
__device__ __forceinline__ void norm_rotate(const AppendArgs& a, bool norm, const Weights& w, const Turn& t, bf16x8 raw1, bf16x8 raw2, bool there, float (&x1)[8],
                                            float (&x2)[8]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x1[i] = there ? static_cast<float>(raw1[i]) : 0.f;
    x2[i] = there ? static_cast<float>(raw2[i]) : 0.f;
  }
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x1[i], x1[i], fmaf(x2[i], x2[i], ss));
#pragma unroll
    for (int off = L2 / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off, ME_WAVE);
    const float inv = rsqrtf(ss / (float)a.D + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) { x1[i] *= inv * w.w1[i]; x2[i] *= inv * w.w2[i]; }
  }
  if (a.table) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = i < 4 ? t.c0[2 * i] : t.c1[2 * i - 8], s = i < 4 ? t.c0[2 * i + 1] : t.c1[2 * i - 7];
      const float u = x1[i], v = x2[i];
      x1[i] = fmaf(u, c, -(v * s));
      x2[i] = fmaf(v, c, u * s);
    }
  }
}

// The same exactly, as far as a rounding to 4 significant bits can see: sum and root in double, products and their sums as the rounded
// number and what it leaves (by fma, and by the sums' own errors, after Dekker and Knuth), and the result rounded to the odd neighbour
// where it is none: the rounding to come then goes as that of the exact number would.
struct Pair { float hi, lo; };
__device__ __forceinline__ Pair sum_of(float a, float b) {
#pragma clang fp contract(off)
  const float s = a + b, t = s - a;
  return Pair{s, (a - (s - t)) + (b - t)};
}
__device__ __forceinline__ float odd(Pair x) {
  const uint32_t bits = __float_as_uint(x.hi);
  const bool moves = x.lo != 0.f && !(bits & 1) && (bits << 1) - 1 < 0xfeffffffu;      // (neither zero nor infinite nor NaN)
  return __uint_as_float(moves ? ((x.lo > 0.f) == (x.hi > 0.f) ? bits + 1 : bits - 1) : bits);
}
template <int L2>
__device__ __forceinline__ void norm_rotate_key(const AppendArgs& a, bool norm, const Weights& w, const Turn& t, bf16x8 raw1, bf16x8 raw2, bool there, float (&y1)[8],
                                                float (&y2)[8]) {
#pragma clang fp contract(off)
  Pair inv = {1.f, 0.f};
  if (norm) {
    double ss = 0.;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double u = there ? static_cast<float>(raw1[i]) : 0.f, v = there ? static_cast<float>(raw2[i]) : 0.f;
      ss = fma(u, u, fma(v, v, ss));
    }
#pragma unroll
    for (int off = L2 / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off, ME_WAVE);
    const double root = rsqrt(ss / (double)a.D + (double)a.eps);
    inv.hi = (float)root;
    inv.lo = (float)(root - (double)inv.hi);
  }
  auto normed = [&](float x, float weight) {
    if (!norm) return Pair{x, 0.f};
    const float m = inv.hi * weight, y = x * m;
    return Pair{y, fmaf(x, m, -y) + x * fmaf(inv.lo, weight, fmaf(inv.hi, weight, -m))};
  };
  auto product = [](Pair x, float c) {
    const float y = x.hi * c;
    return Pair{y, fmaf(x.lo, c, fmaf(x.hi, c, -y))};
  };
  auto sum = [](Pair x, Pair y) {
    const Pair s = sum_of(x.hi, y.hi);
    return sum_of(s.hi, s.lo + (x.lo + y.lo));
  };
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const Pair u = normed(there ? static_cast<float>(raw1[i]) : 0.f, w.w1[i]), v = normed(there ? static_cast<float>(raw2[i]) : 0.f, w.w2[i]);
    if (a.table) {
      const float c = i < 4 ? t.c0[2 * i] : t.c1[2 * i - 8], s = i < 4 ? t.c0[2 * i + 1] : t.c1[2 * i - 7];
      y1[i] = odd(sum(product(u, c), product(v, -s)));
      y2[i] = odd(sum(product(v, c), product(u, s)));
    } else {
      y1[i] = odd(u);
      y2[i] = odd(v);
    }
  }
}

__device__ __forceinline__ int row_position(const AppendArgs& a, int64_t t) {
  return a.table ? min(max(a.positions[min(t, a.T - 1)], 0), a.table_positions - 1) : 0;
}
__device__ __forceinline__ int row_slot(const AppendArgs& a, int64_t t) {
  const int s = t >= 0 && t < a.T ? a.slots[t] : -1;
  return s < a.slot_end ? s : -1;
}

// Whether a number, scaled for its block, lies so near to the middle between two e4m3 numbers that float32 may have put it on the other side:
// within 8 of its steps. There it would be off by a whole step of e4m3 (one number in 650,000 was, most of them by one of the large
// steps; what cancellation leaves further off is small, and so are its steps); one in 65,000 is done again by norm_rotate_key. 64 rows
// of one token 6.4 us in float32 alone, 8.4 so; 7,900 rows of 32 and 8 heads of 128 48.5 and 49.6 (53 where the queries' waves have 132
// registers instead of 128), with every key done so 59, all in double 66.
__device__ __forceinline__ bool between(float x) { return ((__float_as_uint(x) + 0x80008u) & 0xfffffu) < 0x10u; }

// The cnt rows from r on, of one block, of one key head (at most 16, ascending slots). Lane i holds the slot and the position of row r + i
// (i < 16): everything else is asked for at once.
template <int L2>
__device__ __forceinline__ void store_keys(const AppendArgs& a, int64_t r, int cnt, int kvh, int lane, int slots, int positions) {
  constexpr int TOKENS = 64 / L2, PASSES = TOKENS >= E4_BLOCK ? 1 : E4_BLOCK / TOKENS;
  const int l = lane % L2, half = a.D >> 1;
  const bool active = l < (a.D >> 4);
  const int s0 = __builtin_amdgcn_readlane(slots, 0);
  const int64_t pg = s0 >> a.page_shift;
  const int in_page = s0 & (a.page - 1), begin = in_page & (E4_BLOCK - 1);
  uint8_t* code = a.k_powers + ((pg * a.Hkv + kvh) << (a.page_shift - 4)) + (in_page >> 4);
  const int before = begin > 0 ? min((int)*code - E4_BIAS, E4_MOST) : E4_LEAST;
  bf16x8 raw1[PASSES], raw2[PASSES];
  Turn turn[PASSES];
  Weights w;
  const int at = active ? 8 * l : 0;
  auto row_of = [&](int p) { return min(p * TOKENS + lane / L2, cnt - 1); };      // (beyond the run its last one: it changes no maximum)
  auto load = [&](int p, bf16x8& x1, bf16x8& x2, Turn& t) {
    const bf16_t* row = a.rows + (r + row_of(p)) * a.row_stride + (int64_t)(a.Hq + kvh) * a.D + at;
    x1 = load8(row, a.wide); x2 = load8(row + half, a.wide);
    load_turn(a, at, __shfl(positions, row_of(p)), t);
  };
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    if (p > 0 && p * TOKENS >= cnt) continue;      // (a single token is one pass)
    load(p, raw1[p], raw2[p], turn[p]);
  }
  load_weights(a, a.k_w, at, w);
  float x1[PASSES][8], x2[PASSES][8];
  float largest = 0.f;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    if (p > 0 && p * TOKENS >= cnt) continue;
    norm_rotate<L2>(a, a.k_w != nullptr, w, turn[p], raw1[p], raw2[p], active, x1[p], x2[p]);
#pragma unroll
    for (int j = 0; j < 8; ++j) largest = fmaxf(largest, fmaxf(e4_size(x1[p][j]), e4_size(x2[p][j])));
  }
  const int power = max(e4_power(wave_max(largest)), before);
  uint8_t* base = a.k + ((pg * a.Hkv + kvh) * (int64_t)a.page + (in_page & ~(E4_BLOCK - 1))) * a.D;
  if (begin > 0 && power > before) {        // the block grows: what it holds in front of the run is written under the new power
    const float back = e4_pow2(max(before - power, -126));
    uint32_t* held = reinterpret_cast<uint32_t*>(base);
    for (int j = lane; j < begin * a.D / 4; j += 64) held[j] = e4_again(held[j], back);
  }
  const float scale = e4_pow2(-power);
  auto place = [&](int p, float (&y1)[8], float (&y2)[8]) {
    const int at_block = __shfl(slots, row_of(p)) & (E4_BLOCK - 1);
    if (!active || p * TOKENS + lane / L2 >= cnt) return;
    uint8_t* dst = base + (int64_t)at_block * a.D + 8 * l;
    *reinterpret_cast<u32x2*>(dst) = u32x2{e4_pack(y1[0], y1[1], y1[2], y1[3]), e4_pack(y1[4], y1[5], y1[6], y1[7])};
    *reinterpret_cast<u32x2*>(dst + half) = u32x2{e4_pack(y2[0], y2[1], y2[2], y2[3]), e4_pack(y2[4], y2[5], y2[6], y2[7])};
  };
  int again = 0;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    if (p > 0 && p * TOKENS >= cnt) continue;
    bool near = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x1[p][j] = e4_scaled(x1[p][j], scale); x2[p][j] = e4_scaled(x2[p][j], scale);
      near |= between(x1[p][j]) | between(x2[p][j]);
    }
    place(p, x1[p], x2[p]);
    if (__any(near)) again |= 1 << p;
  }
  // Once more where it matters, everything asked for again and written over what has been: nothing is held for it, which would cost the waves
  // of queries their registers.
#pragma unroll 1
  for (int p = 0; __builtin_expect(again >> p, 0); ++p) {
    if (!(again >> p & 1)) continue;
    asm volatile("" ::: "memory");
    bf16x8 t1, t2;
    Turn t;
    Weights weights;
    load(p, t1, t2, t);
    load_weights(a, a.k_w, at, weights);
    float y1[8], y2[8];
    norm_rotate_key<L2>(a, a.k_w != nullptr, weights, t, t1, t2, active, y1, y2);
#pragma unroll
    for (int j = 0; j < 8; ++j) { y1[j] = e4_scaled(y1[j], scale); y2[j] = e4_scaled(y2[j], scale); }
    place(p, y1, y2);
  }
  if (lane == 0) *code = (uint8_t)(power + E4_BIAS);
}

// The same of one value head: a lane has two neighbouring channels of all tokens, a channel's 16 places are 16 bytes of its page.
__device__ __forceinline__ void store_values(const AppendArgs& a, int64_t r, int cnt, int kvh, int lane, int slots) {
  const int s0 = __builtin_amdgcn_readlane(slots, 0);
  const int64_t pg = s0 >> a.page_shift;
  const int in_page = s0 & (a.page - 1), begin = in_page & (E4_BLOCK - 1), block = in_page & ~(E4_BLOCK - 1);
  uint8_t* code = a.v_powers + ((pg * a.Hkv + kvh) << (a.page_shift - 4)) + (in_page >> 4);
  const int before = begin > 0 ? min((int)*code - E4_BIAS, E4_MOST) : E4_LEAST;
  bf16x2 x[2][E4_BLOCK];           // head sizes up to 256: two pairs of channels to a lane
  const int pairs = a.D >> 1;
  float largest = 0.f;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (64 * c >= pairs) break;
    const int at = lane + 64 * c < pairs ? lane + 64 * c : 0;
    const bf16_t* src = a.rows + r * a.row_stride + (int64_t)(a.v_head + kvh) * a.D + 2 * at;
#pragma unroll
    for (int i = 0; i < E4_BLOCK; ++i) {
      x[c][i] = bf16x2{static_cast<bf16_t>(0.f), static_cast<bf16_t>(0.f)};
      if (i < cnt) {
        if (a.wide) x[c][i] = *reinterpret_cast<const bf16x2*>(src + i * a.row_stride);
        else x[c][i] = bf16x2{src[i * a.row_stride], src[i * a.row_stride + 1]};
      }
    }
#pragma unroll
    for (int i = 0; i < E4_BLOCK; ++i) largest = fmaxf(largest, fmaxf(e4_size(static_cast<float>(x[c][i][0])), e4_size(static_cast<float>(x[c][i][1]))));
  }
  const int power = max(e4_power(wave_max(largest)), before);
  const float scale = e4_pow2(-power), back = e4_pow2(max(before - power, -126));
  const bool grows = begin > 0 && power > before;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (64 * c >= pairs) break;
    if (lane + 64 * c >= pairs) continue;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint8_t* dst = a.v + ((pg * a.Hkv + kvh) * (int64_t)a.D + 2 * (lane + 64 * c) + e) * a.page + block;
      float f[E4_BLOCK];
#pragma unroll
      for (int i = 0; i < E4_BLOCK; ++i) f[i] = e4_scaled(static_cast<float>(x[c][i][e]), scale);
      u32x4v w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = e4_pack(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
      if (cnt == E4_BLOCK) {        // 16 ascending places of a block of 16: all of them
        *reinterpret_cast<u32x4v*>(dst) = w;
        continue;
      }
      if (grows) {
        u32x4v held = *reinterpret_cast<const u32x4v*>(dst);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int live = min(max(begin - 4 * i, 0), 4);
          const uint32_t keep = live == 4 ? 0xffffffffu : (1u << (8 * live)) - 1u;
          held[i] = (e4_again(held[i], back) & keep) | (held[i] & ~keep);
        }
        *reinterpret_cast<u32x4v*>(dst) = held;
      }
#pragma unroll
      for (int i = 0; i < E4_BLOCK; ++i)
        if (i < cnt) dst[__builtin_amdgcn_readlane(slots, i) & (E4_BLOCK - 1)] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
  }
  if (lane == 0) *code = (uint8_t)(power + E4_BIAS);
}
