// The write into the 8-bit cache (e4m3.h): per-head RMSNorm of q and k, rotation, and the scatter of k and v into their pages, in
// one launch over the packed rows. q goes out as rows of its own, rounded to bfloat16 once; k and v are rounded to e4m3 once, from
// the float32 results.
//
//   k' = rotated(w * k / rms(k));  block (16 places of a page, head): p = max(p_before if places in front of the call's first
//   place are held, least power with max |k'| <= 448 * 2^p);  stored: e4m3(k' 2^-p), numbers held before: e4m3(old 2^(p_before - p)).
//
// A power hangs on all of a call's tokens of the block, so the unit of work is a block's tokens and a head: one wave has all of
// them in registers, forms their maximum across its lanes, and nothing is read or rounded twice. Which tokens those are is found from
// the slots: consecutive rows whose slots ascend within a block are a run. A run that begins at place 0 opens its block anew; any other
// keeps what stands in front of it. Rows of one block that follow each other out of order (padding rows all name one slot) are runs
// one after the other, and one wave has them all; a run whose successor opens the same block anew is left out, since what
// it writes would be held no longer.
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
  int window;                    // rows whose runs a wave of keys or values walks
  int kv_groups;                 // workgroups of such waves per window
  int64_t kv_grid;               // workgroups of keys and values in front of those of the queries
  int wide;                      // rows, weights and angles are read 16 bytes at a time
};

// Eight neighbouring numbers of a row.
__device__ __forceinline__ void load8(const bf16_t* p, bool wide, float (&v)[8]) {
  bf16x8 t;
  if (wide) {
    t = *reinterpret_cast<const bf16x8*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(t[i]);
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

// Norm and rotation of a head that L2 lanes share: this lane's eight pairs (8 l + i, D / 2 + 8 l + i), l < D / 16. Lanes beyond
// those hold zeros.
template <int L2>
__device__ __forceinline__ void norm_rotate(const AppendArgs& a, const float* w, int l, int position, float (&x1)[8], float (&x2)[8]) {
  const int half = a.D >> 1;
  const bool wide = a.wide;
  float w1[8], w2[8], c0[8], c1[8];
  if (w) { load8(w + 8 * l, wide, w1); load8(w + half + 8 * l, wide, w2); }
  if (a.table) {
    const float* cs = a.table + ((int64_t)position * half + 8 * l) * 2;
    load8(cs, wide, c0); load8(cs + 8, wide, c1);
  }
  if (w) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x1[i] * x1[i] + x2[i] * x2[i];
#pragma unroll
    for (int off = L2 / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off, ME_WAVE);
    const float inv = rsqrtf(ss / (float)a.D + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) { x1[i] *= inv * w1[i]; x2[i] *= inv * w2[i]; }
  }
  if (a.table) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = i < 4 ? c0[2 * i] : c1[2 * i - 8], s = i < 4 ? c0[2 * i + 1] : c1[2 * i - 7];
      const float u = x1[i], v = x2[i];
      x1[i] = u * c - v * s;
      x2[i] = v * c + u * s;
    }
  }
}

__device__ __forceinline__ int row_position(const AppendArgs& a, int64_t t) {
  return a.table ? min(max(a.positions[t], 0), a.table_positions - 1) : 0;
}
__device__ __forceinline__ int row_slot(const AppendArgs& a, int64_t t) {
  const int s = t >= 0 && t < a.T ? a.slots[t] : -1;
  return s < a.slot_end ? s : -1;
}

// The tokens [r, e) of one block, of one key head (e - r <= 16, ascending slots).
template <int L2>
__device__ __forceinline__ void store_keys(const AppendArgs& a, int64_t r, int cnt, int kvh, int lane) {
  constexpr int TOKENS = 64 / L2, PASSES = TOKENS >= E4_BLOCK ? 1 : E4_BLOCK / TOKENS;
  const int l = lane % L2, half = a.D >> 1;
  const bool active = l < (a.D >> 4);
  float x1[PASSES][8], x2[PASSES][8];
  int off[PASSES];
  const int s0 = row_slot(a, r);
  const int64_t pg = s0 >> a.page_shift;
  const int in_page = s0 & (a.page - 1), begin = in_page & (E4_BLOCK - 1);
  uint8_t* code = a.k_powers + ((pg * a.Hkv + kvh) << (a.page_shift - 4)) + (in_page >> 4);
  const int before = begin > 0 ? min((int)*code - E4_BIAS, E4_MOST) : E4_LEAST;
  float largest = 0.f;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int i = p * TOKENS + lane / L2;
    const int64_t t = r + min(i, cnt - 1);
    off[p] = i < cnt ? row_slot(a, t) & (a.page - 1) : -1;
    const bf16_t* row = a.rows + t * a.row_stride + (int64_t)(a.Hq + kvh) * a.D + (active ? 8 * l : 0);
    load8(row, a.wide, x1[p]); load8(row + half, a.wide, x2[p]);
    if (!active) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x1[p][j] = x2[p][j] = 0.f;
    }
    norm_rotate<L2>(a, a.k_w, active ? l : 0, row_position(a, t), x1[p], x2[p]);
    // (rows beyond the run repeat its last one: they change no maximum)
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
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    if (!active || off[p] < 0) continue;
    uint8_t* dst = base + (int64_t)(off[p] & (E4_BLOCK - 1)) * a.D + 8 * l;
#pragma unroll
    for (int j = 0; j < 8; ++j) { x1[p][j] = e4_scaled(x1[p][j], scale); x2[p][j] = e4_scaled(x2[p][j], scale); }
    *reinterpret_cast<u32x2*>(dst) = u32x2{e4_pack(x1[p][0], x1[p][1], x1[p][2], x1[p][3]), e4_pack(x1[p][4], x1[p][5], x1[p][6], x1[p][7])};
    *reinterpret_cast<u32x2*>(dst + half) = u32x2{e4_pack(x2[p][0], x2[p][1], x2[p][2], x2[p][3]), e4_pack(x2[p][4], x2[p][5], x2[p][6], x2[p][7])};
  }
  if (lane == 0) *code = (uint8_t)(power + E4_BIAS);
}

// The same of one value head: a lane has two neighbouring channels of all tokens, a channel's 16 places are 16 bytes of its page.
__device__ __forceinline__ void store_values(const AppendArgs& a, int64_t r, int cnt, int kvh, int lane) {
  const int s0 = row_slot(a, r);
  const int64_t pg = s0 >> a.page_shift;
  const int in_page = s0 & (a.page - 1), begin = in_page & (E4_BLOCK - 1), block = in_page & ~(E4_BLOCK - 1);
  uint8_t* code = a.v_powers + ((pg * a.Hkv + kvh) << (a.page_shift - 4)) + (in_page >> 4);
  const int before = begin > 0 ? min((int)*code - E4_BIAS, E4_MOST) : E4_LEAST;
  const int my_slot = row_slot(a, r + min(lane & 15, cnt - 1)) & (E4_BLOCK - 1);
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
        if (i < cnt) dst[__builtin_amdgcn_readlane(my_slot, i)] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
  }
  if (lane == 0) *code = (uint8_t)(power + E4_BIAS);
}

// Whether row t does not go on from row t - 1 within a block, or opens the block anew.
__device__ __forceinline__ bool breaks(int before, int slot) { return slot < 0 || before < 0 || (slot >> 4) != (before >> 4) || (slot & 15) == 0; }

template <int L2>
__global__ void __launch_bounds__(256) append_e4m3_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int64_t)blockIdx.x >= a.kv_grid) {        // queries: L2 lanes to a head, heads of all rows in a row
    const int64_t head_of_all = (((int64_t)blockIdx.x - a.kv_grid) * 4 + wave) * (64 / L2) + lane / L2;
    const int l = lane % L2;
    const bool active = head_of_all < a.T * a.Hq && l < (a.D >> 4);
    const int64_t t = active ? head_of_all / a.Hq : 0;
    const int head = active ? (int)(head_of_all - t * a.Hq) : 0, half = a.D >> 1;
    const bf16_t* row = a.rows + t * a.row_stride + (int64_t)head * a.D + (active ? 8 * l : 0);
    const int position = row_position(a, t);
    float x1[8], x2[8];
    load8(row, a.wide, x1); load8(row + half, a.wide, x2);
    if (!active) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x1[j] = x2[j] = 0.f;
    }
    norm_rotate<L2>(a, a.q_w, active ? l : 0, position, x1, x2);
    if (!active) return;
    bf16x8 o1, o2;
#pragma unroll
    for (int j = 0; j < 8; ++j) { o1[j] = static_cast<bf16_t>(x1[j]); o2[j] = static_cast<bf16_t>(x2[j]); }
    bf16_t* dst = a.q_out + (t * a.Hq + head) * a.D + 8 * l;
    *reinterpret_cast<bf16x8*>(dst) = o1;
    *reinterpret_cast<bf16x8*>(dst + half) = o2;
    return;
  }
  const int unit = ((int)blockIdx.x % a.kv_groups) * 4 + wave;       // key heads, then value heads
  if (unit >= 2 * a.Hkv) return;
  const int64_t t0 = (int64_t)(blockIdx.x / a.kv_groups) * a.window;
  // lane i: row t0 + i and the one in front of it
  const int slot = row_slot(a, t0 + lane), prev = row_slot(a, t0 + lane - 1);
  const uint64_t stops = __ballot(breaks(prev, slot));
  const uint64_t opens = __ballot(slot >= 0 && prev >= 0 && (slot >> 4) == (prev >> 4) && (slot & 15) == 0);     // ... the block of the row in front
  const uint64_t rises = __ballot(slot > prev);
  uint64_t todo = stops & __ballot(slot >= 0) & ((1ull << a.window) - 1);
  while (todo) {
    const int i = __builtin_ctzll(todo);
    todo &= todo - 1;
    // the chain of rows [i, end) of this block, and whether the row behind it opens the block anew
    const uint64_t behind = i == 63 ? 0 : stops >> (i + 1) << (i + 1);
    int64_t end;
    bool dead;
    if (behind) {
      const int e = __builtin_ctzll(behind);
      end = t0 + e;
      dead = (opens >> e) & 1;
    } else {                       // beyond the 64 rows: only where a block's rows are out of order
      end = t0 + 64;
      while (end < a.T && !breaks(row_slot(a, end - 1), row_slot(a, end))) ++end;
      const int s = row_slot(a, end), p = row_slot(a, end - 1);
      dead = s >= 0 && (s >> 4) == (p >> 4) && (s & 15) == 0;
    }
    if (dead) continue;
    int64_t r = t0 + i;
    while (r < end) {
      int64_t e;
      const int at = (int)(r - t0);
      const uint64_t falls = at >= 0 && at < 63 ? (~rises) >> (at + 1) << (at + 1) : 0;
      if (falls) {
        e = min(end, t0 + (int64_t)__builtin_ctzll(falls));
      } else {
        e = r + 1;
        while (e < end && row_slot(a, e) > row_slot(a, e - 1)) ++e;
      }
      if (unit < a.Hkv) store_keys<L2>(a, r, (int)(e - r), unit, lane);
      else store_values(a, r, (int)(e - r), unit - a.Hkv, lane);
      r = e;
      if (r < end) __threadfence();      // the next run of the block reads what this one has written
    }
  }
}

extern "C" int me_append_e4m3(const void* rows, int64_t row_stride, void* q_out, const float* q_w, const float* k_w, float eps,
                              const float* table, int64_t table_positions, int64_t position_bound, const int32_t* positions,
                              const int32_t* slots, void* k, void* v, void* k_powers, void* v_powers, int64_t num_pages, int64_t num_tokens,
                              int Hq, int Hkv, int D, int page, int values_are_keys, hipStream_t stream) {
  if (num_tokens == 0) return 0;
  ME_CHECK(D >= 16 && D <= 256 && D % 16 == 0, "append_e4m3: head size %d must be a multiple of 16 up to 256", D);
  ME_CHECK(page >= E4_BLOCK && (page & (page - 1)) == 0, "append_e4m3: page size %d must be a power of two, 16 or more", page);
  ME_CHECK(Hq >= 0 && Hkv >= 1 && num_tokens > 0, "append_e4m3: bad head or token counts");
  ME_CHECK(row_stride >= (int64_t)(Hq + (values_are_keys ? 1 : 2) * Hkv) * D, "append_e4m3: row stride too small");
  ME_CHECK(num_pages >= 1 && num_pages * page < (1ll << 31), "append_e4m3: %lld pages of %d tokens are more places than a slot can name", (long long)num_pages, page);
  ME_CHECK((q_w == nullptr) == (k_w == nullptr), "append_e4m3: give both norm weights or neither");
  ME_CHECK(!table || (table_positions > 0 && table_positions < (1ll << 31)), "append_e4m3: bad rotation table");
  ME_CHECK(!table || position_bound <= table_positions, "append_e4m3: positions up to %lld are beyond the rotation table's %lld",
           (long long)position_bound - 1, (long long)table_positions);
  for (const void* p : {(const void*)k, (const void*)v})
    ME_CHECK(p != nullptr && reinterpret_cast<uintptr_t>(p) % 16 == 0, "append_e4m3: caches must be 16-byte aligned");
  ME_CHECK(reinterpret_cast<uintptr_t>(q_out) % 16 == 0, "append_e4m3: the queries' rows must be 16-byte aligned");
  AppendArgs a;
  a.rows = (const bf16_t*)rows; a.row_stride = row_stride; a.q_out = (bf16_t*)q_out; a.q_w = q_w; a.k_w = k_w; a.eps = eps;
  a.table = table; a.table_positions = (int)table_positions; a.positions = positions; a.slots = slots; a.slot_end = (int)(num_pages * page);
  a.k = (uint8_t*)k; a.v = (uint8_t*)v; a.k_powers = (uint8_t*)k_powers; a.v_powers = (uint8_t*)v_powers;
  a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.page = page; a.page_shift = __builtin_ctz(page); a.v_head = values_are_keys ? Hq : Hq + Hkv; a.T = num_tokens;
  a.wide = row_stride % 8 == 0;
  for (const void* p : {rows, (const void*)q_w, (const void*)k_w, (const void*)table}) a.wide = a.wide && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  a.window = num_tokens > 256 ? 16 : 1;
  a.kv_groups = (2 * Hkv + 3) / 4;
  a.kv_grid = (num_tokens + a.window - 1) / a.window * a.kv_groups;
  int l2 = 1;
  while (l2 < D / 16) l2 *= 2;
  const int64_t heads_of_group = 4 * (64 / l2);
  const int64_t grid = a.kv_grid + (num_tokens * Hq + heads_of_group - 1) / heads_of_group;
  ME_CHECK(grid < (1ll << 31), "append_e4m3: too many tokens for one launch");
  switch (l2) {
    case 1: append_e4m3_kernel<1><<<(unsigned)grid, 256, 0, stream>>>(a); break;
    case 2: append_e4m3_kernel<2><<<(unsigned)grid, 256, 0, stream>>>(a); break;
    case 4: append_e4m3_kernel<4><<<(unsigned)grid, 256, 0, stream>>>(a); break;
    case 8: append_e4m3_kernel<8><<<(unsigned)grid, 256, 0, stream>>>(a); break;
    default: append_e4m3_kernel<16><<<(unsigned)grid, 256, 0, stream>>>(a); break;
  }
  ME_LAUNCH_CHECK();
  return 0;
}
