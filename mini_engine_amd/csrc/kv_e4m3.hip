// The write into the 8-bit cache (e4m3.h): per-head RMSNorm of q and k, rotation, and the scatter of k and v into their pages, in
// one launch over the packed rows. q goes out as rows of its own, rounded to bfloat16 once; k and v are rounded to e4m3 once, from
// the float32 results (v is its row's number as it is). A key that lies within 8 float32 steps of the middle between two e4m3 numbers is
// rounded from an exact result; what cancellation in the rotation leaves further off than that may still fall to the other side, and
// a block's power goes by the float32 results.
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
#include "kv_e4m3.h"

// Heads of a lane group that a wave of queries takes, asked for at once (7,900 rows of 32 heads of 128 beside 8 key heads: 1, 2, 4 of them 67, 54, 49 us).
constexpr int Q_PASSES = 4;

// Whether row t does not go on from row t - 1 within a block, or opens the block anew.
__device__ __forceinline__ bool breaks(int before, int slot) { return slot < 0 || before < 0 || (slot >> 4) != (before >> 4) || (slot & 15) == 0; }

template <int L2>
__global__ void __launch_bounds__(256, L2 <= 8 ? 4 : 1) append_e4m3_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int64_t)blockIdx.x >= a.kv_grid) {        // queries: L2 lanes to a head, so many heads of a row to a wave that reads weights and angles once
    constexpr int HEADS = 64 / L2, PASSES = Q_PASSES;
    const int64_t piece = ((int64_t)blockIdx.x - a.kv_grid) * 4 + wave;
    const int64_t t = piece / a.q_parts;
    if (t >= a.T) return;
    const int l = lane % L2, half = a.D >> 1, h0 = (int)(piece - t * a.q_parts) * (PASSES * HEADS) + lane / L2;
    const bool there = l < (a.D >> 4);
    const int at = there ? 8 * l : 0;
    const int position = row_position(a, t);
    const bf16_t* row = a.rows + t * a.row_stride + at;
    bf16x8 raw1[PASSES], raw2[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const bf16_t* from = row + (int64_t)(h0 + i * HEADS < a.Hq ? h0 + i * HEADS : 0) * a.D;
      raw1[i] = load8(from, a.wide); raw2[i] = load8(from + half, a.wide);
    }
    Weights w;
    Turn turn;
    load_weights(a, a.q_w, at, w);
    load_turn(a, at, position, turn);
    bf16_t* out = a.q_out + t * a.Hq * a.D + at;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      float x1[8], x2[8];
      norm_rotate<L2>(a, a.q_w != nullptr, w, turn, raw1[i], raw2[i], there, x1, x2);
      if (!there || h0 + i * HEADS >= a.Hq) continue;
      bf16x8 o1, o2;
#pragma unroll
      for (int j = 0; j < 8; ++j) { o1[j] = static_cast<bf16_t>(x1[j]); o2[j] = static_cast<bf16_t>(x2[j]); }
      bf16_t* dst = out + (int64_t)(h0 + i * HEADS) * a.D;
      *reinterpret_cast<bf16x8*>(dst) = o1;
      *reinterpret_cast<bf16x8*>(dst + half) = o2;
    }
    return;
  }
  const int unit = (int)(blockIdx.x % a.kv_groups) * 4 + wave;       // key heads, then value heads
  if (unit >= 2 * a.Hkv) return;
  const int piece = blockIdx.x / a.kv_groups, first = a.first_rows / a.first_window;
  const int window = piece < first ? a.first_window : a.window;
  const int64_t t0 = piece < first ? (int64_t)piece * window : a.first_rows + (int64_t)(piece - first) * window;
  // lane i: row t0 + i and the one in front of it
  const int slot = row_slot(a, t0 + lane), prev = row_slot(a, t0 + lane - 1), place = row_position(a, t0 + lane);
  const uint64_t stops = __ballot(breaks(prev, slot));
  const uint64_t opens = __ballot(slot >= 0 && prev >= 0 && (slot >> 4) == (prev >> 4) && (slot & 15) == 0);     // ... the block of the row in front
  const uint64_t rises = __ballot(slot > prev);
  uint64_t todo = stops & __ballot(slot >= 0) & ((1ull << window) - 1);
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
      // the run's slots and positions: of the rows at hand, or beyond them
      const bool near = at + E4_BLOCK <= 64;
      const int run_slots = near ? __shfl(slot, (at + lane) & 63) : row_slot(a, r + lane);
      if (unit < a.Hkv) store_keys<L2>(a, r, (int)(e - r), unit, lane, run_slots, near ? __shfl(place, (at + lane) & 63) : row_position(a, r + lane));
      else store_values(a, r, (int)(e - r), unit - a.Hkv, lane, run_slots);
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
  // Rows of prompts go 16 to a wave of every head, which then has a block or two; workgroups that find nothing cost 7 ns each (windows of 8 in place
  // of 16 rows: 67 us for 49), so a window is not smaller there. Decoding requests, which stand in front, bring a run in every row, and a wave
  // walks its runs one after the other: the first 256 rows go 4 to a wave, or 1 where there are no more (60 such rows in front of 7,900 of
  // prompts: 88 us with 16 to a wave).
  a.window = 16;
  a.first_window = num_tokens > 256 ? 4 : 1;
  a.first_rows = num_tokens > 256 ? 256 : (int)num_tokens;
  a.kv_groups = (2 * Hkv + 3) / 4;
  a.kv_grid = (a.first_rows / a.first_window + (num_tokens - a.first_rows + a.window - 1) / a.window) * a.kv_groups;
  int l2 = 1;
  while (l2 < D / 16) l2 *= 2;
  a.q_parts = (Hq + Q_PASSES * (64 / l2) - 1) / (Q_PASSES * (64 / l2));
  const int64_t grid = a.kv_grid + (num_tokens * a.q_parts + 3) / 4;
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
