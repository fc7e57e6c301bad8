// aq_paged_attention.hip -- attention of new tokens of several sequences over
// a paged cache.
//
// out = softmax(scale q k^T + mask) v in one pass over the keys that a block of
// queries can see: with the running maximum m of a query's scores and the sums
// l = sum e^(s - m), o = sum e^(s - m) v so far, a tile of keys with maximum m'
// scales l and o by e^(m - max(m, m')) and adds its own terms.  Parts of the keys
// taken by different workgroups meet the same way (paged_merge_kernel).
//
// The G query heads that share a key/value head are rows of one block: row r of
// a sequence's n G rows is its new token r / G, head r % G of the group.
#include "aq_paged.h"

namespace {

using namespace paged;

constexpr int kQ = 128;  // rows a workgroup, 32 a wave
constexpr int kK = 64;   // keys a tile
constexpr int kFewRows = 32;  // rows of a sequence that the kernel for few takes at most
constexpr float kGrow = 8.0f;

struct AttendArgs {
  Batch b;
  const uint16_t *q, *k, *v;
  int64_t qs[2];  // elements between rows, heads
  uint16_t* out;
  float* part;    // [T, H, slots, D], sums, then [T, H, slots, 2], maxima and denominators
  int H, G, Hkv, window, sinks, items, per;
  int few;                 // sequences of up to so many rows are the first kernel's, the others the second's
  int few_span, few_spans; // steps a workgroup of the first kernel, workgroups a sequence
  int span;                // tiles a workgroup of the second
  int slots;               // the larger number of spans
  int few_eights, many_eights;  // eights of workgroups of both, where they share a launch
  float c;  // |scale| log2(e), above 0: a masked score, -inf, times it stays that
  uint32_t keep, flip;  // for the queries' bits: none for a scale of 0, the sign of a negative one
};

// Maxima and denominators of the spans.
template <int D>
__device__ __forceinline__ float2* ends_of(const AttendArgs& a) {
  return reinterpret_cast<float2*>(a.part + (int64_t)a.b.T * a.H * a.slots * D);
}

// A buffer of `bytes` at p, for loads that read zeros past its end.
__device__ __forceinline__ u32x4 buffer_of(const uint16_t* p, int bytes) {
  return u32x4{(uint32_t)(uintptr_t)p, (uint32_t)((uintptr_t)p >> 32) & 0xFFFFu, (uint32_t)bytes, 0x00020000u};
}

// N times 16 bytes a lane from a buffer's bytes off[n] straight to LDS, to
// dst + 1024 n + 16 lane.  In assembly, since the compiler, which knows of such
// loads, waits for all of them before it reads from LDS anything that it cannot
// tell apart: the waits are the caller's (s_waitcnt vmcnt).  The buffer's registers
// may have been written by the vector unit just before: five wait states.
template <int N>
__device__ __forceinline__ void load_to_lds(u32x4 r, uint32_t dst, const int (&off)[N]) {
#pragma unroll
  for (int n = 0; n < N; n++) {
    if (n == 0)
      asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"{m0}"(dst), "v"(off[0]), "s"(r) : "memory");
    else
      asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"{m0}"(dst + 1024 * n), "v"(off[n]), "s"(r) : "memory");
  }
}

__device__ __forceinline__ uint32_t lds_offset(const uint8_t* p) { return (uint32_t)(uintptr_t)(lds_u8*)p; }

// Four rows of 16 numbers of 16 bits in LDS, 8 bytes given by each of 16 lanes
// in order: lane i gets column i.
__device__ __forceinline__ u32x2 read_turned(const uint8_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds_u8*)p));
}

// The larger of m and the magnitudes of eight numbers, as pairs of bits.
__device__ __forceinline__ u16x2 magnitudes8(u16x2 m, uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
  return m;
}

// Two numbers, those that are not finite as zeros.
template <class T>
__device__ __forceinline__ uint32_t finite2(uint32_t x) {
  const uint32_t lo = (x & 0x7FFF) >= T::kInf ? 0 : x & 0xFFFF, hi = ((x >> 16) & 0x7FFF) >= T::kInf ? 0 : x & 0xFFFF0000u;
  return lo | hi;
}

// Rows of a sequence, and the tiles of `keys` keys that a block of them sees: tiles
// 0 .. na - 1 hold the sinks, then come b0 .. b0 + tiles - na - 1.
struct Block {
  int first, n, len, r0;  // the sequence's first row, its new tokens, its length; the block's first row
  int lo, hi;             // positions of the block's first and last row
  int b0, na, tiles, sink_end;
};

// s: the sequence; r0: the block's first of its rows, of `rows`; all the same in
// every lane.
template <int KEYS>
__device__ __forceinline__ bool find_block(const AttendArgs& a, int s, int r0, int rows, Block& k) {
  k.first = a.b.scalar_start(s);
  k.n = max(a.b.scalar_start(s + 1) - k.first, 0);
  k.len = scalar_int(a.b.lengths, s);
  k.r0 = r0;
  if (r0 >= k.n * a.G || k.n > k.len || k.n > a.b.max_new || k.len > a.b.max_length) return false;
  k.lo = k.len - k.n + r0 / a.G;
  k.hi = k.len - k.n + min(r0 + rows - 1, k.n * a.G - 1) / a.G;
  const int near = max(k.lo - a.window + 1, 0);
  k.b0 = near / KEYS;
  k.sink_end = min(a.sinks, k.hi + 1);
  k.na = k.sink_end > 0 ? min((k.sink_end - 1) / KEYS + 1, k.b0) : 0;
  k.tiles = k.na + k.hi / KEYS - k.b0 + 1;
  return true;
}

// The sequence that block `blk` belongs to, -1 for none, and its first block: sequence
// s's are starts[s] G / 128 + s and on (as many as its rows can need, or one more).
__device__ __forceinline__ int find_sequence(const AttendArgs& a, int blk, int& first) {
  const int s = last_at_most(a.b.S, blk, [&](int i) { return a.b.start(i) * a.G / kQ + i; });
  if (s < 0 || blk > a.b.scalar_start(s + 1) * a.G / kQ + s) return -1;
  first = a.b.scalar_start(s) * a.G / kQ + s;
  return s;
}

// A tile's rows lie in LDS one after the other, 16-byte pieces permuted within each
// so that the reads below meet every bank equally.  Keys, 16 rows at once: piece c of
// row r at c ^ (r & 15), for D = 64, where two rows fill the banks, c ^ (r / 2 & 7).
// Values, 64 bytes of 4 rows at once: pairs of pieces at (c / 2) ^ 2 (r & 3), for
// D = 64 (c / 2) ^ 2 (r / 2 & 1).
template <int D>
__device__ __forceinline__ int k_place(int r, int c) { return r * (D * 2) + (c ^ (D == 128 ? r & 15 : (r >> 1) & 7)) * 16; }
template <int D>
__device__ __forceinline__ int v_place(int r, int c) {
  return r * (D * 2) + ((((c >> 1) ^ (2 * (D == 128 ? r & 3 : (r >> 1) & 1))) << 1) | (c & 1)) * 16;
}

// The same for the values of the kernel for few rows, whose lanes read 16 rows at
// once: pairs of pieces at (c / 2) ^ (r & 7), or ^ (r / 2 & 3) where two rows fill the banks.
template <int D>
__device__ __forceinline__ int few_place(int r, int c) {
  return r * (D * 2) + ((((c >> 1) ^ (D == 128 ? r & 7 : (r >> 1) & 3)) << 1) | (c & 1)) * 16;
}

// One workgroup: 128 rows of a key/value head, 32 a wave; tiles of 64 keys and
// values go straight from their pages to LDS (a wave loads 16 rows of each, which
// lie in one page), and are taken in halves of 32 keys:
//   scores   transposed, s^T = k q^T (mfma 32 x 32 x 16): a lane has 16 scores of
//            one row, another lane the other 16
//   softmax  p = e^(s - m) with m the maximum when it last moved: it moves only
//            when a score passes it by 2^8, which spares scaling the sums nearly always
//   values   o^T = v^T p^T: the numerators, rounded to 16 bits, are the operand as
//            they are (their rest, as the kernel for few rows has it, would be half as many
//            products again where products are what takes the time); the values come out of
//            their rows transposed
//   sums     of the rounded numerators, so that rounding them does not shift the mean
// The products of the next half's scores stand among the exponentials of this one's in
// the code, so that the matrix unit works under them, and a half's keys are in
// registers a half before they are needed.  So when everyone comes to a tile's one
// barrier, its keys and the last tile's values are done with; what takes their places
// in LDS, the keys of two tiles on and the values of the next, has a tile's time.
// A prompt of 8192, 32 heads of 128 over 8 key/value heads: 544 to 590 us, 930 to
// 1010 TFLOP/s of the two products (the library's fp16 product of 8192^3: 1177).  By
// counters 1.0 M cycles, the matrix unit busy in 53 % of them, the vector unit in 48 %, no bank
// conflicts; that is 1.8 GHz at 554 us.  One half after the other, without the places and
// the registers ahead, it took 614.  Nothing gained: workgroups of 256 rows, also with four
// tiles in flight (580 against 590), other proportions of the interleaving (all within 1 %),
// the loads later in the tile (580 against 570).
// lds: many_lds<D> bytes, on a multiple of 1024: keys of even and odd tiles, values
template <int D>
constexpr int many_lds = 4 * kK * D * 2 + 16;

template <class T, int D>
__device__ __forceinline__ void many_block(const AttendArgs& a, int block, int part, uint8_t* lds) {
  constexpr int NC = D / 8;                    // 16-byte pieces of a row
  constexpr int TB = kK * D * 2;               // bytes of a tile of keys, or of values
  constexpr int PN = TB / 1024 / 4;            // 1 KiB loads of each a wave: 16 rows
  // whether a tile that the mask cuts had an infinity or NaN among its values
  volatile int& bad = *reinterpret_cast<volatile int*>(lds + 4 * TB);
  const int t = threadIdx.x, ln = t & 63, c = ln & 31, h = ln >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  // runs of neighbouring items to an XCD (they share keys and values in its L2)
  const int item = (block & 7) * a.per + (block >> 3);
  if ((block >> 3) >= a.per || item >= a.items) return;
  const int blocks = a.items / a.Hkv;
  const int j = item / blocks, blk = blocks - 1 - item % blocks;  // late blocks (more keys) first
  int blk0;
  const int seq = find_sequence(a, blk, blk0);
  if (seq < 0) return;
  Block B;
  if (!find_block<kK>(a, seq, (blk - blk0) * kQ, kQ, B) || B.n * a.G <= a.few) return;
  const int t0 = part * a.span, t1 = min(t0 + a.span, B.tiles);
  if (t0 >= t1) return;
  if (t == 0) bad = 0;  // (before any wave may set it, which is behind the first barrier)
  const int lo = B.lo, hi = B.hi;
  auto tile_at = [&](int i) { return (i < B.na ? i : B.b0 + i - B.na) * kK; };
  auto cut = [&](int k0) { return !(k0 + kK - 1 <= lo && k0 > hi - a.window); };  // whether some row does not see all of it

  const int row = B.r0 + wave * 32 + c, last_row = B.n * a.G - 1;  // this lane's row
  const int tok = min(row, last_row) / a.G, head = j * a.G + (min(row, last_row) - tok * a.G);
  const int qpos = B.len - B.n + tok;
  u32x4 qv[D / 16];
  {
    const uint16_t* qp = a.q + (int64_t)(B.first + tok) * a.qs[0] + head * a.qs[1] + 8 * h;
#pragma unroll
    for (int s = 0; s < D / 16; s++) {
      u32x4 x = *reinterpret_cast<const u32x4*>(qp + 16 * s);
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = (x[i] & a.keep) ^ a.flip;
      qv[s] = x;
    }
  }
  float16v o[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; e++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[e][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  // positions of the wave's rows
  const int wlo = B.len - B.n + min(B.r0 + wave * 32, last_row) / a.G;
  const int whi = B.len - B.n + min(B.r0 + wave * 32 + 31, last_row) / a.G;
  const float grow = kGrow / a.c;

  // this lane's part of the loads: piece n of the wave covers rows of its 16
  int ko[PN], vo[PN];
#pragma unroll
  for (int n = 0; n < PN; n++) {
    const int r = n * (64 / NC) + ln / NC, pc = ln % NC;
    ko[n] = k_place<D>(r, pc);  // (the places are their own inverse)
    vo[n] = v_place<D>(r, pc);
  }
  // The pages of this wave's 16 rows of 64 tiles from p0 on, one a lane (past the last
  // tile: any): read one by one by the scalar unit they would come at any time among the
  // answers of LDS, which would have to be waited for all together.
  const int* table = a.b.table + (int64_t)seq * a.b.W;
  int p0, pages;
  auto read_pages = [&](int i) {
    p0 = i;
    pages = table[min((tile_at(min(i + ln, t1 - 1)) + wave * 16) >> a.b.shift, (B.len - 1) >> a.b.shift)];
    asm volatile("" : "+v"(pages));  // (waited for here)
  };
  auto page_at = [&](int i) { return __builtin_amdgcn_readlane(pages, i - p0); };
  auto load = [&](const uint16_t* base, int i, int page, uint32_t dst, const int (&off)[PN]) {
    const int k0 = tile_at(i) + wave * 16;
    // rows past the last, and those of a page outside the cache, read as zeros
    const bool there = (unsigned)page < (unsigned)a.b.pages;
    // (a median is taken by the vector unit)
    const int bytes = there ? __builtin_amdgcn_readfirstlane(max(min(B.len - k0, 16), 0)) * (D * 2) : 0;
    const int64_t at = (((((int64_t)(there ? page : 0) * a.Hkv + j) << a.b.shift) + (k0 & ((1 << a.b.shift) - 1)))) * D;
    load_to_lds<PN>(buffer_of(base + at, bytes), dst + (i & 1) * TB + wave * PN * 1024, off);
  };
  const uint32_t k_lds = lds_offset(lds), v_lds = k_lds + 2 * TB;
  // LDS offsets of this lane's first fragments: keys of row c, pieces 2 e + h; values of
  // keys 4 h + r, 16 elements of 32 e.  The others' are these with 32 e and 64 e
  // exclusive or (worked out where they are used: kept, they took registers that
  // there are not).
  const int kf = k_place<D>(c, h), vf = v_place<D>(4 * h + ((ln >> 2) & 3), 2 * ((ln >> 4) & 1) + ((ln & 3) >> 1)) + (ln & 1) * 8;

  // Fragments of half y of tile i: its keys, its values (16 s + 4 h + 0 .. 3, then 8 on:
  // the order in which a lane has the numerators).
  u32x4 kr[D / 16];
  u32x2 vr[D / 32][2];
  auto read_keys = [&](int i, int y) {
    const int at = kf + (i & 1) * TB + y * 32 * (D * 2);
#pragma unroll
    for (int e = 0; e < D / 16; e++) kr[e] = *reinterpret_cast<const u32x4*>(lds + (at ^ (32 * e)));
  };
  auto read_values = [&](int i, int y, int s) {
    const int at = vf + 2 * TB + (i & 1) * TB + (32 * y + 16 * s) * (D * 2);
#pragma unroll
    for (int e = 0; e < D / 32; e++)
#pragma unroll
      for (int n = 0; n < 2; n++) vr[e][n] = read_turned(lds + (at ^ (64 * e)) + 8 * n * (D * 2));
  };
  auto products = [&](float16v& x) {
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 16; e++) x = T::mfma32(kr[e], qv[e], x);
  };
  // what the mask leaves of scores from key k0 on, and the maximum moved where they pass it
  auto settle = [&](int k0, float16v& x) {
    if (!(k0 + 31 <= wlo && k0 > whi - a.window)) {
      // a key is seen when it lies in one of two ranges: near the row's position,
      // or among the sinks, both up to that position (each a subtraction, an
      // unsigned comparison and a selection)
      const int last = qpos - k0 - 4 * h, from = max(last - a.window + 1, -k0 - 4 * h);
      const int sink0 = -k0 - 4 * h;
      const uint32_t near_n = (uint32_t)max(last - from + 1, 0);
      const uint32_t sink_n = (uint32_t)max(min(a.sinks, last - sink0 + 1), 0);
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int key = 8 * (e >> 2) + (e & 3);
        const float y = (uint32_t)(key - sink0) < sink_n ? x[e] : -INFINITY;
        x[e] = (uint32_t)(key - from) < near_n ? x[e] : y;
      }
    }
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < 15; e += 2) mx = fmaxf(fmaxf(mx, x[e]), x[e + 1]);  // v_max3
    mx = fmaxf(mx, x[15]);
    if (__ballot(mx > m + grow)) {
      mx = xlane_level_max_f32<6>(mx);  // both lanes of a row move alike
      const float n = fmaxf(m, mx), f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - n) * a.c);
      l *= f;
#pragma unroll
      for (int e = 0; e < D / 32; e++) o[e] *= f;
      m = n;
    }
  };
  // numerators of scores x: p[4 n .. 4 n + 3] are the operand of 16 keys
  auto numerators = [&](const float16v& x, u32x8& p) {
    const float base = m == -INFINITY ? 0.0f : -m * a.c;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      p[e] = T::pack(__builtin_amdgcn_exp2f(fmaf(x[2 * e], a.c, base)), __builtin_amdgcn_exp2f(fmaf(x[2 * e + 1], a.c, base)));
      l = T::add2(p[e], l);
    }
  };
  auto sums = [&](int s, const u32x8& p) {
#pragma unroll
    for (int e = 0; e < D / 32; e++)
      o[e] = T::mfma32(u32x4{vr[e][0].x, vr[e][0].y, vr[e][1].x, vr[e][1].y},
                       u32x4{p[4 * s], p[4 * s + 1], p[4 * s + 2], p[4 * s + 3]}, o[e]);
  };
  read_pages(t0);
  load(a.k, t0, page_at(t0), k_lds, ko);
  load(a.v, t0, page_at(t0), v_lds, vo);
  if (t0 + 1 < t1) {
    load(a.k, t0 + 1, page_at(t0 + 1), k_lds, ko);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PN) : "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PN) : "memory");
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the first keys are there
  float16v x, x1;
  read_keys(t0, 0);
  products(x);
  read_keys(t0, 1);
  settle(tile_at(t0), x);
  for (int i = t0; i < t1; i++) {
    const int k0 = tile_at(i);
    // this wave's part of the values of this tile and the keys of the next is there
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (cut(k0)) {
      // The mask cuts the tile for some row: infinities and NaN among its values count as
      // zeros here, so that a weight of zero leaves them out, and reach the rows that
      // see them at the end.
#pragma unroll
      for (int n = 0; n < PN; n++) {
        uint4* at = reinterpret_cast<uint4*>(lds + 2 * TB + (i & 1) * TB + (wave * PN + n) * 1024 + ln * 16);
        uint4 z = *at;
        const u16x2 most = magnitudes8(0, z);
        if (__ballot(max(most.x, most.y) >= T::kInf)) {
#pragma unroll
          for (int w = 0; w < 4; w++) (&z.x)[w] = finite2<T>((&z.x)[w]);
          *at = z;
          bad = 1;
        }
      }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0), in a form that the compiler takes into account
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (i + 1 < t1) {
      if (i + 2 - p0 >= 64) read_pages(i + 1);
      load(a.v, i + 1, page_at(i + 1), v_lds, vo);
      if (i + 2 < t1) load(a.k, i + 2, page_at(i + 2), k_lds, ko);
    }
    u32x8 p;
#pragma unroll
    for (int y = 0; y < 2; y++) {
      // (behind the last tile, keys that nobody looks at)
      float16v &now = y ? x1 : x, &next = y ? x : x1;
      read_values(i, y, 0);
      __builtin_amdgcn_sched_barrier(0);  // (they are on their way under what follows)
      // (before the other workgroup's wave while there are products to feed: 2 %)
      __builtin_amdgcn_s_setprio(1);
      products(next);
      numerators(now, p);
#pragma unroll
      for (int n = 0; n < D / 16; n++) {  // a product, then 6 (D = 128) of the exponentials' instructions: 3 %
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, 768 / D, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      read_keys(i + 1, y);
      sums(0, p);
      read_values(i, y, 1);
      sums(1, p);
      __builtin_amdgcn_s_setprio(0);
      if (y == 0 || i + 1 < t1) settle(y ? tile_at(i + 1) : k0 + 32, next);
    }
  }
  if (bad) {
    // the values left out above, for the rows that see them: weights are above zero, so
    // they count as they are
#pragma unroll 1
    for (int i = t0; i < t1; i++) {
      const int k0 = tile_at(i);
      if (!cut(k0)) continue;
#pragma unroll 1
      for (int k = k0; k < min(k0 + kK, B.len); k++) {
        const int page = scalar_int(table, k >> a.b.shift);
        if ((unsigned)page >= (unsigned)a.b.pages) continue;
        const bool seen = k <= qpos && (k > qpos - a.window || k < a.sinks);
        const uint16_t* v = a.v + ((((int64_t)page * a.Hkv + j) << a.b.shift) + (k & ((1 << a.b.shift) - 1))) * D + 4 * h;
#pragma unroll
        for (int e = 0; e < D / 32; e++)
#pragma unroll
          for (int u = 0; u < 16; u++) {
            const uint16_t b = v[32 * e + 8 * (u >> 2) + (u & 3)];
            if (seen && (b & 0x7FFF) >= T::kInf) o[e][u] += T::to_f32(b);
          }
      }
    }
  }
  l = xlane_level_sum_f32<6>(l);
  if (row > last_row) return;
  const int64_t at = (int64_t)(B.first + tok) * a.H + head;
  if (B.tiles > a.span) {  // one of several spans: sums, maximum and denominator as they are
    const int64_t slot = at * a.slots + part;
    float* pp = a.part + slot * D + 4 * h;
#pragma unroll
    for (int e = 0; e < D / 32; e++)
#pragma unroll
      for (int n = 0; n < 4; n++)
        *reinterpret_cast<float4*>(pp + 32 * e + 8 * n) = make_float4(o[e][4 * n], o[e][4 * n + 1], o[e][4 * n + 2], o[e][4 * n + 3]);
    if (h == 0) ends_of<D>(a)[slot] = make_float2(m, l);
    return;
  }
  // a row that sees only scores of -inf (l is 0) answers NaN, as the softmax of these
  const float f = l == 0.0f ? NAN : 1.0f / l;
  uint16_t* op = a.out + at * D + 4 * h;
#pragma unroll
  for (int e = 0; e < D / 32; e++)
#pragma unroll
    for (int n = 0; n < 4; n++)
      *reinterpret_cast<uint2*>(op + 32 * e + 8 * n) =
          make_uint2(T::pack(o[e][4 * n] * f, o[e][4 * n + 1] * f), T::pack(o[e][4 * n + 2] * f, o[e][4 * n + 3] * f));
}

constexpr int kStep = 32;  // keys a wave takes at a time below
// Numerators below are 2^7 as large, which sums and denominators share: with kGrow up
// to 2^15, which fp16 holds, and small ones keep 7 bits more.  Their exponents are of
// differences, so that no rounding of a large score is on top of that.
constexpr float kRaise = 7.0f;

// Sequences of few rows (a token or some): one workgroup a span of a sequence's and
// key/value head's keys, all its rows (NR groups of 16) in every wave, the waves
// taking 32 keys in turn.
//   keys     straight to the registers that the product reads: lane 16 g + i has
//            elements 8 g + 32 e .. of key i
//   scores   transposed, s^T = k q^T (mfma 16 x 16 x 32): lane 16 g + r has those of
//            keys 4 g + 0 .. 3 and 16 + 4 g + 0 .. 3 with row r
//   values   by whole rows through registers to the wave's own part of LDS, from
//            where they come transposed as the operand of o^T = v^T p^T, in the
//            order of keys in which the numerators are at hand
// A numerator is two numbers of 16 bits, itself rounded and the rest, with a product for
// each: 2^-22 (fp16) or 2^-16 (bf16) of it is lost, and the output is as near the
// exact one as an f32 softmax's (off by 2.1e-4 instead of 2.6e-4 to 2.9e-4 of it in fp16,
// 1.7e-3 instead of 2.0e-3 to 2.3e-3 in bf16).  The matrix unit has the time: one
// sequence of 700 takes 0.2 us more, others 1 %, 17 to 32 rows 4 %.
// The next keys are asked for when the scores' products have taken the last ones, the
// next values when the last ones are in LDS.
// Bound by memory: 32 sequences of up to 16384 positions, 8 key/value heads of 128, 1 GB
// in 184 us (5.5 TB/s; a copy of 2 GiB runs at 4.9); 8 of 4000 131 MB in 22.6; one of 700
// 6.0, a launch and the chain of loads from the lengths over the pages to the keys; 20 rows each
// of 8 sequences of 4005, with the merge, 32.6 (D = 128: more registers than 256, so one wave a SIMD).
// Eight waves a workgroup instead of four took as long or longer (8 of 4000: 30.7 against
// 27.9 us with the merge of that time), page numbers read ahead into a register, as below,
// 0.2 us longer for one sequence and the same for many.
// lds: few_lds<D, NR> bytes, on a multiple of 16
template <int D, int NR>
constexpr int few_sums = 4 * NR * 16 * (D + 4) * 4 > 4 * kStep * D * 2 ? 4 * NR * 16 * (D + 4) * 4 : 4 * kStep * D * 2;
template <int D, int NR>
constexpr int few_lds = few_sums<D, NR> + 4 * NR * 16 * 8;

template <class T, int D, int NR>
__device__ __forceinline__ void few_block(const AttendArgs& a, int block, int part, uint8_t* lds) {
  constexpr int NW = 4;                 // waves
  constexpr int NC = D / 8;             // 16-byte pieces of a row
  constexpr int RL = 64 / NC;           // rows a load of values
  constexpr int NV = kStep / RL;        // loads of values a step
  constexpr int VB = kStep * D * 2;     // bytes of a step's values
  constexpr int RS = D + 4;             // floats of a row of sums in LDS, so that rows spread over the banks
  float2(*ends)[NR * 16] = reinterpret_cast<float2(*)[NR * 16]>(lds + few_sums<D, NR>);  // of each wave
  const int t = threadIdx.x, ln = t & 63, i16 = ln & 15, g = ln >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int seq = block / a.Hkv, j = block % a.Hkv;
  Block B;
  if (!find_block<kStep>(a, seq, 0, NR * 16, B) || B.n * a.G > a.few) return;
  const int t0 = part * a.few_span, t1 = min(t0 + a.few_span, B.tiles);
  if (t0 >= t1) return;
  const int rows = B.n * a.G;
  auto step_at = [&](int i) { return (i < B.na ? i : B.b0 + i - B.na) * kStep; };

  // this lane's rows: token and head, and the queries
  int qpos[NR];
  u32x4 qv[NR][D / 32];
#pragma unroll
  for (int n = 0; n < NR; n++) {
    const int r = min(16 * n + i16, rows - 1), tok = r / a.G;
    qpos[n] = B.len - B.n + tok;
    const uint16_t* qp = a.q + (int64_t)(B.first + tok) * a.qs[0] + (j * a.G + r - tok * a.G) * a.qs[1] + 8 * g;
#pragma unroll
    for (int e = 0; e < D / 32; e++) {
      u32x4 x = *reinterpret_cast<const u32x4*>(qp + 32 * e);
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = (x[i] & a.keep) ^ a.flip;
      qv[n][e] = x;
    }
  }
  float4v o[NR][D / 16];
  float m[NR], l[NR];
#pragma unroll
  for (int n = 0; n < NR; n++) {
    m[n] = -INFINITY;
    l[n] = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 16; e++) o[n][e] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const float grow = kGrow / a.c;

  const int* table = a.b.table + (int64_t)seq * a.b.W;
  const int last_page = (B.len - 1) >> a.b.shift, in_page = (1 << a.b.shift) - 1;
  // the buffers of 16 rows from k0 on, which lie in one page; rows past the last, and
  // those of a page outside the cache, read as zeros
  auto buffer = [&](const uint16_t* base, int k0) {
    const int page = scalar_int(table, min(k0 >> a.b.shift, last_page));
    const bool there = (unsigned)page < (unsigned)a.b.pages;
    const int bytes = there ? __builtin_amdgcn_readfirstlane(max(min(B.len - k0, 16), 0)) * (D * 2) : 0;
    const int64_t at = ((((int64_t)(there ? page : 0) * a.Hkv + j) << a.b.shift) + (k0 & in_page)) * D;
    return __builtin_amdgcn_make_buffer_rsrc((void*)(base + at), (short)0, bytes, 0x00020000);
  };
  u32x4 kv[2][D / 32], vv[NV];
  const int k_off = i16 * (D * 2) + g * 16, v_off = ln * 16;
  auto load_keys = [&](int k0) {
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const __amdgpu_buffer_rsrc_t r = buffer(a.k, k0 + 16 * x);
#pragma unroll
      for (int e = 0; e < D / 32; e++) kv[x][e] = __builtin_amdgcn_raw_buffer_load_b128(r, k_off + 64 * e, 0, 0);
    }
  };
  auto load_values = [&](int k0) {
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const __amdgpu_buffer_rsrc_t r = buffer(a.v, k0 + 16 * x);
#pragma unroll
      for (int n = 0; n < NV / 2; n++) vv[x * (NV / 2) + n] = __builtin_amdgcn_raw_buffer_load_b128(r, v_off + 1024 * n, 0, 0);
    }
  };
  uint8_t* vs = lds + wave * VB;
  int vw[2], vf;  // LDS offsets of the values' pieces (even and odd loads) and of this lane's part of a fragment
#pragma unroll
  for (int n = 0; n < 2; n++) vw[n] = few_place<D>(n * RL + ln / NC, ln % NC) - n * 1024;
  const int fr = 4 * g + (i16 >> 2);

  int k0 = step_at(min(t0 + wave, t1 - 1));
  if (t0 + wave < t1) {
    load_keys(k0);
    load_values(k0);
  }
  for (int i = t0 + wave; i < t1; i += NW) {
    const int next = i + NW < t1 ? step_at(i + NW) : -1;
    const bool all = k0 + kStep - 1 <= B.lo && k0 > B.hi - a.window;
    u16x2 most = 0;
#pragma unroll
    for (int n = 0; n < NV; n++) most = magnitudes8(most, make_uint4(vv[n][0], vv[n][1], vv[n][2], vv[n][3]));
    const bool bad = __ballot(max(most.x, most.y) >= T::kInf) != 0;  // an infinity or NaN among the step's values
#pragma unroll
    for (int n = 0; n < NV; n++) *reinterpret_cast<u32x4*>(vs + vw[n & 1] + n * 1024) = vv[n];
    if (next >= 0) load_values(next);
    float4v x[NR][2];
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
      for (int y = 0; y < 2; y++) {
        x[n][y] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < D / 32; e++) x[n][y] = T::mfma16(kv[y][e], qv[n][e], x[n][y]);
      }
    if (next >= 0) load_keys(next);
    uint32_t p[NR][4], rest[NR][4];
#pragma unroll
    for (int n = 0; n < NR; n++) {
      if (!all) {
        const int from = qpos[n] - a.window;
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int key = k0 + 16 * y + 4 * g + e;
            const bool near = key > from, sink = key < a.sinks;
            if (key > qpos[n] || !(near || sink)) x[n][y][e] = -INFINITY;
          }
      }
      float mx = fmaxf(fmaxf(fmaxf(x[n][0][0], x[n][0][1]), fmaxf(x[n][0][2], x[n][0][3])),
                       fmaxf(fmaxf(x[n][1][0], x[n][1][1]), fmaxf(x[n][1][2], x[n][1][3])));
      if (__ballot(mx > m[n] + grow)) {
        mx = xlane_level_max_f32<6>(xlane_level_max_f32<5>(mx));  // the four lanes of a row move alike
        const float z = fmaxf(m[n], mx), f = m[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[n] - z) * a.c);
        l[n] *= f;
#pragma unroll
        for (int e = 0; e < D / 16; e++) o[n][e] *= f;
        m[n] = z;
      }
      const float top = m[n] == -INFINITY ? 0.0f : m[n];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float w0 = __builtin_amdgcn_exp2f(fmaf(x[n][e >> 1][2 * e & 3] - top, a.c, kRaise));
        const float w1 = __builtin_amdgcn_exp2f(fmaf(x[n][e >> 1][(2 * e & 3) + 1] - top, a.c, kRaise));
        p[n][e] = T::pack(w0, w1);
        rest[n][e] = T::pack(w0 - T::to_f32((uint16_t)p[n][e]), w1 - T::to_f32((uint16_t)(p[n][e] >> 16)));
        l[n] = T::add2(rest[n][e], T::add2(p[n][e], l[n]));
      }
    }
    if (bad) {
      // the terms one by one, leaving out those of keys that the row does not see (and an
      // infinity times the two parts of a numerator would be NaN)
#pragma unroll 1
      for (int key = 0; key < kStep; key++) {
        const int y = key >> 4, from_g = (key >> 2) & 3, e = key & 3;
#pragma unroll
        for (int n = 0; n < NR; n++) {
          const uint32_t w0 = y ? p[n][2] : p[n][0], w1 = y ? p[n][3] : p[n][1], w = (e & 2 ? w1 : w0) >> 16 * (e & 1);
          const uint32_t z0 = y ? rest[n][2] : rest[n][0], z1 = y ? rest[n][3] : rest[n][1], z = (e & 2 ? z1 : z0) >> 16 * (e & 1);
          const float wf = __shfl(T::to_f32((uint16_t)w) + T::to_f32((uint16_t)z), i16 + 16 * from_g, 64);
          const int at = k0 + key;
          const bool seen = at <= qpos[n] && (at > qpos[n] - a.window || at < a.sinks);
#pragma unroll
          for (int d = 0; d < D / 16; d++)
#pragma unroll
            for (int z = 0; z < 4; z++) {
              const int el = 16 * d + 4 * g + z;
              const uint16_t vd = *reinterpret_cast<const uint16_t*>(vs + few_place<D>(key, el >> 3) + (el & 7) * 2);
              if (seen) o[n][d][z] = fmaf(wf, T::to_f32(vd), o[n][d][z]);
            }
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < D / 16; e++) {
        vf = few_place<D>(fr, 2 * e + ((i16 & 3) >> 1)) + (i16 & 1) * 8;
        const u32x2 w0 = read_turned(vs + vf), w1 = read_turned(vs + vf + 16 * D * 2);
#pragma unroll
        for (int n = 0; n < NR; n++) {
          o[n][e] = T::mfma16(u32x4{w0.x, w0.y, w1.x, w1.y}, u32x4{p[n][0], p[n][1], p[n][2], p[n][3]}, o[n][e]);
          o[n][e] = T::mfma16(u32x4{w0.x, w0.y, w1.x, w1.y}, u32x4{rest[n][0], rest[n][1], rest[n][2], rest[n][3]}, o[n][e]);
        }
      }
    }
    k0 = next;
  }

  // the waves' sums joined
  __syncthreads();
  float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int n = 0; n < NR; n++) {
    l[n] = xlane_level_sum_f32<6>(xlane_level_sum_f32<5>(l[n]));
    const int r = 16 * n + i16;
    if (g == 0) ends[wave][r] = make_float2(m[n], l[n]);
#pragma unroll
    for (int e = 0; e < D / 16; e++)
      *reinterpret_cast<float4v*>(sums + (wave * NR * 16 + r) * RS + 16 * e + 4 * g) = o[n][e];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < (NR * 16 * NC + 64 * NW - 1) / (64 * NW); n++) {
    const int r = (t + 64 * NW * n) / NC, d = (t + 64 * NW * n) % NC * 8;
    if (r >= rows) continue;
    float mx = -INFINITY, den = 0.0f, acc[8];
#pragma unroll
    for (int w = 0; w < NW; w++) mx = fmaxf(mx, ends[w][r].x);
#pragma unroll
    for (int z = 0; z < 8; z++) acc[z] = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w++) {
      const float2 y = ends[w][r];
      // a wave with scores of -inf only has sums of zero, or the NaN of what it saw
      const float f = y.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((y.x - mx) * a.c);
      den = fmaf(y.y, f, den);
      const float* x = sums + (w * NR * 16 + r) * RS + d;
#pragma unroll
      for (int z = 0; z < 8; z++) acc[z] = fmaf(x[z], f, acc[z]);
    }
    const int tok = r / a.G, head = j * a.G + r - tok * a.G;
    const int64_t at = (int64_t)(B.first + tok) * a.H + head;
    if (B.tiles > a.few_span) {
      const int64_t slot = at * a.slots + part;
      *reinterpret_cast<float4*>(a.part + slot * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(a.part + slot * D + d + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (d == 0) ends_of<D>(a)[slot] = make_float2(mx, den);
    } else {
      // a row that sees only scores of -inf (den is 0) answers NaN, as the softmax of these
      const float f = den == 0.0f ? NAN : 1.0f / den;
      *reinterpret_cast<uint4*>(a.out + at * D + d) =
          make_uint4(T::pack(acc[0] * f, acc[1] * f), T::pack(acc[2] * f, acc[3] * f), T::pack(acc[4] * f, acc[5] * f),
                     T::pack(acc[6] * f, acc[7] * f));
    }
  }
}

template <class T, int D, int NR>
__global__ __launch_bounds__(256) void paged_few_kernel(AttendArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[few_lds<D, NR>];
  few_block<T, D, NR>(a, blockIdx.x, blockIdx.y, lds);
}

template <class T, int D>
__global__ __launch_bounds__(256, 2) void paged_many_kernel(AttendArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[many_lds<D>];
  many_block<T, D>(a, blockIdx.x, blockIdx.y, lds);
}

// Both in one launch, their workgroups side by side: the first kernel waits for
// memory, the second for the matrix unit (31 single tokens and a chunk of 1501
// positions: 74 and 65 us one after the other, 97 together).  Eight workgroups
// at a time, one an XCD, in the proportion of their numbers.
template <class T, int D>
__global__ __launch_bounds__(256, 2) void paged_mixed_kernel(AttendArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[many_lds<D> > few_lds<D, 1> ? many_lds<D> : few_lds<D, 1>];
  const int64_t few = a.few_eights, all = few + a.many_eights, n = blockIdx.x >> 3;
  const int before = (int)(n * few / all), x = blockIdx.x & 7;
  if ((int)((n + 1) * few / all) > before) {
    const int f = before * 8 + x, heads = a.b.S * a.Hkv;
    if (f < heads * a.few_spans) few_block<T, D, 1>(a, f % heads, f / heads, lds);
  } else {
    const int m = (int)(n - before) * 8 + x;
    many_block<T, D>(a, m % (8 * a.per), m / (8 * a.per), lds);
  }
}

// For the first kernel, a workgroup a row (3 to 5 us, a wave a row took up to 7): 16
// bytes a lane, the spans dealt to groups of D / 4 lanes, whose sums meet in LDS.  Everything is asked for at once,
// before it is known how many spans there are: what is none is not looked at.
template <class T, int D>
__global__ __launch_bounds__(256) void paged_few_merge_kernel(AttendArgs a) {
  constexpr int N = 256 / (D / 4);  // groups
  __shared__ float4 sums[N][D / 4];
  const int seq = blockIdx.x / a.Hkv, j = blockIdx.x % a.Hkv, r = blockIdx.y;
  const int t = threadIdx.x, ln = t & 63, grp = t / (D / 4), d = t % (D / 4);
  Block B;
  if (!find_block<kStep>(a, seq, 0, kFewRows, B) || B.n * a.G > a.few || r >= B.n * a.G) return;
  const int tok = r / a.G;
  const int64_t at = (int64_t)(B.first + tok) * a.H + j * a.G + r - tok * a.G;
  float2 y = ends_of<D>(a)[at * a.slots + min(ln, a.slots - 1)];
  const float4* pp = reinterpret_cast<const float4*>(a.part + at * a.slots * D) + d;
  constexpr int U = 4;
  float4 x[U];
#pragma unroll
  for (int u = 0; u < U; u++) x[u] = pp[(int64_t)min(grp + N * u, a.slots - 1) * (D / 4)];
  const int spans = (B.tiles + a.few_span - 1) / a.few_span;
  if (spans <= 1) return;
  if (ln >= spans) y = make_float2(-INFINITY, 0.0f);
  const float m = wave_group_max_f32<64>(y.x);
  // a span with scores of -inf only has sums of zero, or the NaN of what it saw
  const float f = y.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((y.x - m) * a.c);
  const float l = wave_group_sum_f32<64>(y.y * f);
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s0 = grp; s0 - grp < spans; s0 += N * U) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int s = s0 + N * u;
      const float w = __shfl(f, min(s, 63), 64);
      if (s0 != grp && s < spans) x[u] = pp[(int64_t)s * (D / 4)];
      if (s < spans) {
        o.x = fmaf(x[u].x, w, o.x);
        o.y = fmaf(x[u].y, w, o.y);
        o.z = fmaf(x[u].z, w, o.z);
        o.w = fmaf(x[u].w, w, o.w);
      }
    }
  }
  sums[grp][d] = o;
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int n = 1; n < N; n++) {
    const float4 z = sums[n][d];
    o.x += z.x;
    o.y += z.y;
    o.z += z.z;
    o.w += z.w;
  }
  const float inv = l == 0.0f ? NAN : 1.0f / l;
  *reinterpret_cast<uint2*>(a.out + at * D + 4 * d) = make_uint2(T::pack(o.x * inv, o.y * inv), T::pack(o.z * inv, o.w * inv));
}

// For the second, a wave a row: 16 bytes a lane, the spans dealt to groups of D / 4
// lanes; lane s has the maximum and denominator of span s (there are up to 64).
template <class T, int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(AttendArgs a) {
  const int ln = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = (int)(at / a.H), head = (int)(at % a.H);
  if (t >= a.b.T) return;
  constexpr int N = 64 / (D / 4);
  const int grp = ln / (D / 4), d = ln % (D / 4);
  const float4* pp = reinterpret_cast<const float4*>(a.part + at * a.slots * D) + d;
  // (read before it is known how many there are: what is none is not looked at)
  float2 y = ends_of<D>(a)[at * a.slots + min(ln, a.slots - 1)];
  // the row's sequence, and the block that it was in
  const int seq = sequence_of(a.b, t);
  if (seq < 0) return;
  const int r = (t - a.b.scalar_start(seq)) * a.G + head % a.G;
  Block B;
  if (!find_block<kK>(a, seq, r / kQ * kQ, kQ, B) || B.n * a.G <= a.few) return;
  const int spans = (B.tiles + a.span - 1) / a.span;
  if (spans <= 1) return;
  if (ln >= spans) y = make_float2(-INFINITY, 0.0f);
  const float m = wave_group_max_f32<64>(y.x);
  // a span with scores of -inf only has sums of zero, or the NaN of what it saw
  const float f = y.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((y.x - m) * a.c);
  const float l = wave_group_sum_f32<64>(y.y * f);
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  // (all lanes stay to the last round: a weight that lies in a lane that has left reads as 0)
#pragma unroll 2
  for (int s0 = 0; s0 < spans; s0 += N) {
    const int s = s0 + grp;
    const float w = __shfl(f, min(s, 63), 64);
    if (s < spans) {
      const float4 x = pp[(int64_t)s * (D / 4)];
      o.x = fmaf(x.x, w, o.x);
      o.y = fmaf(x.y, w, o.y);
      o.z = fmaf(x.z, w, o.z);
      o.w = fmaf(x.w, w, o.w);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float& z = (&o.x)[i];
    if (D == 64) z = xlane_level_sum_f32<5>(z);
    z = xlane_level_sum_f32<6>(z);
  }
  const float inv = l == 0.0f ? NAN : 1.0f / l;
  if (grp == 0)
    *reinterpret_cast<uint2*>(a.out + at * D + 4 * d) = make_uint2(T::pack(o.x * inv, o.y * inv), T::pack(o.z * inv, o.w * inv));
}

// Which kernels run, and how the keys are split: sequences of up to `few` rows by
// the first kernel (nr groups of 16 rows), in spans of few_span steps, the others by
// the second in spans of `span` tiles.
struct Plan {
  int nr;       // 0: the first kernel does not run
  int64_t few_rows;  // rows of a sequence and key/value head there, at most
  bool many;    // whether the second runs
  int64_t few, few_span, few_spans, blocks, items, per, span, spans, slots, bytes;
};

Plan plan(int64_t T, int64_t S, int64_t H, int64_t Hkv, int64_t D, int64_t max_new, int64_t max_length) {
  Plan p = {};
  const int64_t G = H / Hkv, most = std::min(max_new, T) * G;  // rows of a sequence
  if (most <= kFewRows)
    p.nr = most <= 16 ? 1 : 2;
  else if (S > 1 && G <= kFewRows)
    p.nr = G <= 16 ? 1 : 2;
  p.few = 16 * p.nr;
  p.many = most > p.few;
  p.few_spans = p.spans = 1;
  if (p.nr) {
    p.few_rows = std::min(most, p.few);
    const int64_t steps = aq::ceil_div(max_length, kStep) + 1, pairs = S * Hkv;
    // One span where it is short (up to 12 steps, three a wave: 300 positions of one
    // sequence 7.1 us, 7.5 split and merged; 500 9.2 and 7.8) or the sequences and heads
    // are many (256 of 4000 positions 91 us, 96 in two spans each), but for long ones,
    // whose lengths differ more (256 of up to 16384: 220 us, 187 in 8 spans); else 512
    // workgroups (64 of 4000: 26.0, 26.9 with 1024; 8 of 16000 17.4) of a step a wave at
    // least.  All measured with max_length at the longest sequence.  Spans follow that bound,
    // so far above the lengths, where a captured step has it, fewer of them hold keys: with
    // bounds of the length, 32768 and 131072 one sequence of 700 takes 7.5, 12.2 and 12.5 us, of
    // 2000 7.4, 12.0, 24.0, of 20000 20.3, 22.3, 29.4, 8 of 4000 25.4, 46.0, 46.0, 32 of 8000
    // 184, 186, 193.
    if (steps <= 12 || pairs > 512) p.few_spans = 1;
    else if (pairs >= 256) p.few_spans = steps <= 160 ? 1 : std::min<int64_t>(aq::ceil_div(steps, 64), 64);
    else p.few_spans = std::min<int64_t>({512 / pairs, aq::ceil_div(steps, 4), 64});
    p.few_span = aq::ceil_div(steps, p.few_spans);
    p.few_spans = aq::ceil_div(steps, p.few_span);
  }
  if (p.many) {
    p.blocks = S == 1 ? aq::ceil_div(T * G, kQ) : T * G / kQ + S;
    p.items = p.blocks * Hkv;
    p.per = aq::ceil_div(p.items, 8);
    const int64_t tiles = aq::ceil_div(max_length, kK) + 1;
    p.spans = std::max<int64_t>(1, std::min<int64_t>({512 / p.items, aq::ceil_div(tiles, 8), 64}));
    p.span = aq::ceil_div(tiles, p.spans);
    p.spans = aq::ceil_div(tiles, p.span);
  }
  p.slots = std::max(p.spans, p.few_spans);
  p.bytes = p.slots > 1 ? T * H * p.slots * (D + 2) * 4 : 0;
  return p;
}

bool sizes_ok(int64_t T, int64_t S, int64_t H, int64_t Hkv, int64_t D, int64_t max_new, int64_t max_length) {
  return (D == 64 || D == 128) && T > 0 && T < (1 << 24) && S > 0 && S <= 65535 && Hkv > 0 && H > 0 && H <= 1024 &&
         H % Hkv == 0 && max_new > 0 && max_length > 0 && max_length <= INT32_MAX - 2 * kK && T * (H / Hkv) < (1 << 30);
}

template <class T, int D>
void launch(const AttendArgs& a, const Plan& p, hipStream_t stream) {
  const dim3 few((unsigned)(a.b.S * a.Hkv), (unsigned)p.few_spans), many((unsigned)(8 * p.per), (unsigned)p.spans);
  if (p.nr == 1 && p.many) {
    hipLaunchKernelGGL((paged_mixed_kernel<T, D>), dim3(8u * (a.few_eights + a.many_eights)), dim3(256), 0, stream, a);
  } else {
    if (p.nr == 1) hipLaunchKernelGGL((paged_few_kernel<T, D, 1>), few, dim3(256), 0, stream, a);
    if (p.nr == 2) hipLaunchKernelGGL((paged_few_kernel<T, D, 2>), few, dim3(256), 0, stream, a);
    if (p.many) hipLaunchKernelGGL((paged_many_kernel<T, D>), many, dim3(256), 0, stream, a);
  }
  if (p.few_spans > 1)
    hipLaunchKernelGGL((paged_few_merge_kernel<T, D>), dim3(few.x, (unsigned)p.few_rows), dim3(256), 0, stream, a);
  if (p.spans > 1)
    hipLaunchKernelGGL((paged_merge_kernel<T, D>), dim3((unsigned)aq::ceil_div((int64_t)a.b.T * a.H, 4)), dim3(256), 0, stream, a);
}

}  // namespace

extern "C" int64_t aq_paged_attention_workspace(int64_t T, int64_t S, int64_t H, int64_t Hkv, int64_t D, int64_t max_new,
                                                int64_t max_length) {
  return sizes_ok(T, S, H, Hkv, D, max_new, max_length) ? plan(T, S, H, Hkv, D, max_new, max_length).bytes : -1;
}

extern "C" int aq_paged_attention(const void* q, int dtype, int64_t T, int64_t H, int64_t Hkv, int64_t D,
                                  int64_t q_row, int64_t q_head, const void* k_cache, const void* v_cache, int64_t pages,
                                  int64_t page_size, const int32_t* starts, const int32_t* lengths, int64_t S,
                                  const int32_t* table, int64_t W, int64_t max_new, int64_t max_length, int64_t window,
                                  int64_t sinks, float scale, void* workspace, int64_t ws_bytes, void* out, void* stream) {
  const char* me = "aq_paged_attention";
  AQ_CHECK_ARG(q && k_cache && v_cache && starts && lengths && table && out, "%s: null pointer", me);
  AQ_CHECK_ARG(dtype == AQ_F16 || dtype == AQ_BF16, "%s: dtype %d (fp16 and bf16 supported)", me, dtype);
  AQ_CHECK_ARG(D == 64 || D == 128, "%s: head dim %lld (64 or 128 supported)", me, (long long)D);
  AQ_CHECK_ARG(Hkv > 0 && H > 0 && H <= 1024 && H % Hkv == 0, "%s: H (%lld) must be a multiple of Hkv (%lld)", me, (long long)H,
               (long long)Hkv);
  AQ_CHECK_ARG(sizes_ok(T, S, H, Hkv, D, max_new, max_length),
               "%s: sizes out of range (%lld rows, %lld sequences, at most %lld new, %lld positions of one)", me, (long long)T,
               (long long)S, (long long)max_new, (long long)max_length);
  AQ_CHECK_ARG(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
               "%s: page size %lld (a power of two from 16 to 1024)", me, (long long)page_size);
  AQ_CHECK_ARG(pages > 0 && pages <= INT32_MAX && W > 0 && W <= INT32_MAX / page_size && max_length <= W * page_size,
               "%s: %lld pages, %lld of a sequence for %lld positions", me, (long long)pages, (long long)W, (long long)max_length);
  AQ_CHECK_ARG(window >= 1 && sinks >= 0, "%s: window %lld, %lld sinks", me, (long long)window, (long long)sinks);
  AQ_CHECK_ARG(q_row % 8 == 0 && q_head % 8 == 0, "%s: strides must be multiples of 8", me);
  AQ_CHECK_ARG(((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) % 16 == 0 &&
                   ((uintptr_t)starts | (uintptr_t)lengths | (uintptr_t)table) % 4 == 0,
               "%s: q, the caches and out must be 16-byte aligned", me);
  const Plan p = plan(T, S, H, Hkv, D, max_new, max_length);
  AQ_CHECK_ARG(p.bytes == 0 || (workspace && (uintptr_t)workspace % 16 == 0 && ws_bytes >= p.bytes),
               "%s: workspace of %lld bytes, %lld needed, 16-byte aligned", me, (long long)ws_bytes, (long long)p.bytes);
  // (a grid has fewer than 2^32 threads)
  AQ_CHECK_ARG(p.items <= (1 << 23) / p.spans - 16 && S * Hkv <= (1 << 23) / p.few_spans - 16 && T * H <= (1 << 25),
               "%s: %lld rows of %lld heads, %lld sequences", me, (long long)T, (long long)H, (long long)S);
  AttendArgs a;
  a.b = paged::Batch{starts, lengths, table, (int)T, (int)S, (int)W, (int)pages, __builtin_ctz((unsigned)page_size),
                     (int)std::min<int64_t>(max_new, T), (int)max_length};
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k_cache;
  a.v = (const uint16_t*)v_cache;
  a.qs[0] = q_row;
  a.qs[1] = q_head;
  a.out = (uint16_t*)out;
  a.part = (float*)workspace;
  a.H = (int)H;
  a.G = (int)(H / Hkv);
  a.Hkv = (int)Hkv;
  a.window = (int)std::min<int64_t>(window, max_length);
  a.sinks = (int)std::min<int64_t>(sinks, max_length);
  a.items = (int)p.items;
  a.per = (int)p.per;
  a.few = (int)p.few;
  a.few_span = (int)p.few_span;
  a.few_spans = (int)p.few_spans;
  a.span = (int)p.span;
  a.slots = (int)p.slots;
  a.few_eights = p.nr ? (int)aq::ceil_div(S * Hkv * p.few_spans, 8) : 0;
  a.many_eights = (int)(p.per * p.spans);
  a.c = scale == 0.0f ? 1.0f : fabsf(scale) * 1.44269504f;
  a.keep = scale == 0.0f ? 0u : 0xFFFFFFFFu;
  a.flip = scale < 0.0f ? 0x80008000u : 0u;
  if (dtype == AQ_F16)
    D == 64 ? launch<Half, 64>(a, p, (hipStream_t)stream) : launch<Half, 128>(a, p, (hipStream_t)stream);
  else
    D == 64 ? launch<Bf16, 64>(a, p, (hipStream_t)stream) : launch<Bf16, 128>(a, p, (hipStream_t)stream);
  AQ_LAUNCH_CHECK(me);
  return AQ_OK;
}
