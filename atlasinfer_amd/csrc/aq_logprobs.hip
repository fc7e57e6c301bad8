// aq_logprobs.hip -- log probabilities and ranks of given tokens, entropies and
// the most likely alternatives.
//
// With m = max x, Z = sum e^(x_i - m) and E = sum e^(x_i - m) (x_i - m):
//   log p_t = x_t - m - log Z,   entropy = -sum p log p = log Z - E / Z
// in one pass, each lane with a maximum of its own: where it grows by d, Z and E so
// far become Z e^-d and (E - d Z) e^-d.  Lanes, and parts of a row, meet the same way.
//
// The alternatives need no sort of the row.  The n-th largest of the lanes' maxima is
// a value that n elements at least reach; it cuts the row to a short list (a few more
// than n), which is ranked by counting.
#include "aq_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kHeld = 8;   // pieces that a thread keeps (in LDS): 2048 a workgroup
constexpr int kList = 576;  // places of a wave's list: all that fewer than 64 lanes have is at most 518
constexpr int kMaxTop = 64, kMaxParts = 32;
constexpr int kMaxVocab = 1 << 18;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Where the largest logit of a part has to lie for the pass over it, whose exponents are
// off by the rounding of that times log2(e), 1 at most, until it is put right at the end; a
// part with another largest (all fp16 ones but infinities lie between) is looked at
// again, number by number.
constexpr float kLow = -16777216.0f, kHigh = 16777216.0f;

typedef unsigned long long u64;
typedef u64 u64x2 __attribute__((ext_vector_type(2)));

struct Sums {
  float m, z, e;
  int before;  // elements that stand before the given token
};

struct Args {
  const uint8_t* logits;
  int64_t stride;  // bytes
  const int64_t* tokens;
  float *logprob, *entropy, *top_logprobs;
  int64_t *rank, *top_tokens;
  Sums* sums;  // [B, parts]
  u64* lists;  // [B, parts, top], falling
  int V, top, parts;
};

template <int FMT>
struct Type {
  static constexpr int kSize = FMT == AQ_F32 ? 4 : 2;
  static constexpr int E = 16 / kSize;
  // element i of a piece
  static __device__ __forceinline__ float get(const uint4& w, int i) {
    const uint32_t* p = &w.x;
    if (FMT == AQ_F32) return __builtin_bit_cast(float, p[i]);
    const uint32_t b = p[i >> 1];
    if (FMT == AQ_BF16) return __builtin_bit_cast(float, i & 1 ? b & 0xFFFF0000u : b << 16);
    return (float)bits_to_h((uint16_t)(i & 1 ? b >> 16 : b));
  }
  static __device__ __forceinline__ uint4 none() {  // -inf
    const uint32_t w = FMT == AQ_F32 ? 0xFF800000u : FMT == AQ_BF16 ? 0xFF80FF80u : 0xFC00FC00u;
    return make_uint4(w, w, w, w);
  }
};

// Larger keys for larger numbers (NaN as -inf, -0 as 0), and back.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, fmaxf(x, -INFINITY) + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __builtin_bit_cast(float, k ^ ((uint32_t)((int32_t)~k >> 31) | 0x80000000u));
}
// An element's place in the order: by falling value, then by index.
__device__ __forceinline__ u64 entry_of(float x, int i) { return (u64)key_of(x) << 32 | (uint32_t)~i; }
__device__ __forceinline__ float next_below(float x) {
  const uint32_t k = key_of(x) - 1;
  return of_key(k == 0x7FFFFFFFu ? k - 1 : k);  // below 0 comes -0, which is the same
}

// Logit i of a row that starts on any element, i the same for all lanes: the scalar
// unit reads the word that holds it.
template <int FMT>
__device__ __forceinline__ float scalar_logit(const uint8_t* x, int64_t i) {
  typedef const __attribute__((address_space(4))) uint32_t const_u32;
  const uintptr_t at = (uintptr_t)x + i * Type<FMT>::kSize;
  const uint32_t w = *(const_u32*)(at & ~(uintptr_t)3);
  if (FMT == AQ_F32) return __builtin_bit_cast(float, w);
  const uint16_t b = (uint16_t)(w >> (8 * (at & 2)));
  return FMT == AQ_BF16 ? __builtin_bit_cast(float, (uint32_t)b << 16) : (float)bits_to_h(b);
}
__device__ __forceinline__ int64_t scalar_token(const int64_t* tokens, int row) {
  typedef const __attribute__((address_space(4))) int64_t const_i64;
  return ((const_i64*)(uintptr_t)tokens)[row];
}

// Part of a row: whole 16-byte pieces p0 .. p1 - 1, and up to 2 E - 2 single
// elements before the first and behind the last of the row's.
template <int FMT>
struct Part {
  typedef Type<FMT> T;
  const uint8_t* x;
  const uint4* pieces;
  int V, lead, np, p0, p1, singles, tail0;
  bool first, last;

  __device__ __forceinline__ Part(const Args& a, int row, int part) {
    x = a.logits + row * a.stride;
    V = a.V;
    lead = min((int)((16 - ((uintptr_t)x & 15)) & 15) / T::kSize, V);
    np = (V - lead) / T::E;
    tail0 = lead + np * T::E;
    pieces = reinterpret_cast<const uint4*>(x + lead * T::kSize);
    const int per = (np + a.parts - 1) / a.parts;
    p0 = min(part * per, np);
    p1 = min(p0 + per, np);
    first = part == 0;
    last = part == a.parts - 1;
    singles = (first ? lead : 0) + (last ? V - tail0 : 0);
  }
  // index of the n-th single element
  __device__ __forceinline__ int single(int n) const {
    const int head = first ? lead : 0;
    return n < head ? n : tail0 + n - head;
  }
  __device__ __forceinline__ float value(int i) const {
    if (FMT == AQ_F32) return reinterpret_cast<const float*>(x)[i];
    const uint16_t b = reinterpret_cast<const uint16_t*>(x)[i];
    return FMT == AQ_BF16 ? __builtin_bit_cast(float, (uint32_t)b << 16) : (float)bits_to_h(b);
  }
  // element i, the same for all lanes, by the scalar unit
  __device__ __forceinline__ float scalar_value(int i) const { return scalar_logit<FMT>(x, i); }
};

__device__ __forceinline__ int wave_sum_i32(int v) {
  const int s = wave_incl_scan_i32<64>(v);
  return __builtin_amdgcn_readlane(s, 63);
}

struct Shared {
  uint4 held[kHeld * kThreads];
  __attribute__((aligned(16))) u64 list[kWaves][kList];
  u64 top[kMaxTop];
  Sums sums[kWaves];
  float largest[kWaves];
  uint32_t keys[kThreads];
  int count[kWaves];
  u64 best[kWaves];
};

// f(value, index, whether it is one) for this thread's elements, the wave's lanes
// together; `there`: the part's pieces are in s.held.
template <int FMT, class F>
__device__ __forceinline__ void each(const Shared& s, const Part<FMT>& r, bool there, F f) {
  typedef Type<FMT> T;
  const int t = threadIdx.x, first = __builtin_amdgcn_readfirstlane(t & ~63);
  if (first < r.singles) f(t < r.singles ? r.value(r.single(t)) : -INFINITY, r.single(t), t < r.singles);
  if (there) {
#pragma unroll 1
    for (int p = r.p0 + first, u = 0; p < r.p1; p += kThreads, u++) {
      const uint4 w = s.held[t + u * kThreads];
      const int at = p + (t & 63);
#pragma unroll
      for (int i = 0; i < T::E; i++) f(T::get(w, i), r.lead + at * T::E + i, at < r.p1);
    }
  } else {
#pragma unroll 1
    for (int p = r.p0 + first; p < r.p1; p += kThreads) {
      const int at = p + (t & 63);
      const uint4 w = at < r.p1 ? r.pieces[at] : T::none();
#pragma unroll
      for (int i = 0; i < T::E; i++) f(T::get(w, i), r.lead + at * T::E + i, at < r.p1);
    }
  }
}

// The largest over the workgroup.
__device__ __forceinline__ float block_max(Shared& s, float x) {
  x = wave_group_max_f32<64>(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.largest[threadIdx.x >> 6] = x;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; w++) x = fmaxf(x, s.largest[w]);
  return x;
}

// z, e and before (a wave's count in each of its lanes) summed over the workgroup.
__device__ __forceinline__ Sums block_sum(Shared& s, Sums v) {
  v.z = wave_group_sum_f32<64>(v.z);
  v.e = wave_group_sum_f32<64>(v.e);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.sums[threadIdx.x >> 6] = v;
  __syncthreads();
  v.z = v.e = 0.0f;
  v.before = 0;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    v.z += s.sums[w].z;
    v.e += s.sums[w].e;
    v.before += s.sums[w].before;
  }
  return v;
}

// How many of n numbers (a multiple of 32) are larger than e, counted by four
// neighbouring lanes, which all have e.
__device__ __forceinline__ int count_above(const u64* list, int n, u64 e) {
  int above = 0;
#pragma unroll 1
  for (int i = 2 * (threadIdx.x & 3); i < n; i += 32) {
    u64x2 x[4];
#pragma unroll
    for (int u = 0; u < 4; u++) x[u] = *reinterpret_cast<const u64x2*>(list + i + 8 * u);
#pragma unroll
    for (int u = 0; u < 4; u++) above += (x[u].x > e) + (x[u].y > e);
  }
  above += __builtin_amdgcn_mov_dpp(above, 0xB1, 0xF, 0xF, false);  // quad_perm [1,0,3,2]
  return above + __builtin_amdgcn_mov_dpp(above, 0x4E, 0xF, 0xF, false);  // [2,3,0,1]
}

// Sums number by number, for parts that the pass over them cannot weigh, or where the
// token's logit is -inf: e^(x - m) with the largest exactly 1, +inf too.
template <int FMT>
__device__ __forceinline__ Sums exact_sums(Shared& s, const Part<FMT>& r, bool there, float own, int token) {
  float m = -INFINITY;
  each(s, r, there, [&](float x, int, bool) { m = fmaxf(m, x); });
  m = block_max(s, m);
  Sums v = {m, 0.0f, 0.0f, 0};
  each(s, r, there, [&](float x, int i, bool in) {
    x = fmaxf(x, -INFINITY);
    v.before += __popcll(__ballot(in && (x > own || (x == own && i < token))));
    const float d = x == m ? 0.0f : x - m, w = x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(d * kLog2e);
    v.z += w;
    v.e += w > 0.0f ? w * d : 0.0f;
  });
  return block_sum(s, v);
}

// The `n` first elements of the part, by falling value and then by index, in s.top
// (fewer if it has fewer); mine: this thread's largest, has: whether it has any.
template <int FMT>
__device__ __forceinline__ int part_top(Shared& s, const Part<FMT>& r, bool there, int n, float mine, bool has) {
  typedef Type<FMT> T;
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const uint32_t key = has ? key_of(mine) : 0u;
  // The largest value that n of the lanes reach (0: fewer have any), two bits at a time;
  // the low bits of 16-bit numbers are all alike.  For more than 8 of all lanes, whose
  // keys every wave has; up to 8 of each wave by itself, the largest of the waves'
  // values: a quarter of the work, lists of 4 n (2048 rows of 128256 with n = 5 177 us
  // so, 186 by all lanes; with n = 20 222 and 202, with n = 64 3140 and 279).
  constexpr int kLowest = FMT == AQ_F32 ? 0 : FMT == AQ_BF16 ? 16 : 12;
  auto highest = [&](auto reach) {
    uint32_t c = 0;
#pragma unroll 1
    for (int bit = 30; bit >= kLowest; bit -= 2) {
      const uint32_t c1 = c | 1u << bit, c2 = c | 2u << bit, c3 = c | 3u << bit;
      const int k1 = reach(c1), k2 = reach(c2), k3 = reach(c3);
      c = k3 >= n ? c3 : k2 >= n ? c2 : k1 >= n ? c1 : c;
    }
    return c && !(c >> 31) ? c | ((1u << kLowest) - 1) : c;
  };
  uint32_t cut = 0;
  __syncthreads();
  if (n <= 8) {
    cut = highest([&](uint32_t c) { return __popcll(__ballot(key >= c)); });
    if ((t & 63) == 0) s.keys[wave] = cut;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; w++) cut = max(cut, s.keys[w]);
  } else {
    s.keys[t] = key;
    __syncthreads();
    uint32_t keys[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; w++) keys[w] = s.keys[(t & 63) + 64 * w];
    cut = highest([&](uint32_t c) {
      int k = 0;
#pragma unroll
      for (int w = 0; w < kWaves; w++) k += __popcll(__ballot(keys[w] >= c));
      return k;
    });
  }
  // Each wave lists its elements with keys of `low` and above (where it has one); the
  // second time, where very many are equal to the cut, those above it.
  int c = 0, before = 0;
  bool over = false;
#pragma unroll 1
  for (uint32_t low = cut; low <= cut + 1; low++) {
    const float least = low > key_of(-INFINITY) ? of_key(low) : -INFINITY;
    int k = 0;
    auto list = [&](float x, int i, bool in) {
      const bool take = in && fmaxf(x, -INFINITY) >= least;
      const uint64_t mask = __ballot(take);
      const int at = k + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
      if (take && at < kList) s.list[wave][at] = entry_of(x, i);
      k += __popcll(mask);
    };
    uint64_t reach = __ballot(key >= low);
    if (!there) {
      if (reach) each(s, r, there, list);
    } else {
      // lane by lane of those whose maxima reach it, an element of its pieces a lane
      // (two lanes at once for numbers of 32 bits): 64 rows of 128256 1.6 us less than
      // with every lane walking over its own
      if (wave == 0 && r.singles) list(t < r.singles ? r.value(r.single(t)) : -INFINITY, r.single(min(t, r.singles - 1)), t < r.singles);
      constexpr int kAtOnce = 64 / (kHeld * T::E);
      const int ln = t & 63, u = ln / T::E % kHeld, el = ln % T::E, half = ln / (kHeld * T::E);
      const uint8_t* from = reinterpret_cast<const uint8_t*>(s.held) + (wave * 64 + u * kThreads) * 16 + el * T::kSize;
#pragma unroll 1
      while (reach) {
        constexpr int U = 4;
        int src[U];
        float x[U];
#pragma unroll
        for (int n = 0; n < U; n++) {
          src[n] = reach ? __builtin_ctzll(reach) : -1;
          reach &= reach - 1;
          if (kAtOnce == 2) {
            const int other = reach ? __builtin_ctzll(reach) : -1;
            reach &= reach - 1;
            src[n] = half ? other : src[n];
          }
          const uint8_t* at = from + max(src[n], 0) * 16;
          if (FMT == AQ_F32) x[n] = *reinterpret_cast<const float*>(at);
          else if (FMT == AQ_BF16) x[n] = __builtin_bit_cast(float, (uint32_t)*reinterpret_cast<const uint16_t*>(at) << 16);
          else x[n] = (float)bits_to_h(*reinterpret_cast<const uint16_t*>(at));
        }
#pragma unroll
        for (int n = 0; n < U; n++) {
          const int piece = r.p0 + wave * 64 + src[n] + u * kThreads;
          list(x[n], r.lead + piece * T::E + el, src[n] >= 0 && piece < r.p1);
        }
      }
    }
    __syncthreads();
    if ((t & 63) == 0) s.count[wave] = k;
    __syncthreads();
    c = before = 0;
    over = false;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      before += w < wave ? s.count[w] : 0;
      c += s.count[w];
      over |= s.count[w] > kList;
    }
    if (!over) break;
  }
  if (over) {  // a few lanes hold very many large ones: one by one
    u64 below = ~0ull;
#pragma unroll 1
    for (c = 0; c < n; c++) {
      u64 best = 0;
      each(s, r, there, [&](float x, int i, bool in) {
        const u64 e = entry_of(x, i);
        if (in && e < below && e > best) best = e;
      });
#pragma unroll 1
      for (int d = 1; d < 64; d *= 2) best = max(best, (u64)__shfl_xor((unsigned long long)best, d, 64));
      __syncthreads();
      if ((t & 63) == 0) s.best[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; w++) best = max(best, s.best[w]);
      if (t == 0) s.top[c] = best;
      below = best;
    }
    __syncthreads();
    return c;
  }
  // the waves' lists as one, where the pieces were; behind it zeros, which nothing is below
  u64* list = reinterpret_cast<u64*>(s.held);
  const int mine_n = s.count[wave];
  for (int i = t & 63; i < mine_n; i += 64) list[before + i] = s.list[wave][i];
  if (c < n) {
    // the first ones at the cut, by index
    const int head = r.first ? r.lead : 0;
    auto place = [&](int mask, int base) {  // elements base + i of this thread for the bits i
      const int k = __popc(mask);
      const int inc = wave_incl_scan_i32<64>(k);
      __syncthreads();
      if ((t & 63) == 63) s.count[wave] = inc;
      __syncthreads();
      int to = c + inc - k, all = 0;
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        to += w < wave ? s.count[w] : 0;
        all += s.count[w];
      }
      for (int m = mask; m && to < n; m &= m - 1) list[to++] = (u64)cut << 32 | (uint32_t)~(base + __builtin_ctz(m));
      c = min(c + all, n);
    };
    place(t < head && key_of(r.value(t)) == cut, t);
#pragma unroll 1
    for (int p = r.p0; p < r.p1 && c < n; p += kThreads) {
      int mask = 0;
      if (p + t < r.p1) {
        const uint4 w = r.pieces[p + t];
#pragma unroll
        for (int i = 0; i < T::E; i++) mask |= (key_of(T::get(w, i)) == cut) << i;
      }
      place(mask, r.lead + (p + t) * T::E);
    }
    if (r.last && c < n) place(t < r.V - r.tail0 && key_of(r.value(min(r.tail0 + t, r.V - 1))) == cut, r.tail0 + t);
  }
  const int padded = (c + 31) & ~31;
  if (t < padded - c) list[c + t] = 0;
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < c; k += kThreads / 4) {  // four lanes an element
    const u64 e = list[min(k + t / 4, c - 1)];
    const int at = count_above(list, padded, e);
    if (at < n) s.top[at] = e;
  }
  __syncthreads();
  return min(c, n);
}

__device__ __forceinline__ void write_row(const Args& a, int row, const Sums& v, float own, bool valid, float log_z) {
  if (threadIdx.x == 0) {
    // a row without a logit above -inf has no probabilities
    const bool some = v.m > -INFINITY;
    a.logprob[row] = valid && some ? (own == v.m ? 0.0f : own - v.m) - log_z : NAN;
    a.entropy[row] = some ? log_z - v.e / v.z : NAN;
    a.rank[row] = valid ? v.before : -1;
  }
}
__device__ __forceinline__ void write_top(const Args& a, int row, int at, u64 e, const Sums& v, float log_z) {
  const float x = of_key((uint32_t)(e >> 32));
  a.top_tokens[(int64_t)row * a.top + at] = (int64_t)(int)~(uint32_t)e;
  a.top_logprobs[(int64_t)row * a.top + at] = v.m > -INFINITY ? (x == v.m ? 0.0f : x - v.m) - log_z : NAN;
}

// One workgroup a part of a row (grid: parts, rows).  2048 rows of 128256 fp16: 132
// to 138 us without alternatives (525 MB at 3.9 TB/s; the library's row maximum takes 126), 204
// with 20, 278 with 64: memory, and 12.6, 18.2 and 23.1 vector instructions an element by
// counters (9.5 of them the pass, an exponential among these).  As many fp32 logits: 204, 375,
// 572.  64 rows: 11.9 and 4.1 for the merge, steps one after the other: the row's loads 2
// to 3, the pass 2.5, sums, cut, list and ranks 5.
template <int FMT>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Args a) {
  typedef Type<FMT> T;
  __shared__ Shared s;
  const int row = blockIdx.y, part = blockIdx.x, t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Part<FMT> r(a, row, part);
  // a thread's pieces, and its single element, are asked for at once
  uint4 held[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; u++) held[u] = r.p0 + t + u * kThreads < r.p1 ? r.pieces[r.p0 + t + u * kThreads] : T::none();
  const float single = t < r.singles ? r.value(r.single(t)) : -INFINITY;
  const int64_t token64 = scalar_token(a.tokens, row);
  const bool valid = token64 >= 0 && token64 < a.V;
  const int token = valid ? (int)token64 : 0;
  const float own = fmaxf(r.scalar_value(token), -INFINITY);
  const float own_low = next_below(own);
  const int own_piece = token < r.lead ? -1 : (token - r.lead) / T::E;

  // Exponents of 2: t = x log2(e) - m2, m2 about m log2(e), which every term shares, so
  // that its rounding is put right at the end.  Counts are the wave's, by the
  // scalar unit.
  float m = kLow, m2 = kLow * kLog2e, mine = -INFINITY;  // mine: the largest as it is
  Sums v = {0.0f, 0.0f, 0.0f, 0};
  auto weigh = [&](float x) {
    const float y = fmaxf(fmaf(x, kLog2e, -m2), -150.0f), w = __builtin_amdgcn_exp2f(y);  // NaN, -inf: 0
    v.z += w;
    v.e = fmaf(w, y, v.e);
  };
  auto raise = [&](float largest) {
    mine = fmaxf(mine, largest);
    m = fmaxf(m, largest);
    const float n2 = m * kLog2e, d = m2 - n2, f = __builtin_amdgcn_exp2f(d);
    v.e = fmaf(d, v.z, v.e) * f;
    v.z *= f;
    m2 = n2;
  };
  const bool there = r.p1 - r.p0 <= kHeld * kThreads;
#pragma unroll
  for (int u = 0; u < kHeld; u++) s.held[t + u * kThreads] = held[u];
  if (wave == 0 && r.singles) {
    raise(single);
    if (t < r.singles) weigh(single);
    v.before += __popcll(__ballot(t < r.singles && (single > own || (single == own && r.single(t) < token))));
  }
  auto add = [&](const uint4& w, int p) {
    float x[T::E], largest = -INFINITY;
    // before the token's piece, elements equal to it stand before it too
    const float limit = p < own_piece ? own_low : own;
#pragma unroll
    for (int i = 0; i < T::E; i++) {
      x[i] = T::get(w, i);
      largest = fmaxf(largest, x[i]);
    }
    raise(largest);
#pragma unroll
    for (int i = 0; i < T::E; i++) {
      weigh(x[i]);
      v.before += __popcll(__ballot(x[i] > limit));
    }
  };
#pragma unroll 1
  for (int u = 0; u < kHeld && r.p0 + wave * 64 + u * kThreads < r.p1; u++) add(s.held[t + u * kThreads], r.p0 + t + u * kThreads);
#pragma unroll 1
  for (int p = r.p0 + wave * 64 + kHeld * kThreads; p < r.p1; p += kThreads) {
    const int at = p + (t & 63);
    add(at < r.p1 ? r.pieces[at] : T::none(), at);
  }
  // elements of the token's own piece that are equal to it and stand before it
  if (own_piece >= r.p0 && own_piece < r.p1 && (own_piece - r.p0) % kThreads / 64 == wave)
    for (int i = r.lead + own_piece * T::E; i < token; i++) v.before += r.scalar_value(i) == own;
  const bool has = t < r.singles || r.p0 + t < r.p1;
  const float all = block_max(s, m);
  if (!(all > kLow && all < kHigh) || own == -INFINITY) {  // (nothing at all, too: it counts as -inf)
    v = exact_sums(s, r, there, own, token);
  } else {
    m = all;
    const float n2 = m * kLog2e, d = m2 - n2, f = __builtin_amdgcn_exp2f(d);
    v.e = fmaf(d, v.z, v.e) * f;
    v.z *= f;
    v = block_sum(s, v);
    // from n2 to the maximum itself, which is off by the rounding of their product
    const float off = fmaf(m, kLog2e, -n2), g = __builtin_amdgcn_exp2f(-off);
    v.e = (v.e - off * v.z) * g * kLn2;
    v.z *= g;
    v.m = m;
  }
  const int c = a.top ? part_top(s, r, there, a.top, mine, has) : 0;
  if (a.parts == 1) {
    const float log_z = logf(v.z);
    write_row(a, row, v, own, valid, log_z);
    if (t < c) write_top(a, row, t, s.top[t], v, log_z);
    return;
  }
  const int64_t at = (int64_t)row * a.parts + part;
  if (t == 0) a.sums[at] = v;
  if (t < a.top) a.lists[at * a.top + t] = t < c ? s.top[t] : 0;
}

// The parts of a row joined, a workgroup a row; lane p has the sums of part p.
template <int FMT>
__global__ __launch_bounds__(kThreads) void logprobs_merge_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) u64 list[kMaxParts * kMaxTop];
  const int row = blockIdx.x, t = threadIdx.x, ln = t & 63;
  const int n = a.parts * a.top;
  const Sums mine = a.sums[(int64_t)row * a.parts + min(ln, a.parts - 1)];
  for (int i = t; i < n; i += kThreads) list[i] = a.lists[(int64_t)row * n + i];
  if (t < 32 && n + t < kMaxParts * kMaxTop) list[n + t] = 0;
  const int64_t token = scalar_token(a.tokens, row);
  const bool valid = token >= 0 && token < a.V;
  const float own = fmaxf(scalar_logit<FMT>(a.logits + row * a.stride, valid ? token : 0), -INFINITY);
  Sums v = ln < a.parts ? mine : Sums{-INFINITY, 0.0f, 0.0f, 0};
  const float m = wave_group_max_f32<64>(v.m), d = v.m == m ? 0.0f : v.m - m, f = __builtin_amdgcn_exp2f(d * kLog2e);
  v.e = wave_group_sum_f32<64>(f > 0.0f ? fmaf(d, v.z, v.e) * f : 0.0f);
  v.z = wave_group_sum_f32<64>(v.z * f);
  v.before = wave_sum_i32(v.before);
  v.m = m;
  const float log_z = logf(v.z);
  write_row(a, row, v, own, valid, log_z);
  __syncthreads();
  const int padded = (n + 31) & ~31;
#pragma unroll 1
  for (int k = 0; k < n; k += kThreads / 4) {  // four lanes an entry
    const u64 e = list[min(k + t / 4, n - 1)];
    const int at = count_above(list, padded, e);
    if (e && at < a.top && (t & 3) == 0 && k + t / 4 < n) write_top(a, row, at, e, v, log_z);
  }
}

// Parts whose pieces the threads can hold (up to 32 of 2048), and more for few rows: as
// many as make 512 workgroups, of 512 pieces each at least.
int parts_of(int64_t B, int64_t V, int dtype) {
  const int64_t pieces = V * (dtype == AQ_F32 ? 4 : 2) / 16;
  return (int)std::max<int64_t>({1, aq::ceil_div(pieces, kHeld * kThreads), std::min<int64_t>({512 / B, pieces / 512, kMaxParts})});
}

bool sizes_ok(int64_t B, int64_t V, int dtype, int64_t top) {
  return B > 0 && B <= 65535 && V > 0 && V <= kMaxVocab && dtype >= AQ_F16 && dtype <= AQ_F32 && top >= 0 && top <= kMaxTop && top <= V;
}

}  // namespace

extern "C" int64_t aq_token_logprobs_workspace(int64_t B, int64_t V, int dtype, int64_t top) {
  if (!sizes_ok(B, V, dtype, top)) return -1;
  const int64_t parts = parts_of(B, V, dtype);
  return parts > 1 ? B * parts * (int64_t)(sizeof(Sums) + 8 * top) : 0;
}

extern "C" int aq_token_logprobs(const void* logits, int dtype, int64_t B, int64_t V, int64_t stride, const int64_t* tokens,
                                 int64_t top, float* logprobs, float* entropies, int64_t* ranks, float* top_logprobs,
                                 int64_t* top_tokens, void* workspace, int64_t ws_bytes, void* stream) {
  const char* me = "aq_token_logprobs";
  AQ_CHECK_ARG(logits && tokens && logprobs && entropies && ranks && (top == 0 || (top_logprobs && top_tokens)), "%s: null pointer", me);
  AQ_CHECK_ARG(dtype == AQ_F16 || dtype == AQ_BF16 || dtype == AQ_F32, "%s: dtype %d", me, dtype);
  AQ_CHECK_ARG(V > 0 && V <= kMaxVocab, "%s: %lld logits a row (1 .. %d)", me, (long long)V, kMaxVocab);
  AQ_CHECK_ARG(B > 0 && B <= 65535 && (stride >= V || B == 1) && stride >= 0, "%s: %lld rows, %lld elements apart", me, (long long)B,
               (long long)stride);
  AQ_CHECK_ARG(top >= 0 && top <= kMaxTop && top <= V, "%s: %lld alternatives (0 .. %d, at most a row's logits)", me, (long long)top,
               kMaxTop);
  const int size = dtype == AQ_F32 ? 4 : 2;
  AQ_CHECK_ARG((uintptr_t)logits % size == 0 && ((uintptr_t)logprobs | (uintptr_t)entropies | (uintptr_t)top_logprobs) % 4 == 0 &&
                   ((uintptr_t)tokens | (uintptr_t)ranks | (uintptr_t)top_tokens) % 8 == 0,
               "%s: misaligned buffer", me);
  AQ_CHECK_ARG((uintptr_t)workspace % 16 == 0, "%s: the workspace must be 16-byte aligned", me);
  Args a;
  a.parts = parts_of(B, V, dtype);
  const int64_t need = a.parts > 1 ? B * a.parts * (int64_t)(sizeof(Sums) + 8 * top) : 0;
  if (!workspace || ws_bytes < need) a.parts = 1;
  a.logits = (const uint8_t*)logits;
  a.stride = stride * size;
  a.tokens = tokens;
  a.logprob = logprobs;
  a.entropy = entropies;
  a.rank = ranks;
  a.top_logprobs = top_logprobs;
  a.top_tokens = top_tokens;
  a.sums = (Sums*)workspace;
  a.lists = (u64*)((uint8_t*)workspace + B * a.parts * (int64_t)sizeof(Sums));
  a.V = (int)V;
  a.top = (int)top;
  const dim3 grid((unsigned)a.parts, (unsigned)B);
  const hipStream_t st = (hipStream_t)stream;
#define AQ_RUN(F)                                                                                       \
  hipLaunchKernelGGL((logprobs_kernel<F>), grid, dim3(kThreads), 0, st, a);                             \
  if (a.parts > 1) hipLaunchKernelGGL((logprobs_merge_kernel<F>), dim3((unsigned)B), dim3(kThreads), 0, st, a)
  if (dtype == AQ_F16) {
    AQ_RUN(AQ_F16);
  } else if (dtype == AQ_BF16) {
    AQ_RUN(AQ_BF16);
  } else {
    AQ_RUN(AQ_F32);
  }
#undef AQ_RUN
  AQ_LAUNCH_CHECK(me);
  return AQ_OK;
}
