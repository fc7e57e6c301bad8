// aq_logprobs.hip -- log probabilities and ranks of given tokens, entropies and
// the most likely alternatives.
//
// With m = max x, Z = sum e^(x_i - m) and E = sum e^(x_i - m) (x_i - m):
//   log p_t = x_t - m - log Z,   entropy = -sum p log p = log Z - E / Z
// in one pass: where the running maximum m grows by d, Z and E so far become
// Z e^-d and (E - d Z) e^-d.  Parts of a row meet the same way.
//
// The alternatives need no sort of the row.  In each wave, the n-th largest of the
// lanes' maxima is a value that n elements at least reach; the largest of the
// waves' values cuts the row to a short list (a few times n), gathered by the
// lanes whose maxima reach it and ranked by counting.
#include "aq_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kList = 1024;
constexpr int kMaxTop = 64, kMaxParts = 32;
constexpr int kMaxVocab = 1 << 18;
constexpr float kLog2e = 1.4426950408889634f;
// What the pass over a row takes everything below, -inf and NaN too, for: no
// weight beside a logit above it (and rows without one are looked at again).
constexpr float kLow = -1e30f;

typedef unsigned long long u64;

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
  // f(value, index) for this thread's elements, in order of index but for the single one
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int t = threadIdx.x;
    if (t < singles) f(value(single(t)), single(t));
    for (int p = p0 + t; p < p1; p += kThreads) {
      const uint4 w = pieces[p];
#pragma unroll
      for (int i = 0; i < T::E; i++) f(T::get(w, i), lead + p * T::E + i);
    }
  }
};

__device__ __forceinline__ int wave_sum_i32(int v) {
  const int s = wave_incl_scan_i32<64>(v);
  return __builtin_amdgcn_readlane(s, 63);
}

struct Shared {
  u64 list[kList];
  Sums sums[kWaves];
  uint32_t cut[kWaves];
  int scan[kWaves];
  u64 best[kWaves];
  int count;
};

// Sums of two sets of elements joined.  -inf: an empty one, or one of only -inf;
// two of +inf count alike.
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float da = a.m == r.m ? 0.0f : a.m - r.m, db = b.m == r.m ? 0.0f : b.m - r.m;
  const float fa = __builtin_amdgcn_exp2f(da * kLog2e), fb = __builtin_amdgcn_exp2f(db * kLog2e);
  r.z = a.z * fa + b.z * fb;
  r.e = (fa > 0.0f ? fmaf(da, a.z, a.e) * fa : 0.0f) + (fb > 0.0f ? fmaf(db, b.z, b.e) * fb : 0.0f);
  r.before = a.before + b.before;
  return r;
}

__device__ __forceinline__ float shfl_xor_f32(float x, int d) { return __shfl_xor(x, d, 64); }

__device__ __forceinline__ Sums block_join(Shared& s, Sums v) {
  for (int d = 1; d < 64; d *= 2) {
    const Sums o = {shfl_xor_f32(v.m, d), shfl_xor_f32(v.z, d), shfl_xor_f32(v.e, d), 0};
    const int n = v.before;
    v = (threadIdx.x & d) ? join(o, v) : join(v, o);  // the same order in both lanes
    v.before = n;
  }
  v.before = wave_sum_i32(v.before);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.sums[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s.sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; w++) v = join(v, s.sums[w]);
  return v;
}

// The same sums number by number, for parts with a +inf, without a logit above
// kLow, or of a token whose logit is not above kLow.
template <int FMT>
__device__ __forceinline__ Sums exact_sums(Shared& s, const Part<FMT>& r, float own, int token) {
  float m = -INFINITY;
  r.each([&](float x, int) { m = fmaxf(m, x); });
  m = wave_group_max_f32<64>(m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.sums[threadIdx.x >> 6].m = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; w++) m = fmaxf(m, s.sums[w].m);
  Sums v = {m, 0.0f, 0.0f, 0};
  r.each([&](float x, int i) {
    x = fmaxf(x, -INFINITY);
    v.before += x > own || (x == own && i < token);
    if (x == -INFINITY) return;
    const float d = x == m ? 0.0f : x - m, w = __builtin_amdgcn_exp2f(d * kLog2e);
    v.z += w;
    v.e += w > 0.0f ? w * d : 0.0f;
  });
  return block_join(s, v);
}

// The `n` first elements of the part, by falling value and then by index, in
// s.list (fewer if it has fewer); mine: this thread's largest, has: whether it has any.
template <int FMT>
__device__ __forceinline__ int part_top(Shared& s, const Part<FMT>& r, int n, float mine, bool has) {
  typedef Type<FMT> T;
  const int t = threadIdx.x, wave = t >> 6;
  const uint32_t key = has ? key_of(mine) : 0u;
  // the largest value that n of the wave's lanes reach (0: fewer have any); the low
  // bits of 16-bit numbers are all alike
  constexpr int kLowest = FMT == AQ_F32 ? 0 : FMT == AQ_BF16 ? 16 : 13;
  uint32_t cut = 0;
  for (int bit = 31; bit >= kLowest; bit--) {
    const uint32_t c = cut | 1u << bit;
    if (__popcll(__ballot(key >= c)) >= n) cut = c;
  }
  if (cut && !(cut >> 31)) cut |= (1u << kLowest) - 1;
  __syncthreads();
  if ((t & 63) == 0) s.cut[wave] = cut;
  if (t == 0) s.count = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; w++) cut = max(cut, s.cut[w]);
  auto gather = [&](uint32_t low) {  // what has keys of `low` and above; where a lane has none it does not look
    if (key >= low)
      r.each([&](float x, int i) {
        if (key_of(x) >= low) {
          const int at = atomicAdd(&s.count, 1);
          if (at < kList) s.list[at] = entry_of(x, i);
        }
      });
    __syncthreads();
    const int c = s.count;
    __syncthreads();
    return c;
  };
  int c = gather(cut);
  if (c > kList) {  // many at the cut: those above it, then the first ones at it, by index
    if (t == 0) s.count = 0;
    __syncthreads();
    c = gather(cut + 1);
    if (c < n) {
      auto place = [&](int mask, int base) {  // elements base + i of this thread for the bits i
        const int k = __popc(mask);
        const int inc = wave_incl_scan_i32<64>(k);
        if ((t & 63) == 63) s.scan[wave] = inc;
        __syncthreads();
        int at = c + inc - k, all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
          at += w < wave ? s.scan[w] : 0;
          all += s.scan[w];
        }
        for (int m = mask; m && at < n; m &= m - 1) s.list[at++] = (u64)cut << 32 | (uint32_t)~(base + __builtin_ctz(m));
        c = min(c + all, n);
        __syncthreads();
      };
      const int head = r.first ? r.lead : 0;
      place(t < head && key_of(r.value(t)) == cut, t);
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
  }
  if (c > kList) {  // a few lanes hold very many large ones: one by one
    u64 below = ~0ull;
    for (c = 0; c < n; c++) {
      u64 best = 0;
      r.each([&](float x, int i) {
        const u64 e = entry_of(x, i);
        if (e < below && e > best) best = e;
      });
      for (int d = 1; d < 64; d *= 2) best = max(best, (u64)__shfl_xor((unsigned long long)best, d, 64));
      __syncthreads();
      if ((t & 63) == 0) s.best[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; w++) best = max(best, s.best[w]);
      if (t == 0) s.list[c] = best;
      below = best;
    }
    __syncthreads();
    return c;
  }
  // ranked by counting
  u64 mineq[kList / kThreads];
  int place[kList / kThreads];
#pragma unroll
  for (int k = 0; k < kList / kThreads; k++) {
    place[k] = kList;
    if (t + k * kThreads < c) {
      mineq[k] = s.list[t + k * kThreads];
      int at = 0;
      for (int i = 0; i < c; i++) at += s.list[i] > mineq[k];
      place[k] = at;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kList / kThreads; k++)
    if (place[k] < n) s.list[place[k]] = mineq[k];
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

// One workgroup a part of a row (grid: parts, rows).
template <int FMT>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Args a) {
  typedef Type<FMT> T;
  __shared__ Shared s;
  const int row = blockIdx.y, part = blockIdx.x, t = threadIdx.x;
  const Part<FMT> r(a, row, part);
  const int64_t token64 = a.tokens[row];
  const bool valid = token64 >= 0 && token64 < a.V;
  const int token = valid ? (int)token64 : 0;
  const float own = fmaxf(r.value(token), -INFINITY);
  const float own_low = next_below(own);
  const int own_piece = token < r.lead ? -1 : (token - r.lead) / T::E;

  Sums v = {kLow, 0.0f, 0.0f, 0};
  float mine = -INFINITY;  // the largest as it is
  auto add = [&](float x, bool before) {
    mine = fmaxf(mine, x);
    v.before += before;
    x = fmaxf(x, kLow);
    const float m = fmaxf(v.m, x), d = v.m - m, f = __builtin_amdgcn_exp2f(d * kLog2e);
    const float w = __builtin_amdgcn_exp2f((x - m) * kLog2e);
    v.e = fmaf(d, v.z, v.e) * f + w * (x - m);
    v.z = v.z * f + w;
    v.m = m;
  };
  if (t < r.singles) {
    const int i = r.single(t);
    const float x = r.value(i);
    add(x, x > own || (x == own && i < token));
  }
  constexpr int U = 4;  // pieces in flight
  for (int p = r.p0 + t; p < r.p1; p += U * kThreads) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; u++) w[u] = p + u * kThreads < r.p1 ? r.pieces[p + u * kThreads] : T::none();
#pragma unroll
    for (int u = 0; u < U; u++) {
      float x[T::E];
      // before the token's piece, elements equal to it stand before it too
      const float limit = p + u * kThreads < own_piece ? own_low : own;
#pragma unroll
      for (int i = 0; i < T::E; i++) {
        x[i] = T::get(w[u], i);
        mine = fmaxf(mine, x[i]);
        x[i] = fmaxf(x[i], kLow);
        v.before += x[i] > limit;
      }
      float m = v.m;
#pragma unroll
      for (int i = 0; i < T::E; i++) m = fmaxf(m, x[i]);
      const float d = v.m - m, f = __builtin_amdgcn_exp2f(d * kLog2e);
      v.e = fmaf(d, v.z, v.e) * f;
      v.z *= f;
      v.m = m;
#pragma unroll
      for (int i = 0; i < T::E; i++) {
        const float y = x[i] - m, z = __builtin_amdgcn_exp2f(y * kLog2e);
        v.z += z;
        v.e = fmaf(z, y, v.e);
      }
    }
  }
  // elements of the token's own piece that are equal to it and stand before it
  if (own_piece >= r.p0 && own_piece < r.p1 && (own_piece - r.p0) % kThreads == t)
    for (int i = r.lead + own_piece * T::E; i < token; i++) v.before += r.value(i) == own;
  const bool has = t < r.singles || r.p0 + t < r.p1;
  v = block_join(s, v);
  // (also where there is nothing: an empty part joins as one of -inf)
  if (!(v.m > kLow && v.m < INFINITY) || !(own > kLow)) v = exact_sums(s, r, own, token);
  const int c = a.top ? part_top(s, r, a.top, mine, has) : 0;
  if (a.parts == 1) {
    const float log_z = logf(v.z);
    write_row(a, row, v, own, valid, log_z);
    if (t < c) write_top(a, row, t, s.list[t], v, log_z);
    return;
  }
  const int64_t at = (int64_t)row * a.parts + part;
  if (t == 0) a.sums[at] = v;
  if (t < a.top) a.lists[at * a.top + t] = t < c ? s.list[t] : 0;
}

// The parts of a row joined, a workgroup a row.
template <int FMT>
__global__ __launch_bounds__(kThreads) void logprobs_merge_kernel(Args a) {
  __shared__ u64 list[kMaxParts * kMaxTop];
  const int row = blockIdx.x, t = threadIdx.x;
  const int n = a.parts * a.top;
  for (int i = t; i < n; i += kThreads) list[i] = a.lists[(int64_t)row * n + i];
  Sums v = a.sums[(int64_t)row * a.parts];
  for (int p = 1; p < a.parts; p++) v = join(v, a.sums[(int64_t)row * a.parts + p]);
  const float log_z = logf(v.z);
  const int64_t token = a.tokens[row];
  const bool valid = token >= 0 && token < a.V;
  const uint8_t* x = a.logits + row * a.stride + (valid ? token : 0) * Type<FMT>::kSize;
  float own = 0.0f;
  if (FMT == AQ_F32)
    own = *reinterpret_cast<const float*>(x);
  else
    own = FMT == AQ_BF16 ? __builtin_bit_cast(float, (uint32_t)*reinterpret_cast<const uint16_t*>(x) << 16)
                         : (float)bits_to_h(*reinterpret_cast<const uint16_t*>(x));
  write_row(a, row, v, fmaxf(own, -INFINITY), valid, log_z);
  __syncthreads();
  for (int i = t; i < n; i += kThreads) {
    const u64 e = list[i];
    if (!e) continue;
    int at = 0;  // in each list, those before it
    for (int p = 0; p < a.parts && at < a.top; p++) {
      int lo = 0, hi = a.top;
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (list[p * a.top + mid] > e) lo = mid + 1;
        else hi = mid;
      }
      at += lo;
    }
    if (at < a.top) write_top(a, row, at, e, v, log_z);
  }
}

int parts_of(int64_t B, int64_t V, int dtype) {
  const int64_t pieces = V * (dtype == AQ_F32 ? 4 : 2) / 16;
  return (int)std::max<int64_t>(1, std::min<int64_t>({512 / B, pieces / 512, kMaxParts}));
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
