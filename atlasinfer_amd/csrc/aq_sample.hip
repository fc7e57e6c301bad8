// aq_sample.hip -- the next token of every sequence from its logits and one
// given random number: temperature, top-k, top-p, min-p.
//
// The mathematics.  Tokens in the order of falling logit, equal ones by index;
// w_i = exp((x_i - max) / T).  Every filter keeps a beginning of that order:
// the first k; of those the tokens before which less than p of their mass
// lies; the tokens of w >= min_p.  So the kept set is known by one key (the
// last logit kept) and the number of its ties kept -- the cut -- and min_p.  The
// token is the first kept one, by index, whose running mass passes u times the
// kept mass.
//
// Masses are whole numbers, w rounded to 2^-42 (V <= 2^18 of them stay below
// 2^61): sums do not depend on their order, so the same call gives the same
// token on every run, however the work is dealt.  The exponentials are taken in
// 64 bits: with V tokens there are V borders a random number can fall beside,
// and errors of 2^-24 in the sums would choose another token in one row of a
// hundred where tens of thousands are kept.
//
// One workgroup takes a row (long rows of few are split, see below).  A full sort is
// never made:
//   max      one pass, 16 bytes a thread and load, packed maxima
//   top-k    (k <= 512) of the 1024 threads' own maxima the k-th largest is a
//            key that at least k tokens reach; the tokens that do (k and a few,
//            for logits in any order) go to a list in LDS, which is the whole rest
//            where it has up to 256
//   cuts     2048 bins by how far a logit lies below the maximum, counts and
//            masses: the bin in which the running count reaches k, or the running
//            mass p, then the order of its members.  Up to 256 are compared with each
//            other, four threads a member; more (ties, high temperatures) are ordered
//            by the bits of their keys, 11 at a time, with the same histograms.
//            (Bins by the keys' own first bits fall on the few exponents that most
//            logits share: nearly every row went through all bits, top-p of 256 fp32
//            rows of 32000 took 53 us, here 46; of one fp16 row of 50272 40, here 35.)
//   token    kept masses by segments of 1 KiB, summed in the pass that lists the
//            bin's members; one wave goes through the segment that the number falls in
//
// Bound by instructions: an exponential is 30 of them, a pass over 32 tokens a thread
// 10 to 15 us, and what every call does once (finding a bin, ordering a list, the last
// segment) 2 to 4 us a step; reading the row is a tenth of it.
// Passes are short loops over the row in memory (the L2 has it after the first):
// with every element of a thread unrolled, and kept in registers, the kernel was
// 20 000 instructions long, ran once through them and took 25 us for a greedy row
// of 50272, most of it waiting for instructions.  (Four tokens at a time in a thread: no
// faster, 5 us slower where it spilled.)
#include "aq_common.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;  // 11 bits
constexpr int64_t kMaxVocab = 1 << 18;
constexpr double kOne = 4398046511104.0;  // 2^42
constexpr int kList = 4096;
constexpr int kSmallList = kThreads / 4;
constexpr int kTable = 512;
constexpr int kMaxParts = 32;
constexpr int kMaxListK = 512;
constexpr int kMaxSegments = 1024 + 16;  // 2^18 f32 and a misaligned start

struct Settings {
  const float *t, *p, *m;
  const int* k;
  float t0, p0, m0;
  int k0;
};

// A logit's key: its bits as a signed number (so that -0 and 0 are one), moved
// up until -inf is the lowest and infinity the highest key there is; NaNs wrap
// below -inf and are raised to it.
template <int FMT>
struct Logit {
  static constexpr int kBits = FMT == AQ_F32 ? 32 : 16;
  static constexpr int kPer = FMT == AQ_F32 ? 4 : 8;  // elements of a 16-byte piece
  static constexpr uint32_t kSign = 1u << (kBits - 1);
  static constexpr uint32_t kInf = FMT == AQ_F16 ? 0x7C00u : FMT == AQ_BF16 ? 0x7F80u : 0x7F800000u;
  static constexpr uint32_t kUp = kSign - 1 - kInf;
  static constexpr uint32_t kLowest = 2 * kUp + 1;  // key of -inf

  static __device__ __forceinline__ float value(uint32_t b) {
    if (FMT == AQ_F16) return (float)bits_to_h((uint16_t)b);
    return __builtin_bit_cast(float, FMT == AQ_BF16 ? b << 16 : b);
  }
  static __device__ __forceinline__ uint32_t bits_of_key(uint32_t key) {
    const int32_t s = (int32_t)(key - kSign - kUp);
    return s >= 0 ? (uint32_t)s : kSign | (uint32_t)-s;
  }
  static __device__ __forceinline__ float value_of_key(uint32_t key) { return value(bits_of_key(key)); }
};

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));

// Keys of the two 16-bit logits of a word, or of one 32-bit logit.
template <int FMT>
__device__ __forceinline__ uint32_t keys_of_word(uint32_t w) {
  typedef Logit<FMT> L;
  if constexpr (FMT == AQ_F32) {
    const uint32_t g = (uint32_t)((int32_t)w >> 31);
    return max((((w & 0x7FFFFFFFu) ^ g) - g) + (L::kSign + L::kUp), L::kLowest);
  } else {
    const i16x2 g = __builtin_bit_cast(i16x2, w) >> 15;
    const u16x2 gu = __builtin_bit_cast(u16x2, g);
    u16x2 k = (__builtin_bit_cast(u16x2, w & 0x7FFF7FFFu) ^ gu) - gu;
    k = k + (uint16_t)(L::kSign + L::kUp);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(k, (u16x2)((uint16_t)L::kLowest)));
  }
}

// exp((x - mx) / T) in units of 2^-42, rounded to a whole number: 2^(n / 512)
// 2^(r / 512) with y = n + r, y = (x - mx) c, c = 512 log2(e) / T, from a table of
// 2^(j / 512 + 42) and a polynomial of degree 3 (|r| <= 1/2: relative error 1e-14).
// Adding 1.5 2^52 to y rounds it to n and leaves n in the low bits; its upper part
// goes to the exponent; the last product is added to 2^52, which rounds it and
// leaves it in the low bits.  (Conversions between 64 bits and whole numbers, and
// rndne and ldexp, take four times as long as an addition.)  x is taken from lo
// on, where the weight is 2^-60 or less, and -inf and NaN with it.
struct Weigh {
  static constexpr double kMagic = 6755399441055744.0;  // 1.5 2^52
  double mx, c;
  const double* table;
  float lo, hi;
  // 0: a row with infinities: these weigh 1 and every number nothing; 1/2: one of large
  // negative numbers, taken by their halves (exact), mx, lo and hi too, so that there are
  // numbers below the lowest that weighs something; 1: every other (then `other` is 0)
  float factor;
  int other;
  // d = x - mx and t = y + 1.5 2^52
  __device__ __forceinline__ void step(float x, double* d, double* t) const {
    if (other) {
      asm volatile("");  // a branch, which few rows take
      x = x == INFINITY ? hi : x * factor;
    }
    *d = (double)__builtin_amdgcn_fmed3f(x, lo, hi) - mx;
    *t = fma(*d, c, kMagic);
  }
  __device__ __forceinline__ uint64_t weight(double d, double t) const {
    constexpr double a = 0.0013538030870311431, a2 = a * a / 2, a3 = a * a * a / 6;  // ln 2 / 512
    constexpr double one = 4503599627370496.0;
    const double r = fma(d, c, kMagic - t);
    const int n = (int)__builtin_bit_cast(uint64_t, t);
    const uint64_t e = __builtin_bit_cast(uint64_t, table[n & (kTable - 1)]) + ((uint64_t)(uint32_t)((n >> 9) << 20) << 32);
    const double v = fma(__builtin_bit_cast(double, e), fma(r, fma(r, fma(r, a3, a2), a), 1.0), one);
    return __builtin_bit_cast(uint64_t, v) - __builtin_bit_cast(uint64_t, one);
  }
  // The bin, by how far below the maximum x lies: kBins - 1 has the largest, and what
  // bin 0 has (n <= -22065, 43 halvings and more) weighs 0.  Never turns an order
  // around, as n does not.
  static __device__ __forceinline__ int bin_of(double t) {
    const int n = (int)__builtin_bit_cast(uint64_t, t);
    return max(kBins - 1 - ((-n * 95) >> 10), 0);
  }
  __device__ __forceinline__ uint64_t operator()(float x) const {
    double d, t;
    step(x, &d, &t);
    return weight(d, t);
  }
  __device__ __forceinline__ int bin(float x) const {
    double d, t;
    step(x, &d, &t);
    return bin_of(t);
  }
};

template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)v, CTRL, ROWS, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(v >> 32), CTRL, ROWS, 0xF, true);
  return (uint64_t)hi << 32 | lo;
}

// Inclusive prefix sum over the wave: row shifts within 16 lanes (zeros come
// in), then lane 15 into rows 1 and 3, lane 31 into rows 2 and 3.
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
  v += dpp_u64<0x111, 0xF>(v);
  v += dpp_u64<0x112, 0xF>(v);
  v += dpp_u64<0x114, 0xF>(v);
  v += dpp_u64<0x118, 0xF>(v);
  v += dpp_u64<0x142, 0xA>(v);
  v += dpp_u64<0x143, 0xC>(v);
  return v;
}

// The thread's index, worked out where it is used: kept over the loops, what
// follows from it took more registers than there are (the kernel then spilled 100 and
// ran 5 to 15 us longer, writing them out).
__device__ __forceinline__ int tid() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// Inclusive prefix sum over the workgroup; *total its whole sum.
__device__ __forceinline__ uint64_t block_scan_u64(uint64_t v, uint64_t* lds, uint64_t* total) {
  const int w = tid() >> 6;
  v = wave_scan_u64(v);
  __syncthreads();
  if ((tid() & 63) == 63) lds[w] = v;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    if (i < w) before += lds[i];
    all += lds[i];
  }
  *total = all;
  return v + before;
}

struct Shared {
  uint64_t mass[kBins];
  uint32_t count[kBins];
  uint64_t seg_mass[kMaxSegments];
  uint32_t seg_ties[kMaxSegments];
  uint2 list[kList];  // (key, index)
  double table[kTable];
  uint64_t sorted_mass[kSmallList];
  uint32_t sorted_index[kSmallList];
  uint2 members[kSmallList];
  uint64_t red[kWaves];
  uint64_t found_mass;
  uint32_t found_bin, found_count, n_list, n_members, segment, seg_rank, token;
  uint64_t seg_before;
};

struct Found {
  uint32_t bin, count;
  uint64_t mass;
};

// A token stays while less than this of the mass m lies before it; the first one
// always.
__device__ __forceinline__ uint64_t reach(float p, uint64_t m) {
  return min(m, (uint64_t)fmax(ceil((double)p * (double)m), 1.0));
}

// The bin, from the highest down, in which the running count (by_mass: the
// running mass) reaches `most` (0: that of the bins' whole mass and p), and what
// lies above it; bin 0 and everything if none does.
__device__ __forceinline__ Found find_bin(Shared& s, bool by_mass, uint64_t& most, float p) {
  const int t = tid();
  const int b0 = kBins - 1 - 2 * t, b1 = b0 - 1;  // this thread's
  const uint64_t m0 = s.mass[b0], m1 = s.mass[b1], c0 = s.count[b0], c1 = s.count[b1];
  uint64_t bm = 0, bc = 0, am = 0, ac = 0;
#pragma unroll 1
  for (int i = 0; i < 2; i++) {  // both scans by the same instructions: they run once, most time goes to fetching them
    const uint64_t v = i ? c0 + c1 : m0 + m1;
    uint64_t all;
    const uint64_t before = block_scan_u64(v, s.red, &all) - v;
    if (i) {
      bc = before;
      ac = all;
    } else {
      bm = before;
      am = all;
      if (most == 0) most = reach(p, all);
    }
  }
  if ((by_mass ? am : ac) < most) return {0, (uint32_t)ac, am};
  // a bin is the one if what lies above it does not reach `most` and with it does
  auto take = [&](int bin, uint64_t mb, uint64_t cb, uint64_t m, uint64_t c) {
    const uint64_t lo = by_mass ? mb : cb, hi = by_mass ? mb + m : cb + c;
    if (lo < most && hi >= most) {
      s.found_bin = bin;
      s.found_count = (uint32_t)cb;
      s.found_mass = mb;
    }
  };
  take(b0, bm, bc, m0, c0);
  take(b1, bm + m0, bc + c0, m1, c1);
  __syncthreads();
  const Found f = {s.found_bin, s.found_count, s.found_mass};
  return f;
}

// The highest key edge (of the first 11 bits) that at least k of the threads'
// keys reach; s.count is the scratch.
__device__ __forceinline__ uint32_t edge_of_kth(Shared& s, uint32_t key, int bits, uint32_t k) {
  const int t = tid(), w = t >> 6;
  uint32_t* red = reinterpret_cast<uint32_t*>(s.red);
  s.count[t] = 0;
  s.count[t + kThreads] = 0;
  __syncthreads();
  atomicAdd(&s.count[key >> (bits - 11)], 1u);
  __syncthreads();
  const int b0 = kBins - 1 - 2 * t;
  const uint32_t c0 = s.count[b0], c1 = s.count[b0 - 1];
  uint32_t inc = (uint32_t)wave_incl_scan_i32<64>((int)(c0 + c1));
  if ((t & 63) == 63) red[w] = inc;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; i++) inc += i < w ? red[i] : 0;
  const uint32_t before = inc - c0 - c1;
  if (before < k && inc >= k) s.found_bin = before + c0 >= k ? b0 : b0 - 1;
  __syncthreads();
  return s.found_bin << (bits - 11);
}

// A cut: keys above `key`, and the first `ties` of those equal to it.
struct Cut {
  uint32_t key, ties;
};

// A row, or the part of it from piece c0 to c1, as 16-byte pieces dealt to the
// workgroup's threads in turn; `skip` elements of the first piece lie before the
// row.
template <int FMT>
struct Row {
  typedef Logit<FMT> L;
  static constexpr int E = L::kPer;
  const uint8_t* x;
  const uint4* pieces;
  int V, skip, np, inside, outside, c0, c1;
  uint4* ends;  // in LDS: the pieces that reach over the row's ends

  // NaNs, which count as -inf
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu); }

  __device__ __forceinline__ Row(const void* logits, int64_t row, int64_t stride, int V_, uint4* ends_) : V(V_), ends(ends_) {
    x = (const uint8_t*)logits + row * stride * (L::kBits / 8);
    skip = (int)((uintptr_t)x % 16) / (L::kBits / 8);
    pieces = reinterpret_cast<const uint4*>(x - skip * (L::kBits / 8));
    np = (V + skip + E - 1) / E;
    // pieces inside .. outside - 1 lie in the row as a whole
    inside = skip ? 1 : 0;
    outside = (V + skip) / E;
    c0 = 0;
    c1 = np;
    const int t = tid();
    if (t < 2) ends[t] = edge(t ? np - 1 : 0);
    __syncthreads();
  }
  __device__ __forceinline__ void take(int from, int to) {
    c0 = from;
    c1 = to;
  }
  __device__ __forceinline__ uint4 edge(int c) const {  // the elements that there are
    uint4 r = none();
    const int i = c * E - skip;
#pragma unroll
    for (int e = 0; e < E; e++)
      if ((uint32_t)(i + e) < (uint32_t)V) {
        if (FMT == AQ_F32)
          (&r.x)[e] = reinterpret_cast<const uint32_t*>(x)[i + e];
        else
          reinterpret_cast<uint16_t*>(&r)[e] = reinterpret_cast<const uint16_t*>(x)[i + e];
      }
    return r;
  }
  __device__ __forceinline__ uint4 load(int c) const {
    uint4 v = inside < outside ? pieces[min(max(c, inside), outside - 1)] : none();
    if (c >= outside) v = c == np - 1 ? ends[1] : none();
    if (c < inside) v = ends[0];
    return v;
  }
  // f(piece, its 16 bytes) for every piece, in order within a thread; the next
  // one's load is on its way meanwhile.  The whole workgroup calls f together, for
  // pieces past the end too (of a part: pieces of the next one, which are not this
  // part's, as nothing).
  template <class F>
  __device__ __forceinline__ void each_piece(F f) const {
    uint4 next = load(c0 + tid());
#pragma unroll 1
    for (int c = c0 + tid(); c - tid() < c1; c += kThreads) {
      const uint4 v = c < c1 ? next : none();
      next = load(c + kThreads);
      f(c, v);
    }
  }
  // f(index, bits, key) for a piece's elements
  template <class F>
  __device__ __forceinline__ void each_element(int c, uint4 v, F f) const {
    const int i0 = c * E - skip;
#pragma unroll 1
    for (int i = i0; i < i0 + E; i += E / 4) {
      const uint32_t q = keys_of_word<FMT>(v.x);
      f(i, FMT == AQ_F32 ? v.x : v.x & 0xFFFF, FMT == AQ_F32 ? q : q & 0xFFFF);
      if (FMT != AQ_F32) f(i + 1, v.x >> 16, q >> 16);
      v.x = v.y, v.y = v.z, v.z = v.w;
    }
  }
  static __device__ __forceinline__ uint32_t largest_key(const uint4& v) {
    const uint4 q = make_uint4(keys_of_word<FMT>(v.x), keys_of_word<FMT>(v.y), keys_of_word<FMT>(v.z), keys_of_word<FMT>(v.w));
    if constexpr (FMT == AQ_F32) {
      return max(max(q.x, q.y), max(q.z, q.w));
    } else {
      const u16x2 m = __builtin_elementwise_max(
          __builtin_elementwise_max(__builtin_bit_cast(u16x2, q.x), __builtin_bit_cast(u16x2, q.y)),
          __builtin_elementwise_max(__builtin_bit_cast(u16x2, q.z), __builtin_bit_cast(u16x2, q.w)));
      return max(m.x, m.y);
    }
  }
  // the largest keys of the thread's pieces c, c + 1024, .. (eight), and of all eight
  __device__ __forceinline__ uint32_t largest_of_eight(int c, uint32_t (&keys)[8]) const {
    uint4 v[8];
#pragma unroll
    for (int n = 0; n < 8; n++) v[n] = load(c + n * kThreads);
    uint32_t own = 0;
#pragma unroll
    for (int n = 0; n < 8; n++) {
      keys[n] = c + n * kThreads < c1 ? largest_key(v[n]) : 0;
      own = max(own, keys[n]);
    }
    return own;
  }
  // the thread's own largest key (and those of its last eight pieces), and the
  // workgroup's in *best
  __device__ __forceinline__ uint32_t largest(uint64_t* lds, uint32_t (&keys)[8], uint32_t* best) const {
    uint32_t own = 0;
#pragma unroll 1
    for (int c = c0 + tid(); c - tid() < c1; c += 8 * kThreads) own = max(own, largest_of_eight(c, keys));
    uint32_t b = own;
#pragma unroll
    for (int d = 32; d; d >>= 1) b = max(b, (uint32_t)__shfl_xor((int)b, d, 64));
    __syncthreads();
    if ((tid() & 63) == 0) lds[tid() >> 6] = b;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; i++) b = max(b, (uint32_t)lds[i]);
    *best = b;
    return own;
  }
};

// What the parts of a row leave for each other and for the last kernel.
struct PartsOfRow {
  uint64_t mass[kBins];
  uint64_t seg_mass[kMaxSegments];
  uint2 list[kList];
  uint32_t best[kMaxParts];
  uint64_t most, above;  // the mass that top-p reaches, the mass above the bin in which it does
  uint32_t n_list, bin, pad[2];
};

__device__ __forceinline__ Weigh weigh_from(float mx, float T, const double* table) {
  if (mx == INFINITY) return Weigh{1.0, 30720.0, table, 0.0f, 1.0f, 0.0f, 1};
  // lo lies at least 60 halvings below the maximum and is a finite number: for rows
  // below half the lowest of fp32 by way of their halves (T counts as 1e34 at most)
  const float f = mx < -1.7014118e38f ? 0.5f : 1.0f;
  const double m = f * mx, t = (double)f * (double)fminf(T, 1e34f);
  double c = 738.65986093514927 / t;  // 512 log2(e) / T
  float lo = (float)(m - 41.588830833596719 * t);
  if (!((m - (double)lo) * c >= 30720.0)) {
    asm volatile("");  // a branch: lo was rounded up; T may be far below the logits' steps, the next one weighs nothing
    lo = nextafterf(lo, -INFINITY);
    c = fmin(c, 92160.0 / (m - (double)lo));
  }
  return Weigh{m, c, table, lo, (float)m, f, __builtin_amdgcn_readfirstlane(f != 1.0f)};  // mx is the row's
}
__device__ __forceinline__ uint64_t whole_of(float min_p) {  // the least weight that min-p leaves
  return min_p > 0.0f ? (uint64_t)ceil(fmin((double)min_p, 1.0) * kOne) : 0;
}
__device__ __forceinline__ void fill_table(double* table) {
  if (tid() < kTable) table[tid()] = exp2((double)tid() / kTable) * kOne;
}

__device__ __forceinline__ void append(Shared& s, int V, int i, uint32_t key) {
  if ((uint32_t)i >= (uint32_t)V) return;
  const uint32_t at = atomicAdd(&s.n_list, 1u);
  if (at < kList) s.list[at] = make_uint2(key, (uint32_t)i);
}

// Masses (of w >= wmin) by segment, to seg_mass.  LISTING: of what lies in the bins
// above `bin`; what lies in it goes to the list (bin 0 does not).  Else of the keys
// above `cut`; those equal to it are counted by segment.
template <int FMT, bool LISTING>
__device__ __forceinline__ void sum_segments(Shared& s, const Row<FMT>& row, const Weigh& weigh, uint64_t wmin,
                                             int bin, uint32_t cut, uint64_t* seg_mass) {
  row.each_piece([&](int c, const uint4& v) {
    uint64_t sum = 0;
    uint32_t ties = 0;
    row.each_element(c, v, [&](int i, uint32_t bits, uint32_t key) {
      double d, t;
      weigh.step(Logit<FMT>::value(bits), &d, &t);
      const int at = LISTING ? Weigh::bin_of(t) : 0;
      const bool above = LISTING ? at > bin : key > cut;
      if (__ballot(above)) {  // the exponential only where a lane asks for it
        const uint64_t w = weigh.weight(d, t);
        sum += above && w >= wmin ? w : 0;
      }
      if (LISTING) {
        if (bin && at == bin && c < row.c1) append(s, row.V, i, key);
      } else {
        ties += (uint32_t)__popcll(__ballot(key == cut && (uint32_t)i < (uint32_t)row.V));
      }
    });
    sum = wave_scan_u64(sum);
    if ((tid() & 63) == 63 && c - 63 < row.c1) {  // 64 pieces are a segment
      seg_mass[c >> 6] = sum;
      if (!LISTING) s.seg_ties[c >> 6] = ties;
    }
  });
  __syncthreads();
}

__device__ __forceinline__ void clear_bins(Shared& s) {
  __syncthreads();
  for (int i = tid(); i < kBins; i += kThreads) {
    s.mass[i] = 0;
    s.count[i] = 0;
  }
  __syncthreads();
}

// ---- long rows that one workgroup each would leave most of the GPU idle for:
// parts of a row in a workgroup each, three passes, and then sample_kernel for what
// is left (a list and the segments' masses).  For rows without top-k, whose every
// exponential is needed; the others are left to sample_kernel whole.

template <int FMT>
__device__ __forceinline__ Row<FMT> part_of(const void* logits, int V, int64_t stride, int per, uint4* ends) {
  Row<FMT> row(logits, blockIdx.y, stride, V, ends);
  row.take((int)blockIdx.x * per, min((int)(blockIdx.x + 1) * per, row.np));
  return row;
}

__device__ __forceinline__ bool in_parts(const Settings& set, int row, int V) {
  const int k = set.k ? set.k[row] : set.k0;
  const float T = set.t ? set.t[row] : set.t0;
  return !(k > 0 && k < V) && T > 0.0f;
}

// The part's largest key; the row's bins and list emptied.
template <int FMT>
__global__ __launch_bounds__(kThreads) void sample_max_kernel(const void* __restrict__ logits, int V, int64_t stride,
                                                              int per, Settings set, PartsOfRow* __restrict__ ws) {
  __shared__ uint64_t red[kWaves];
  __shared__ uint4 ends[2];
  if (!in_parts(set, blockIdx.y, V)) return;
  const Row<FMT> row = part_of<FMT>(logits, V, stride, per, ends);
  PartsOfRow& w = ws[blockIdx.y];
  uint32_t best, keys8[8];
  row.largest(red, keys8, &best);
  if (tid() == 0) w.best[blockIdx.x] = best;
  for (int i = blockIdx.x * kThreads + tid(); i < kBins; i += gridDim.x * kThreads) w.mass[i] = 0;
  if (blockIdx.x == 0 && tid() == 0) w.n_list = 0;
}

// The row's largest key.  (All at once: loads one after the other, 31 of them, took 3 us
// a kernel.)
__device__ __forceinline__ uint32_t best_of(const PartsOfRow& w, int parts) {
  uint32_t b = 0;
#pragma unroll
  for (int i = 0; i < kMaxParts; i++) {
    const uint32_t x = w.best[i];  // past the parts whatever is there
    b = i < parts ? max(b, x) : b;
  }
  return b;
}

// The part's masses by bins, added to the row's.
template <int FMT>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(const void* __restrict__ logits, int V, int64_t stride,
                                                               int per, Settings set, PartsOfRow* __restrict__ ws) {
  __shared__ uint64_t mass[kBins];
  __shared__ double table[kTable];
  __shared__ uint4 ends[2];
  const int b = blockIdx.y;
  const float p = set.p ? set.p[b] : set.p0, T = set.t ? set.t[b] : set.t0;
  if (!in_parts(set, b, V) || !(p < 1.0f)) return;
  const Row<FMT> row = part_of<FMT>(logits, V, stride, per, ends);
  PartsOfRow& w = ws[b];
  const float mx = Logit<FMT>::value_of_key(best_of(w, gridDim.x));
  if (mx == -INFINITY) return;
  for (int i = tid(); i < kBins; i += kThreads) mass[i] = 0;
  fill_table(table);
  __syncthreads();
  const Weigh weigh = weigh_from(mx, T, table);
  row.each_piece([&](int c, const uint4& v) {
    row.each_element(c, v, [&](int, uint32_t bits, uint32_t) {
      double d, t;
      weigh.step(Logit<FMT>::value(bits), &d, &t);
      const int at = Weigh::bin_of(t);
      if (at) atomicAdd((unsigned long long*)&mass[at], weigh.weight(d, t));
    });
  });
  __syncthreads();
  for (int i = tid(); i < kBins; i += kThreads)
    if (mass[i]) atomicAdd((unsigned long long*)&w.mass[i], (unsigned long long)mass[i]);
}

// The part's segments above the bin in which the running mass reaches p, and its
// members of that bin (without top-p: all segments).
template <int FMT>
__global__ __launch_bounds__(kThreads) void sample_segments_kernel(const void* __restrict__ logits, int V,
                                                                   int64_t stride, int per, Settings set,
                                                                   PartsOfRow* __restrict__ ws) {
  __shared__ Shared s;
  __shared__ uint32_t at;
  __shared__ uint4 ends[2];
  const int b = blockIdx.y, t = tid();
  const float p = set.p ? set.p[b] : set.p0, T = set.t ? set.t[b] : set.t0, mp = set.m ? set.m[b] : set.m0;
  if (!in_parts(set, b, V)) return;
  const Row<FMT> row = part_of<FMT>(logits, V, stride, per, ends);
  PartsOfRow& w = ws[b];
  const float mx = Logit<FMT>::value_of_key(best_of(w, gridDim.x));
  if (mx == -INFINITY) return;
  fill_table(s.table);
  if (t == 0) s.n_list = 0;
  int bin = 0;  // no list: everything that weighs something lies above
  if (p < 1.0f) {
    for (int i = t; i < kBins; i += kThreads) {
      s.mass[i] = w.mass[i];
      s.count[i] = 0;
    }
    __syncthreads();
    uint64_t most = 0;
    const Found f = find_bin(s, true, most, p);
    bin = (int)f.bin;
    if (blockIdx.x == 0 && t == 0) {
      w.most = most;
      w.above = f.mass;
      w.bin = f.bin;
    }
  }
  __syncthreads();
  const uint64_t wmin = whole_of(mp);
  sum_segments<FMT, true>(s, row, weigh_from(mx, T, s.table), wmin, bin, 0, w.seg_mass);
  const uint32_t n = s.n_list;  // more than there is room for is counted all the same
  if (t == 0) at = atomicAdd(&w.n_list, n);
  __syncthreads();
  for (uint32_t i = t; i < min(n, (uint32_t)kList) && at + i < kList; i += kThreads) w.list[at + i] = s.list[i];
}

template <int FMT>
__global__ __launch_bounds__(kThreads) void sample_kernel(const void* __restrict__ logits, int V, int64_t stride,
                                                          const float* __restrict__ u, Settings set,
                                                          const PartsOfRow* __restrict__ ws, int parts,
                                                          int64_t* __restrict__ out) {
  typedef Logit<FMT> L;
  constexpr int B = L::kBits, E = L::kPer;
  __shared__ Shared s;
  const int t = tid(), row = blockIdx.x;
  const float T = set.t ? set.t[row] : set.t0, p = set.p ? set.p[row] : set.p0, mp = set.m ? set.m[row] : set.m0;
  const int k = set.k ? set.k[row] : set.k0;
  __shared__ uint4 ends[2];
  const Row<FMT> r(logits, row, stride, V, ends);
  const int skip = r.skip, np = r.np;

  // ---- the largest key, each thread's own on the way
  if (t == 0) s.n_list = 0;
  // a row whose parts have been summed: what they left
  const PartsOfRow* done = parts > 1 && in_parts(set, row, V) && best_of(ws[row], parts) > L::kLowest ? ws + row : nullptr;
  for (int i = t; i < kMaxSegments; i += kThreads) {
    s.seg_mass[i] = done && i < (np + 63) / 64 ? done->seg_mass[i] : 0;
    s.seg_ties[i] = 0;
  }
  if (done && p < 1.0f) {
    if (t == 0) s.n_list = done->n_list;
    for (int i = t; i < (int)min(done->n_list, (uint32_t)kList); i += kThreads) s.list[i] = done->list[i];
  }
  uint32_t own = 0, best, keys8[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (done)
    best = best_of(*done, parts);
  else
    own = r.largest(s.red, keys8, &best);
  best = __builtin_amdgcn_readfirstlane(best);
  const float mx = L::value_of_key(best);
  const Weigh weigh = weigh_from(mx, T, s.table);
  const bool greedy = !(T > 0.0f) || mx == -INFINITY;  // also a row without a token to choose: its first
  const uint64_t wmin = whole_of(mp);
  if (greedy) {
    if (t == 0) s.token = 0xFFFFFFFFu;
    __syncthreads();
    if (own == best) {  // few threads
      uint32_t i0 = 0xFFFFFFFFu;
#pragma unroll 1
      for (int c = t; c < np && i0 == 0xFFFFFFFFu; c += kThreads)
        r.each_element(c, r.load(c), [&](int i, uint32_t, uint32_t key) {
          if (key == best && (uint32_t)i < (uint32_t)V) i0 = min(i0, (uint32_t)i);
        });
      atomicMin(&s.token, i0);
    }
    __syncthreads();
    if (t == 0) out[row] = s.token;
    return;
  }
  fill_table(s.table);
  __syncthreads();

  const bool by_k = k > 0 && k < V, by_p = p < 1.0f;
  const float uu = u[row];
  auto goal_of = [&](uint64_t total) {
    const uint64_t g = uu > 0.0f ? (uint64_t)fmin((double)uu * (double)total, 9.2e18) : 0;
    return min(g, total - 1);
  };
  // The whole rest for a list of at most 256 that holds the first k: four
  // threads a member count what comes before it.
  auto small_list = [&] {
    const int n = (int)s.n_list, t = tid(), i = t >> 2, ln = t & 63;
    const uint2 me = i < n ? s.list[i] : make_uint2(0, 0);
    uint32_t r = 0;
#pragma unroll 4
    for (int j = t & 3; j < n; j += 4) {
      const uint2 o = s.list[j];
      r += (o.x > me.x) | ((o.x == me.x) & (o.y < me.y));
    }
    r += xlane_partner_u32<1>(r);
    r += xlane_partner_u32<2>(r);
    const uint64_t w = i < n ? weigh(L::value_of_key(me.x)) : 0;
    if (i < n && (t & 3) == 0) {
      s.sorted_mass[r] = w;
      s.sorted_index[r] = me.y;
    }
    __syncthreads();
    // every wave by itself: four of the sorted members a lane
    uint64_t m[4], sum = 0;
    int last = min(n, k);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      m[e] = 4 * ln + e < last ? s.sorted_mass[4 * ln + e] : 0;
      sum += m[e];
    }
    uint64_t inc = wave_scan_u64(sum);
    const uint64_t most = by_p ? reach(p, __shfl(inc, 63, 64)) : ~0ull;
    uint64_t at = inc - sum;
    int stay = 0;
    sum = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const bool in = 4 * ln + e < last && at < most && m[e] >= wmin;
      at += m[e];
      stay += in;
      sum += in ? m[e] : 0;
    }
    last = __builtin_amdgcn_readlane(wave_incl_scan_i32<64>(stay), 63);
    const uint64_t goal = goal_of(__shfl(wave_scan_u64(sum), 63, 64));
    // the kept ones by index
    uint64_t before = 0;
#pragma unroll 4
    for (int j = t & 3; j < last; j += 4) before += s.sorted_index[j] < me.y ? s.sorted_mass[j] : 0;
    before += (uint64_t)__shfl_xor((long long)before, 1, 64);
    before += (uint64_t)__shfl_xor((long long)before, 2, 64);
    if ((t & 3) == 0 && i < n && (int)r < last && before <= goal && goal < before + w) out[row] = me.y;
  };

  Cut cut = {0, 0};  // everything
  bool from_list = false, summed = false, binned = false;
  uint64_t mass = 0;
  // f(index, key) for the list's members or the row's tokens
  auto each = [&](auto f) {
    if (from_list) {
      const int n = (int)s.n_list;
#pragma unroll 1
      for (int i = tid(); i < n; i += kThreads) f((int)s.list[i].y, s.list[i].x);
    } else {
      r.each_piece([&](int c, const uint4& v) { r.each_element(c, v, [&](int i, uint32_t, uint32_t key) { f(i, key); }); });
    }
  };
  if (by_k && k <= kMaxListK) {
    const int t = tid();
    const uint32_t least = edge_of_kth(s, own, B, (uint32_t)k);
    if (own >= least) {  // a thread whose largest is less has none
#pragma unroll 1
      for (int c = t; c < np; c += 8 * kThreads) {
        if (np > 8 * kThreads) r.largest_of_eight(c, keys8);
        uint32_t which = 0;  // of eight pieces those that have one
#pragma unroll
        for (int n = 0; n < 8; n++) which |= (keys8[n] >= least ? 1u : 0u) << n;
        for (; which; which &= which - 1) {
          const int d = c + __builtin_ctz(which) * kThreads;
          r.each_element(d, r.load(d), [&](int i, uint32_t, uint32_t key) {
            if (key >= least) append(s, V, i, key);
          });
        }
      }
    }
    __syncthreads();
    from_list = s.n_list <= kList;
    if (s.n_list <= kSmallList) {
      small_list();
      return;
    }
  }

  // the cut of the first k, then that of the mass p of these
#pragma unroll 1
  for (int stage = 0; stage < 2; stage++) {
    const bool by_mass = stage == 1;
    if (by_mass ? !by_p : !by_k) continue;
    uint64_t most = by_mass ? (by_k ? reach(p, mass) : 0) : (uint64_t)k;
    // the bin in which the running count (by_mass: the running mass) reaches `most`;
    // then, unless its members are few, the bits of their keys, 11 at a time
    int bin = 0;
    uint32_t key = 0, above = 0, ties = 0;  // the last key kept, how many of it
    uint64_t above_mass = 0;
    bool all = false;
#pragma unroll 1
    for (int shift = B + 11; shift > 0;) {
      const bool first = shift > B;
      const int bits = min(11, shift), next = shift - bits, t = tid(), ln = t & 63;
      Found f;
      if (first && done) {
        most = done->most;
        f = {done->bin, 0, done->above};
      } else {
        if (!first || !binned) {
          clear_bins(s);
          each([&](int i, uint32_t y) {
            double d, t;
            weigh.step(L::value_of_key(y), &d, &t);
            const int at = Weigh::bin_of(t);
            if (!at || (uint32_t)i >= (uint32_t)V) return;  // the rest weighs nothing
            if (!first && !(at == bin && (shift == B || y >> (shift & 31) == key))) return;
            const uint32_t to = first ? (uint32_t)at : (y >> next) & ((1u << bits) - 1);
            if (by_k || !first) atomicAdd(&s.count[to], 1u);
            atomicAdd((unsigned long long*)&s.mass[to], weigh.weight(d, t));
          });
          __syncthreads();
        }
        binned = first;
        uint64_t left = first ? most : most - (by_mass ? above_mass : above);
        f = find_bin(s, by_mass, left, p);
        if (first) most = left;
      }
      above += f.count;
      above_mass += f.mass;
      shift = next;
      if (!first) {
        key = key << bits | f.bin;
        if (shift == 0) {
          const uint64_t each_mass = s.mass[f.bin] / s.count[f.bin];  // of one of the ties
          ties = by_mass ? (uint32_t)((most - above_mass + each_mass - 1) / each_mass) : (uint32_t)(most - above);
          above_mass += ties * each_mass;
        }
        continue;
      }
      if (f.bin == 0) {  // the first k have everything that weighs something
        all = true;
        break;
      }
      bin = (int)f.bin;
      // its members: the list, or `members`
      if (t == 0) s.n_members = 0;
      __syncthreads();
      const uint2* members = s.members;
      uint32_t n;
      if (by_mass && !by_k) {
        if (!done) sum_segments<FMT, true>(s, r, weigh, wmin, bin, 0, s.seg_mass);
        members = s.list;
        n = s.n_list;
        summed = from_list = n <= kList;
      } else {
        each([&](int i, uint32_t key) {
          if (weigh.bin(L::value_of_key(key)) == bin && (uint32_t)i < (uint32_t)V) {
            const uint32_t at = atomicAdd(&s.n_members, 1u);
            if (at < kSmallList) s.members[at] = make_uint2(key, (uint32_t)i);
          }
        });
        __syncthreads();
        n = s.n_members;
      }

      if (n > kSmallList) continue;
      // by comparing the members with each other, four threads each
      const int i = t >> 2;
      const uint2 me = i < (int)n ? members[i] : make_uint2(0, 0);
      uint32_t rank = 0;
#pragma unroll 4
      for (int j = t & 3; j < (int)n; j += 4) {
        const uint2 o = members[j];
        rank += (o.x > me.x) | ((o.x == me.x) & (o.y < me.y));
      }
      rank += xlane_partner_u32<1>(rank);
      rank += xlane_partner_u32<2>(rank);
      if (i < (int)n && (t & 3) == 0) {
        s.sorted_mass[rank] = weigh(L::value_of_key(me.x));
        s.sorted_index[rank] = me.x;
      }
      __syncthreads();
      // every wave by itself, four of the sorted members a lane: how many lie before
      // the one that reaches `most`
      uint64_t m[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        m[e] = 4 * ln + e < (int)n ? s.sorted_mass[4 * ln + e] : 0;
        sum += m[e];
      }
      uint64_t at = above_mass + wave_scan_u64(sum) - sum;
      int before = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        at += m[e];
        before += 4 * ln + e < (int)n - 1 && (by_mass ? at < most : above + 4 * ln + e + 1 < most);
      }
      before = __builtin_amdgcn_readlane(wave_incl_scan_i32<64>(before), 63);
      key = s.sorted_index[before];
      sum = 0;
      int same = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const bool in = 4 * ln + e <= before;
        sum += in ? m[e] : 0;
        same += in && s.sorted_index[4 * ln + e] == key;
      }
      above_mass += __shfl(wave_scan_u64(sum), 63, 64);
      ties = (uint32_t)__builtin_amdgcn_readlane(wave_incl_scan_i32<64>(same), 63);
      __syncthreads();
      break;
    }
    if (all) {
      mass = above_mass;
      continue;
    }
    if (!by_mass) {
      cut = {key, ties};
      mass = above_mass;
    } else if (key > cut.key) {
      cut = {key, ties};
    } else if (key == cut.key) {
      cut.ties = min(cut.ties, ties);
    }
  }

  // ---- kept masses and ties by segment
  uint64_t wcut = cut.key ? weigh(L::value_of_key(cut.key)) : 0;
  if (wcut < wmin) wcut = 0;
  __syncthreads();
  if (done && !by_p) summed = true;
  if (from_list) {
    for (int i = t; i < (int)s.n_list; i += kThreads) {
      const uint2 y = s.list[i];
      const int seg = ((int)y.y + skip) / (E * 64);
      if (y.x == cut.key) {
        atomicAdd(&s.seg_ties[seg], 1u);
      } else if (y.x > cut.key) {
        const uint64_t w = weigh(L::value_of_key(y.x));
        if (w >= wmin) atomicAdd((unsigned long long*)&s.seg_mass[seg], w);
      }
    }
  } else if (!summed) {
    sum_segments<FMT, false>(s, r, weigh, wmin, 0, cut.key, s.seg_mass);
  }
  __syncthreads();

  // ---- the segment: thread t has segment t (and the few past 1024 thread 1023)
  const int ns = (np + 63) / 64;
  uint64_t total;
  uint32_t tie0;
  uint64_t m0;
  {
    uint32_t ties = 0;
    const int s0 = t, s1 = t == kThreads - 1 ? ns : min(ns, t + 1);
    for (int i = s0; i < s1; i++) ties += s.seg_ties[i];
    uint64_t all;
    tie0 = (uint32_t)block_scan_u64(ties, s.red, &all) - ties;
    uint64_t sum = 0;
    uint32_t rank = tie0;
    for (int i = s0; i < s1; i++) {
      sum += s.seg_mass[i] + wcut * (uint64_t)min(s.seg_ties[i], cut.ties - min(rank, cut.ties));
      rank += s.seg_ties[i];
    }
    m0 = block_scan_u64(sum, s.red, &total) - sum;
    const uint64_t goal = goal_of(total);
    if (m0 <= goal && goal < m0 + sum) {
      uint64_t at = m0;
      rank = tie0;
      for (int i = s0; i < s1; i++) {
        const uint64_t m = s.seg_mass[i] + wcut * (uint64_t)min(s.seg_ties[i], cut.ties - min(rank, cut.ties));
        if (at <= goal && goal < at + m) {
          s.segment = i;
          s.seg_before = goal - at;  // what is left of the goal inside
          s.seg_rank = rank;
        }
        at += m;
        rank += s.seg_ties[i];
      }
    }
  }
  __syncthreads();
  // ---- the token: one wave, a piece a lane
  if (t < 64) {
    const int c = (int)s.segment * 64 + t;
    const uint4 v = r.load(c);
    uint32_t ties = 0;
    r.each_element(c, v, [&](int i, uint32_t, uint32_t key) { ties += key == cut.key && (uint32_t)i < (uint32_t)V; });
    const uint32_t rank = s.seg_rank + (uint32_t)wave_scan_u64(ties) - ties;
    auto mass_of = [&](int i, uint32_t bits, uint32_t key, uint32_t& n) -> uint64_t {
      if ((uint32_t)i >= (uint32_t)V || key < cut.key) return 0;
      if (key == cut.key) return n++ < cut.ties ? wcut : 0;
      const uint64_t w = weigh(L::value(bits));
      return w >= wmin ? w : 0;
    };
    uint64_t sum = 0;
    uint32_t n = rank;
    r.each_element(c, v, [&](int i, uint32_t bits, uint32_t key) { sum += mass_of(i, bits, key, n); });
    uint64_t at = wave_scan_u64(sum) - sum;
    const uint64_t goal = s.seg_before;
    n = rank;
    if (at <= goal && goal < at + sum)
      r.each_element(c, v, [&](int i, uint32_t bits, uint32_t key) {
        const uint64_t w = mass_of(i, bits, key, n);
        if (at <= goal && goal < at + w) out[row] = i;
        at += w;
      });
  }
}

}  // namespace

// Workgroups a row is split into: enough to fill the GPU, 1024 pieces each at
// least, for rows that have 2048 (top-p of 64 rows of 128256: one workgroup each
// 106 us, four 55; of one row in fp32 118 us and, in 31, 33).  One setting of top-k
// for all rows rules the split out.
static int parts_of(int64_t B, int64_t V, int dtype, bool top_k) {
  const int64_t per = dtype == AQ_F32 ? 4 : 8, pieces = V / per;
  if (top_k || pieces < 2048) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(kMaxParts, 256 / B), pieces / 1024));
}

extern "C" int64_t aq_sample_workspace(int64_t B, int64_t V, int dtype, int32_t top_k0) {
  if (B <= 0 || B > 65535 || V <= 0 || V > kMaxVocab || dtype < AQ_F16 || dtype > AQ_F32) return -1;
  return parts_of(B, V, dtype, top_k0 > 0 && top_k0 < V) > 1 ? B * (int64_t)sizeof(PartsOfRow) : 0;
}

extern "C" int aq_sample(const void* logits, int dtype, int64_t B, int64_t V, int64_t stride, const float* u,
                         const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                         float temperature0, int32_t top_k0, float top_p0, float min_p0, int64_t* tokens,
                         void* workspace, int64_t ws_bytes, void* stream) {
  AQ_CHECK_ARG(logits && u && tokens, "aq_sample: null pointer");
  AQ_CHECK_ARG(dtype == AQ_F16 || dtype == AQ_BF16 || dtype == AQ_F32, "aq_sample: dtype %d (fp16, bf16, fp32)", dtype);
  AQ_CHECK_ARG(V > 0 && V <= kMaxVocab, "aq_sample: %lld logits a row (1 .. %lld)", (long long)V, (long long)kMaxVocab);
  AQ_CHECK_ARG(B > 0 && B <= 65535 && stride >= V, "aq_sample: %lld rows (1 .. 65535) %lld apart", (long long)B,
               (long long)stride);
  const int64_t size = dtype == AQ_F32 ? 4 : 2;
  AQ_CHECK_ARG((uintptr_t)logits % size == 0 && (uintptr_t)u % 4 == 0 && (uintptr_t)tokens % 8 == 0 &&
                   (uintptr_t)temperature % 4 == 0 && (uintptr_t)top_k % 4 == 0 && (uintptr_t)top_p % 4 == 0 &&
                   (uintptr_t)min_p % 4 == 0,
               "aq_sample: misaligned buffer");
  const Settings set = {temperature, top_p, min_p, top_k, temperature0, top_p0, min_p0, top_k0};
  hipStream_t s = (hipStream_t)stream;
  // (greedy rows need one pass and no exponential)
  int parts = parts_of(B, V, dtype, !top_k && ((top_k0 > 0 && top_k0 < V) || (!temperature && !(temperature0 > 0.0f))));
  AQ_CHECK_ARG(!workspace || (uintptr_t)workspace % 16 == 0, "aq_sample: the workspace must be 16-byte aligned");
  if (parts > 1 && (!workspace || ws_bytes < B * (int64_t)sizeof(PartsOfRow))) parts = 1;
  PartsOfRow* ws = (PartsOfRow*)workspace;
  // parts of whole segments; a misaligned row has one piece more
  const int64_t pieces = V / (16 / size) + 2;
  const int per = (int)(aq::ceil_div(aq::ceil_div(pieces, parts), 64) * 64);
  parts = (int)aq::ceil_div(pieces, per);
  const dim3 grid((unsigned)B), cut((unsigned)parts, (unsigned)B), block(kThreads);
#define AQ_SAMPLE(F)                                                                                                  \
  do {                                                                                                                \
    if (parts > 1) {                                                                                                  \
      hipLaunchKernelGGL(sample_max_kernel<F>, cut, block, 0, s, logits, (int)V, stride, per, set, ws);               \
      if (top_p || top_p0 < 1.0f)                                                                                     \
        hipLaunchKernelGGL(sample_bins_kernel<F>, cut, block, 0, s, logits, (int)V, stride, per, set, ws);            \
      hipLaunchKernelGGL(sample_segments_kernel<F>, cut, block, 0, s, logits, (int)V, stride, per, set, ws);          \
    }                                                                                                                 \
    hipLaunchKernelGGL(sample_kernel<F>, grid, block, 0, s, logits, (int)V, stride, u, set, (const PartsOfRow*)ws,    \
                       parts, tokens);                                                                                \
  } while (0)
  if (dtype == AQ_F16) AQ_SAMPLE(AQ_F16);
  else if (dtype == AQ_BF16) AQ_SAMPLE(AQ_BF16);
  else AQ_SAMPLE(AQ_F32);
#undef AQ_SAMPLE
  AQ_LAUNCH_CHECK("aq_sample");
  return AQ_OK;
}
