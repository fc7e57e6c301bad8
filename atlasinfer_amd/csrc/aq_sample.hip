// aq_sample.hip -- the next token of every sequence from its logits and one
// given random number: temperature, top-k, top-p, min-p.
//
// The mathematics.  Tokens in the order of falling logit, equal ones by index;
// w_i = exp((x_i - max) / T).  Every filter keeps a beginning of that order:
// the first k; of those the tokens before which less than p of their mass
// lies; the tokens of w >= min_p.  So the kept set is known by one key (the
// last logit kept) and the number of its ties kept, found by descending the
// bits of the logits with histograms of counts and masses.  The token is the
// first kept one, by index, whose running mass passes u times the kept mass.
//
// Masses are integers, w rounded to 2^-45 (V <= 2^18 of them stay below
// 2^63): sums do not depend on their order, the same call gives the same
// token on every run, and a border lies within V 2^-46 of its place (2^-28 of
// the largest weight, were all the roundings one way).  The exponentials are
// taken in 64 bits: a border between two of V tokens lies in an interval as
// narrow as 1 / V, so an error of 2^-24 in the sums would choose another token
// now and then.
#include "aq_common.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int64_t kMaxVocab = 1 << 18;
constexpr int kTileShift = 13;  // 8192 elements: 8 a thread
constexpr int kTile = 1 << kTileShift;
constexpr int kMaxTiles = (int)(kMaxVocab >> kTileShift);
constexpr double kOne = 35184372088832.0;  // 2^45

struct Settings {
  const float *t, *p, *m;
  const int* k;
  float t0, p0, m0;
  int k0;
};

// 16-bit or 32-bit keys whose order as integers is the logits' order: NaN as
// -inf, -0 as 0.
template <int FMT>
struct Logit;
template <>
struct Logit<AQ_F16> {
  typedef uint16_t raw;
  static constexpr int kBits = 16;
  static __device__ float value(raw r) { return (float)bits_to_h(r); }
};
template <>
struct Logit<AQ_BF16> {
  typedef uint16_t raw;
  static constexpr int kBits = 16;
  static __device__ float value(raw r) { return __builtin_bit_cast(float, (uint32_t)r << 16); }
};
template <>
struct Logit<AQ_F32> {
  typedef uint32_t raw;
  static constexpr int kBits = 32;
  static __device__ float value(raw r) { return __builtin_bit_cast(float, r); }
};

template <int FMT>
__device__ __forceinline__ float logit(typename Logit<FMT>::raw r) {
  const float f = Logit<FMT>::value(r);
  return f != f ? -INFINITY : f + 0.0f;
}

// Key of a logit: the sign bit flipped, every bit of negative numbers.
template <int FMT>
__device__ __forceinline__ uint32_t key_of(typename Logit<FMT>::raw r) {
  constexpr int B = Logit<FMT>::kBits;
  constexpr uint32_t sign = 1u << (B - 1), all = B == 32 ? 0xFFFFFFFFu : (1u << (B & 31)) - 1;
  const float f = Logit<FMT>::value(r);
  uint32_t b = r;
  if (f == 0.0f) b = 0;
  if (f != f) b = FMT == AQ_F16 ? 0xFC00u : FMT == AQ_BF16 ? 0xFF80u : 0xFF800000u;  // -inf
  return b & sign ? ~b & all : b | sign;
}

template <int FMT>
__device__ __forceinline__ float logit_of_key(uint32_t key) {
  constexpr int B = Logit<FMT>::kBits;
  constexpr uint32_t sign = 1u << (B - 1), all = B == 32 ? 0xFFFFFFFFu : (1u << (B & 31)) - 1;
  const uint32_t b = key & sign ? key & ~sign : ~key & all;
  return Logit<FMT>::value((typename Logit<FMT>::raw)b);
}

// exp((x - max) / T) with c = log2(e) / T; the largest logit weighs 1 also
// where it is infinite or T so small that c is.
__device__ __forceinline__ double weight(float x, float mx, double c) {
  if (x == mx) return 1.0;
  if (x == -INFINITY) return 0.0;
  return exp2(((double)x - (double)mx) * c);
}
__device__ __forceinline__ uint64_t fixed(double w) { return (uint64_t)(w * kOne + 0.5); }

__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t t = __shfl_up(v, d, 64);
    if ((threadIdx.x & 63) >= d) v += t;
  }
  return v;
}

// Inclusive prefix sum over the workgroup; *total its whole sum.
__device__ __forceinline__ uint64_t block_scan_u64(uint64_t v, uint64_t* lds, uint64_t* total) {
  const int w = threadIdx.x >> 6;
  v = wave_scan_u64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[w] = v;
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
  uint64_t red[kWaves];
  uint64_t tile_mass[kMaxTiles];
  uint32_t tile_ties[kMaxTiles];
  uint64_t found_mass;
  uint32_t found_bin, found_count, token;
};

// A cut: keys above `key`, and the first `ties` of those equal to it.
struct Cut {
  uint32_t key, ties;
};

// The bin, from the highest down, in which the running count (by_mass: the
// running mass) reaches `most`, and what lies above it.  The caller knows that
// one does.
__device__ __forceinline__ void find_bin(Shared& s, bool by_mass, uint64_t most, uint32_t* bin,
                                         uint32_t* count, uint64_t* mass) {
  const int t = threadIdx.x;
  // thread t has bins 2047 - 2t and 2046 - 2t
  const int b0 = kBins - 1 - 2 * t, b1 = b0 - 1;
  const uint64_t m0 = s.mass[b0], m1 = s.mass[b1], c0 = s.count[b0], c1 = s.count[b1];
  uint64_t all_m, all_c;
  const uint64_t im = block_scan_u64(m0 + m1, s.red, &all_m);
  const uint64_t ic = block_scan_u64(c0 + c1, s.red, &all_c);
  const uint64_t bm0 = im - m0 - m1, bc0 = ic - c0 - c1, bm1 = im - m1, bc1 = ic - c1;
  // a bin is the one if the next one's first token is cut, and its own is not
  auto cut = [&](uint64_t m, uint64_t c) { return (by_mass ? m : c) >= most; };
  if (c0 && !cut(bm0, bc0) && cut(bm1, bc1)) {
    s.found_bin = b0;
    s.found_count = (uint32_t)bc0;
    s.found_mass = bm0;
  }
  if (c1 && !cut(bm1, bc1) && cut(im, ic)) {
    s.found_bin = b1;
    s.found_count = (uint32_t)bc1;
    s.found_mass = bm1;
  }
  __syncthreads();
  *bin = s.found_bin;
  *count = s.found_count;
  *mass = s.found_mass;
  __syncthreads();
}

template <int FMT>
__global__ __launch_bounds__(kThreads) void sample_kernel(const typename Logit<FMT>::raw* __restrict__ logits, int V,
                                                          int64_t stride, const float* __restrict__ u, Settings set,
                                                          int64_t* __restrict__ out) {
  constexpr int B = Logit<FMT>::kBits;
  __shared__ Shared s;
  const int t = threadIdx.x, row = blockIdx.x;
  const typename Logit<FMT>::raw* x = logits + row * stride;
  const float T = set.t ? set.t[row] : set.t0, p = set.p ? set.p[row] : set.p0, mp = set.m ? set.m[row] : set.m0;
  const int k = set.k ? set.k[row] : set.k0;

  uint32_t best = 0;
  for (int i = t; i < V; i += kThreads) best = max(best, key_of<FMT>(x[i]));
#pragma unroll
  for (int d = 32; d; d >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, d, 64));
  if ((t & 63) == 0) s.red[t >> 6] = best;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; i++) best = max(best, (uint32_t)s.red[i]);
  const float mx = logit_of_key<FMT>(best);
  const double c = 1.4426950408889634 / (double)T;

  // descends the keys' bits, 11 at a time, to the key at which the running
  // count (by_mass: the running mass) reaches `most`
  auto descend = [&](bool by_mass, uint64_t most, uint32_t* above, uint64_t* above_mass, uint64_t* each,
                     uint32_t* ties) -> uint32_t {
    uint32_t prefix = 0, cnt = 0;
    uint64_t mass = 0;
    int shift = B;
    uint32_t bin_count = 0;
    uint64_t bin_mass = 0;
    while (shift > 0) {
      const int bits = min(11, shift), next = shift - bits;
      __syncthreads();
      for (int i = t; i < kBins; i += kThreads) {
        s.mass[i] = 0;
        s.count[i] = 0;
      }
      __syncthreads();
      for (int i = t; i < V; i += kThreads) {
        const uint32_t key = key_of<FMT>(x[i]);
        if (shift < 32 && shift < B && (key >> shift) != prefix) continue;
        const uint32_t bin = (key >> next) & ((1u << bits) - 1);
        atomicAdd(&s.count[bin], 1u);
        const uint64_t w = fixed(weight(logit<FMT>(x[i]), mx, c));
        if (w) atomicAdd((unsigned long long*)&s.mass[bin], (unsigned long long)w);
      }
      __syncthreads();
      uint32_t bin, bc;
      uint64_t bm;
      find_bin(s, by_mass, most - (by_mass ? mass : cnt), &bin, &bc, &bm);
      cnt += bc;
      mass += bm;
      bin_count = s.count[bin];
      bin_mass = s.mass[bin];
      prefix = shift == B ? bin : (prefix << bits) | bin;
      shift = next;
      __syncthreads();
    }
    *above = cnt;
    *above_mass = mass;
    *ties = bin_count;
    *each = bin_mass / bin_count;
    return prefix;
  };

  Cut cut = {0, (uint32_t)V};  // everything
  const bool greedy = !(T > 0.0f) || mx == -INFINITY;  // also a row without a token to choose: its first
  if (greedy) {
    cut = {best, 1};
  } else {
    uint32_t above, ties;
    uint64_t above_mass, each, mass = 0;
    bool have_mass = false;
    if (k > 0 && k < V) {
      const uint32_t key = descend(false, (uint64_t)k, &above, &above_mass, &each, &ties);
      cut = {key, (uint32_t)k - above};
      mass = above_mass + cut.ties * each;
      have_mass = true;
    }
    if (p < 1.0f) {
      if (!have_mass) {
        uint64_t part = 0;
        for (int i = t; i < V; i += kThreads) part += fixed(weight(logit<FMT>(x[i]), mx, c));
        block_scan_u64(part, s.red, &mass);
      }
      // a token stays while less than this lies before it; the first one always
      const uint64_t most = min(mass, (uint64_t)fmax(ceil((double)p * (double)mass), 1.0));
      const uint32_t key = descend(true, most, &above, &above_mass, &each, &ties);
      const uint32_t n = (uint32_t)((most - above_mass + each - 1) / each);
      if (key > cut.key)
        cut = {key, n};
      else if (key == cut.key)
        cut.ties = min(cut.ties, n);
    }
  }
  const double wmin = !greedy && mp > 0.0f ? fmin((double)mp, 1.0) : 0.0;
  auto kept = [&](uint32_t key, float f, uint64_t* w) {  // keys above the cut
    const double e = weight(f, mx, c);
    *w = fixed(e);
    return key > cut.key && e >= wmin;
  };
  const float xcut = cut.key ? logit_of_key<FMT>(cut.key) : -INFINITY;
  const double ecut = cut.key ? (greedy ? 1.0 : weight(xcut, mx, c)) : 0.0;
  const uint64_t wcut = ecut >= wmin ? fixed(ecut) : 0;

  // masses above the cut and ties at it, tile by tile
  const int tiles = (V + kTile - 1) >> kTileShift;
  __syncthreads();
  if (t < kMaxTiles) {
    s.tile_mass[t] = 0;
    s.tile_ties[t] = 0;
  }
  if (t == 0) s.token = 0;
  __syncthreads();
  for (int tile = 0; tile < tiles; tile++) {
    uint64_t sum = 0;
    uint32_t eq = 0;
    const int hi = min(V, (tile + 1) << kTileShift);
    for (int i = (tile << kTileShift) + t; i < hi; i += kThreads) {
      const uint32_t key = key_of<FMT>(x[i]);
      uint64_t w;
      if (key > cut.key && kept(key, logit<FMT>(x[i]), &w)) sum += w;
      eq += key == cut.key;
    }
    sum = wave_scan_u64(sum);
#pragma unroll
    for (int d = 32; d; d >>= 1) eq += __shfl_xor((int)eq, d, 64);
    if ((t & 63) == 63) {
      if (sum) atomicAdd((unsigned long long*)&s.tile_mass[tile], (unsigned long long)sum);
      if (eq) atomicAdd(&s.tile_ties[tile], eq);
    }
  }
  __syncthreads();
  uint64_t total = 0;
  uint32_t eq = 0;
  for (int i = 0; i < tiles; i++) {
    total += s.tile_mass[i] + wcut * (uint64_t)min(s.tile_ties[i], cut.ties - min(eq, cut.ties));
    eq += s.tile_ties[i];
  }
  const float uu = u[row];
  uint64_t goal = uu > 0.0f ? (uint64_t)fmin((double)uu * (double)total, 9.2e18) : 0;
  if (goal >= total) goal = total - 1;
  // the tile, then the thread (8 tokens in order each), then the token
  uint64_t before = 0;
  uint32_t eq_before = 0;
  int tile = 0;
  for (; tile < tiles - 1; tile++) {
    const uint64_t m = s.tile_mass[tile] +
                       wcut * (uint64_t)min(s.tile_ties[tile], cut.ties - min(eq_before, cut.ties));
    if (before + m > goal) break;
    before += m;
    eq_before += s.tile_ties[tile];
  }
  const int i0 = (tile << kTileShift) + t * (kTile / kThreads), i1 = min(V, i0 + kTile / kThreads);
  uint32_t mine = 0;
  for (int i = i0; i < i1; i++) mine += key_of<FMT>(x[i]) == cut.key;
  uint64_t all;
  uint32_t rank = eq_before + (uint32_t)block_scan_u64(mine, s.red, &all) - mine;
  uint64_t sum = 0;
  {
    uint32_t r = rank;
    for (int i = i0; i < i1; i++) {
      const uint32_t key = key_of<FMT>(x[i]);
      uint64_t w;
      if (key == cut.key)
        sum += r++ < cut.ties ? wcut : 0;
      else if (key > cut.key && kept(key, logit<FMT>(x[i]), &w))
        sum += w;
    }
  }
  uint64_t at = before + block_scan_u64(sum, s.red, &all) - sum;
  if (at <= goal && goal < at + sum) {
    for (int i = i0; i < i1; i++) {
      const uint32_t key = key_of<FMT>(x[i]);
      uint64_t w = 0;
      if (key == cut.key)
        w = rank++ < cut.ties ? wcut : 0;
      else if (!(key > cut.key && kept(key, logit<FMT>(x[i]), &w)))
        w = 0;
      if (at <= goal && goal < at + w) s.token = i;
      at += w;
    }
  }
  __syncthreads();
  if (t == 0) out[row] = s.token;
}

}  // namespace

extern "C" int aq_sample(const void* logits, int dtype, int64_t B, int64_t V, int64_t stride, const float* u,
                         const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                         float temperature0, int32_t top_k0, float top_p0, float min_p0, int64_t* tokens,
                         void* stream) {
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
  const dim3 grid((unsigned)B), block(kThreads);
  if (dtype == AQ_F16)
    hipLaunchKernelGGL(sample_kernel<AQ_F16>, grid, block, 0, s, (const uint16_t*)logits, (int)V, stride, u, set, tokens);
  else if (dtype == AQ_BF16)
    hipLaunchKernelGGL(sample_kernel<AQ_BF16>, grid, block, 0, s, (const uint16_t*)logits, (int)V, stride, u, set, tokens);
  else
    hipLaunchKernelGGL(sample_kernel<AQ_F32>, grid, block, 0, s, (const uint32_t*)logits, (int)V, stride, u, set, tokens);
  AQ_LAUNCH_CHECK("aq_sample");
  return AQ_OK;
}
