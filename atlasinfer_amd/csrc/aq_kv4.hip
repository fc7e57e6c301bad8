// aq_kv4.hip -- a key/value cache held in 4 bits: rows written (a prompt, or
// the step's own row inside the attention), read back, and attended to by a
// decode step.
//
// A row of D elements is cut into groups of 32; a group has its minimum m and
// a scale s = fp16((max - m) / 15), an element x the code
// c = min(rint((x - m) / s), 15) and the value s c + m: 5 bits an element, 5/16
// of an fp16 cache's bytes, which is what bounds a decode step at long
// contexts.  s is taken one step less where m + 15 s would round past the
// largest fp16 number; a group with an infinity or NaN reads as NaN.
//
// Layout (c = slots rounded up to 32):
//   k_codes  [B, Hkv, c, D / 2]         element d in nibble d % 8 of word d / 8
//   k_params [B, Hkv, c, D / 32, 2]     (s, m) fp16
//   v_codes  [B, Hkv, c / 32, 16 D]     per block of 32 slots the words [D / 64]
//            [r: 4][l: 16][e: 4], slot 16 t + 4 r + i of element 64 a + 16 e + l
//            in nibble 4 t + i of word (a, r, l, e)
//   v_params [B, Hkv, c / 32, D / 32, r: 4, i: 4, 4]   (s of t = 0, 1, m of t = 0, 1)
// so that both products of the attention find their operands where a lane of
// the 16 x 16 x 32 matrix instruction needs them: a lane has a piece of one key
// row (the contraction runs over its elements) and, of the values, eight slots
// of one element (the contraction runs over slots).
#include "aq_common.h"

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));

constexpr int kSlotBlock = 32;
constexpr uint16_t kNaN16 = 0x7E00;

struct Cache4 {
  uint8_t* kc;
  uint16_t* kp;
  uint8_t* vc;
  uint16_t* vp;
};

// Slot of position p: p itself while the cache has room; then, with sinks, the
// slots behind the first `sinks` are used over and over.
__device__ __forceinline__ int slot_of(int64_t p, int slots, int sinks) {
  if (p < slots) return (int)p;
  return sinks + (int)((uint32_t)(p - sinks) % (uint32_t)(slots - sinks));
}

// Offset (in fp16) of a block's parameters of (group, r, i).
__device__ __forceinline__ int v_param(int g, int r, int i) { return ((g * 4 + r) * 4 + i) * 4; }

// Eight consecutive elements of a group of 32 in four neighbouring lanes:
// the group's (s, m) as fp16 bits, and the lane's codes as eight nibbles.
__device__ __forceinline__ uint32_t quantize8(const uint16_t (&h)[8], uint16_t* s_bits, uint16_t* m_bits) {
  float x[8], lo = INFINITY, hi = -INFINITY, bad = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    x[i] = (float)bits_to_h(h[i]);
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    if ((h[i] & 0x7C00) == 0x7C00) bad = 1.0f;
  }
  lo = -xlane_level_max_f32<2>(xlane_level_max_f32<1>(-lo));
  hi = xlane_level_max_f32<2>(xlane_level_max_f32<1>(hi));
  bad = xlane_level_max_f32<2>(xlane_level_max_f32<1>(bad));
  f16 s16 = rn_h((hi - lo) / 15.0f);
  if (lo + 15.0f * (float)s16 >= 65520.0f) s16 = bits_to_h(h_to_bits(s16) - 1);
  const float s = (float)s16;
  // a / s as IEEE division gives it: one correction of a * RN(1 / s) (s has 11
  // significant bits, so RN(1 / s) is never the exception of that theorem)
  const float r = s > 0.0f ? 1.0f / s : 0.0f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float a = x[i] - lo, q0 = a * r;
    const float q = fmaf(fmaf(-q0, s, a), r, q0);
    w |= (uint32_t)fminf(rintf(q), 15.0f) << (4 * i);
  }
  *s_bits = bad != 0.0f ? kNaN16 : h_to_bits(s16);
  *m_bits = bad != 0.0f ? kNaN16 : h_to_bits(rn_h(lo));
  return bad != 0.0f ? 0 : w;
}

// ---------------------------------------------------------------- a prompt

// One workgroup per block of 32 slots of a sequence's head, 256 threads: 8
// elements a thread and step, keys first.  A slot takes the newest of the
// given positions that belongs to it; slots without one keep what they hold.
// The codes of the values are turned in LDS.
// Bound by its instructions, about 90 a thread for 8 elements (the vector units are
// four fifths busy): 4 sequences x 8 heads x 8192 positions of 128, 134 MB read and 42
// written, 49 us, 3.6 TB/s.  (Heads next to each other in the grid, several blocks a
// workgroup with the next one's rows on the way, extremes by pairs: all the same.)
template <int D>
__global__ __launch_bounds__(256) void kv4_store_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                        int64_t ksb, int64_t ksh, int64_t kss, int64_t vsb, int64_t vsh,
                                                        int64_t vss, int S, int64_t start,
                                                        const int64_t* __restrict__ lengths, Cache4 c, int Hkv,
                                                        int slots, int sinks, int first_block) {
  constexpr int TPR = D / 8;        // threads a row
  constexpr int RPS = 256 / TPR;    // rows a step
  const int t = threadIdx.x, j = blockIdx.y, b = blockIdx.z;
  const int blk = first_block + blockIdx.x, nblk = (slots + kSlotBlock - 1) / kSlotBlock;
  const int64_t len = lengths ? lengths[b] : S;
  const int64_t end = start + max((int64_t)0, min(len, (int64_t)S));  // positions [start, end)
  // the position (relative to start) that a slot takes, or -1
  auto source = [&](int slot) -> int64_t {
    if (slot >= slots || slot >= end) return -1;
    int64_t p = slot;
    if (sinks >= 0 && slot >= sinks) {
      const uint32_t W = slots - sinks;
      p += (int64_t)((uint32_t)(end - 1 - slot) / W) * W;
    }
    return p >= start ? p - start : -1;
  };
  __shared__ uint8_t codes[kSlotBlock][D];
  __shared__ uint8_t has[kSlotBlock];
  const int64_t head = (int64_t)b * Hkv + j;
  uint8_t* kc = c.kc + (head * nblk + blk) * (kSlotBlock * D / 2);
  uint16_t* kp = c.kp + (head * nblk + blk) * (kSlotBlock * (D / 32) * 2);
  uint8_t* vc = c.vc + (head * nblk + blk) * (16 * D);
  uint16_t* vp = c.vp + (head * nblk + blk) * ((D / 32) * 64);
  const uint16_t* kb = k + b * ksb + j * ksh;
  const uint16_t* vb = v + b * vsb + j * vsh;
  const int d = t % TPR * 8;
#pragma unroll
  for (int n = 0; n < kSlotBlock / RPS; n++) {
    const int r = n * RPS + t / TPR;
    const int64_t p = source(blk * kSlotBlock + r);
    uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
    if (p >= 0) {
      kx = *reinterpret_cast<const uint4*>(kb + p * kss + d);
      vx = *reinterpret_cast<const uint4*>(vb + p * vss + d);
    }
    uint16_t sb, mb;
    uint32_t w = quantize8(reinterpret_cast<const uint16_t(&)[8]>(kx), &sb, &mb);
    if (p >= 0) {
      *reinterpret_cast<uint32_t*>(kc + r * (D / 2) + d / 2) = w;
      if ((t & 3) == 0)
        *reinterpret_cast<uint32_t*>(kp + (r * (D / 32) + d / 32) * 2) = (uint32_t)sb | (uint32_t)mb << 16;
    }
    w = quantize8(reinterpret_cast<const uint16_t(&)[8]>(vx), &sb, &mb);
    if (p >= 0 && (t & 3) == 0) {
      uint16_t* q = vp + v_param(d / 32, (r & 15) >> 2, r & 3) + (r >> 4);
      q[0] = sb;
      q[2] = mb;
    }
    uint2 by;  // a code a byte
    by.x = (w & 0xF) | (w & 0xF0) << 4 | (w & 0xF00) << 8 | (w & 0xF000) << 12;
    w >>= 16;
    by.y = (w & 0xF) | (w & 0xF0) << 4 | (w & 0xF00) << 8 | (w & 0xF000) << 12;
    *reinterpret_cast<uint2*>(&codes[r][d]) = by;
    if (t % TPR == 0) has[r] = p >= 0;
  }
  __syncthreads();
  for (int i = t; i < 4 * D; i += 256) {
    // word i of the block: (a, r, l, e)
    const int e = i & 3, l = (i >> 2) & 15, r = (i >> 6) & 3, a = i >> 8;
    const int el = a * 64 + e * 16 + l;
    uint32_t w = 0, mask = 0;
#pragma unroll
    for (int n = 0; n < 8; n++) {
      const int slot = 16 * (n >> 2) + 4 * r + (n & 3);
      if (has[slot]) {
        w |= (uint32_t)codes[slot][el] << (4 * n);
        mask |= 0xFu << (4 * n);
      }
    }
    uint32_t* q = reinterpret_cast<uint32_t*>(vc) + i;
    if (mask == 0xFFFFFFFFu)
      *q = w;
    else if (mask)
      *q = (*q & ~mask) | w;
  }
}

// Slots [0, count) back in fp16: fp16(s c + m), the product exact in f32.  Bound by
// HBM: the case above, 42 MB read and 134 written, 27 us, 6.5 TB/s.
template <int D>
__global__ __launch_bounds__(256) void kv4_load_kernel(Cache4 c, int slots, int count, uint16_t* __restrict__ k,
                                                       uint16_t* __restrict__ v) {
  constexpr int TPR = D / 8, RPS = 256 / TPR;
  const int t = threadIdx.x, blk = blockIdx.x, nblk = (slots + kSlotBlock - 1) / kSlotBlock;
  const int64_t head = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
  const uint8_t* kc = c.kc + (head * nblk + blk) * (kSlotBlock * D / 2);
  const uint16_t* kp = c.kp + (head * nblk + blk) * (kSlotBlock * (D / 32) * 2);
  const uint8_t* vc = c.vc + (head * nblk + blk) * (16 * D);
  const uint16_t* vp = c.vp + (head * nblk + blk) * ((D / 32) * 64);
  __shared__ uint8_t codes[kSlotBlock][D];
  for (int i = t; i < 4 * D; i += 256) {
    const int e = i & 3, l = (i >> 2) & 15, r = (i >> 6) & 3, a = i >> 8;
    const uint32_t w = reinterpret_cast<const uint32_t*>(vc)[i];
#pragma unroll
    for (int n = 0; n < 8; n++) codes[16 * (n >> 2) + 4 * r + (n & 3)][a * 64 + e * 16 + l] = (w >> (4 * n)) & 15;
  }
  __syncthreads();
  const int d = t % TPR * 8;
#pragma unroll
  for (int n = 0; n < kSlotBlock / RPS; n++) {
    const int r = n * RPS + t / TPR;
    const int64_t slot = (int64_t)blk * kSlotBlock + r;
    if (slot >= count) continue;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(kc + r * (D / 2) + d / 2);
    const uint16_t* q = kp + (r * (D / 32) + d / 32) * 2;
    float s = (float)bits_to_h(q[0]), m = (float)bits_to_h(q[1]);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
      o[i] = (uint32_t)h_to_bits(rn_h(s * (float)((w >> (8 * i)) & 15) + m)) |
             (uint32_t)h_to_bits(rn_h(s * (float)((w >> (8 * i + 4)) & 15) + m)) << 16;
    *reinterpret_cast<uint4*>(k + (head * count + slot) * D + d) = make_uint4(o[0], o[1], o[2], o[3]);
    q = vp + v_param(d / 32, (r & 15) >> 2, r & 3) + (r >> 4);
    s = (float)bits_to_h(q[0]);
    m = (float)bits_to_h(q[2]);
#pragma unroll
    for (int i = 0; i < 4; i++)
      o[i] = (uint32_t)h_to_bits(rn_h(s * (float)codes[r][d + 2 * i] + m)) |
             (uint32_t)h_to_bits(rn_h(s * (float)codes[r][d + 2 * i + 1] + m)) << 16;
    *reinterpret_cast<uint4*>(v + (head * count + slot) * D + d) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ---------------------------------------------------------------- a decode step

// Splitting of the slots among workgroups: up to 16 blocks are one span of up to
// 8 waves, one block each in turn (16 sequences x 8 heads at 300 of 512: 7.3 us,
// in 4 spans 10.7; one sequence of 24 blocks 10.5 against 8.8, so split).  Else
// spans of nt blocks and 4 waves, nt the smallest power of two from 4 that leaves
// at most 64 spans a head and at most 1024 workgroups, or reaches 32 (8 sequences
// x 8 heads at 4000: 9 spans of 16 17.4 us, 17 of 8 19.7; 32 sequences of up to
// 16384: 16 spans of 32 94 us, 8 of 64 96, 4 of 128 107, 32 of 16 103).
constexpr int kMaxWaves4 = 8;
constexpr int64_t kOneSpan4 = 16, kFirstSpan4 = 4, kLongSpan4 = 32;
constexpr int64_t kMaxSpans4 = 64, kMaxGroups4 = 1024;
constexpr int kHeads = 16;  // query heads a workgroup takes: a tile's columns
constexpr float kCodeUnit = 1.0f / (1 << 24);  // of the codes in the scores' product

struct Split4 {
  int64_t nt, ns, nw, hb, part_floats, bytes;  // blocks a span, spans, waves, head tiles
};

inline Split4 split4_of(int64_t B, int64_t Hkv, int64_t G, int64_t D, int64_t slots) {
  Split4 sp;
  const int64_t blocks = (slots + kSlotBlock - 1) / kSlotBlock;
  sp.hb = (G + kHeads - 1) / kHeads;
  auto spans = [&](int64_t nt) { return (blocks + nt - 1) / nt; };
  sp.nt = kFirstSpan4;
  while (sp.nt < blocks && (spans(sp.nt) > kMaxSpans4 || (B * Hkv * sp.hb * spans(sp.nt) > kMaxGroups4 && sp.nt < kLongSpan4)))
    sp.nt *= 2;
  if (blocks <= kOneSpan4) sp.nt = blocks;
  sp.ns = spans(sp.nt);
  sp.nw = std::min<int64_t>(sp.ns == 1 ? kMaxWaves4 : 4, std::min(blocks, sp.nt));
  sp.part_floats = kHeads * D + 2 * kHeads;
  sp.bytes = sp.ns > 1 ? B * Hkv * sp.hb * sp.ns * sp.part_floats * 4 : 0;
  return sp;
}

__device__ __forceinline__ f16 turned(f16 x, f16 partner, bool lo, uint16_t c, uint16_t s) {
  const float r = lo ? -(float)partner : (float)partner;
  const f16 a = rn_h((float)x * (float)bits_to_h(c));
  const f16 b2 = rn_h(r * (float)bits_to_h(s));
  return rn_h((float)a + (float)b2);
}

// Nibbles n and n + 4 of a word, n = 0 .. 3, as a pair of fp16 numbers 0 .. 15:
// under the exponent of 1024 a nibble in the lowest bits counts 1 each, one
// four bits up 16 each; taking the 1024 away again is exact.  `magic` is 1024
// twice in a vector register (a vector instruction takes one scalar operand, and
// the mask is that), so that mask and exponent are one instruction.
__device__ __forceinline__ half2v pair_of(uint32_t w, int n, uint32_t magic) {
  const half2v big = {(f16)1024.0f, (f16)1024.0f}, sixteenth = {(f16)0.0625f, (f16)0.0625f}, off = {(f16)-64.0f, (f16)-64.0f};
  if (n & 2) w >>= 8;
  if (n & 1) return __builtin_elementwise_fma(__builtin_bit_cast(half2v, (w & 0x00F000F0u) | magic), sixteenth, off);
  return __builtin_bit_cast(half2v, (w & 0x000F000Fu) | magic) - big;
}

// The same pair as it is: a nibble in the lowest bits is a subnormal number, 2^-24
// times the nibble, which the matrix instructions take like any other.
// (The highest nibbles come by one shift of both halves of the word.)
__device__ __forceinline__ uint32_t small_pair_of(uint32_t w, int n) {
  if (n == 3) return __builtin_bit_cast(uint32_t, __builtin_bit_cast(ushort2v, w) >> (uint16_t)12);
  return (w >> (4 * n)) & 0x000F000Fu;
}

// Words n of the lanes (l, r), r = lane / 16, a group of keys each (D = 128: group r
// in words 0 .. 3; D = 64: group r / 2 in words 0, 1), exchanged among the r so that
// word n is of group n in every lane: word_of says which word of the group.
template <int D>
__device__ __forceinline__ void groups_apart(u32x4& w) {
  if constexpr (D == 128) {
    const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    w = u32x4{c[0], c[1], d[0], d[1]};
  } else {
    const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[1], false, false);
    w = u32x4{a[0], a[1], 0, 0};
  }
}
template <int D>
__device__ __forceinline__ int word_of(int r) {
  return D == 128 ? r : 2 * (r & 1) + (r >> 1);
}

// The pair of lane n of each row of 16 lanes, in the whole row: one instruction for
// both words (the builtin has one word only, the intrinsic behind it two).
extern "C" __device__ uint64_t update_dpp_u64(uint64_t old, uint64_t x, int ctrl, int rows, int banks,
                                              bool bound) __asm("llvm.amdgcn.update.dpp.i64");
template <int N>
__device__ __forceinline__ uint2 row16_bcast(uint2 x) {
  const uint64_t v = update_dpp_u64(0, (uint64_t)x.y << 32 | x.x, 0x150 + N, 0xF, 0xF, true);  // row_newbcast
  return make_uint2((uint32_t)v, (uint32_t)(v >> 32));
}

__device__ __forceinline__ float max_quarters(float x) { return xlane_level_max_f32<6>(xlane_level_max_f32<5>(x)); }

// Workgroup (j, b, z) takes key/value head j (and head tile) of sequence b and
// blocks z nt .. of its slots; wave w every nw-th of them.  The last spans, which
// short sequences do not have, come first: the workgroups that have nothing to do are
// gone before the GPU runs empty (lengths of 1 to 16384: with first spans first 3 us more).
// One step is a block of 32 slots: scores of 2 x 16 slots against up to 16 query
// heads (mfma 16 x 16 x 32, keys as rows, so that a lane's results are 2 x 4 slots
// of one head), the running softmax of a head in the four lanes that hold it, the
// numerators as the second product's operand, which they are without an exchange,
// and the values' rows.
//   Scores: the products of one group's codes, whole numbers times 2^-24 as fp16,
// with the query are exact to f32 and scaled there; the minima meet the sums of the
// query (times 2^-24 too) in a product of f32 (16 x 16 x 4).  (Codes raised by 1024 and
// 64, one instruction a pair fewer, whose share was taken away again after the product:
// for queries far from zero on average, as biases make them, scores were off by 2e-2.)
// Keys rounded to fp16 (a fused multiply-add a
// pair, the scales then inside the product) gave 4.2e-4 of the result against 2.1e-4
// of the output's own rounding, at 88 us for the long case below, no less.
//   Numerators are two fp16 numbers each, the second what the first leaves over: with
// one alone the error is 3.0e-4, the long case 4 us shorter.  With both 2.6e-4: what is left beside
// the output's rounding is that of the values s c + m to fp16, once each (fma).  The
// denominator is the product of the same numerators with ones.
// Bound by HBM and by the instructions together: a step of 32 slots of D = 128 is 310
// vector and 28 matrix instructions a wave for 5 KiB (32 sequences x 8 heads of up to
// 16384 slots, half of them in use: 336 MB in 88.5 us, 3.8 TB/s; all of 8192, two caches
// in turn: 87, 3.9; 32 x 32 heads of 64: 167, 4.0).
template <int D>
__global__ __launch_bounds__(64 * kMaxWaves4, D == 64 ? 4 : 3) void kv4_attention_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ k_new, const uint16_t* __restrict__ v_new, Cache4 c,
    const int64_t* __restrict__ pos_p, int pos_stride, int H, int Hkv, int hb, int slots, int sinks, float scale2,
    float q_scale, const uint16_t* __restrict__ rcos, const uint16_t* __restrict__ rsin, int64_t max_pos, int nt,
    int ns, float* __restrict__ part, uint16_t* __restrict__ out) {
  constexpr int NK = D / 32;   // k-steps of the scores, groups of a row
  constexpr int ND = D / 16;   // row tiles of the output
  const int t = threadIdx.x, ln = t & 63, nw = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int j = blockIdx.x / hb, h0 = blockIdx.x % hb * kHeads, b = blockIdx.y;
  const int z = ns - 1 - (int)blockIdx.z;
  const int G = H / Hkv, heads = min(kHeads, G - h0);
  const int64_t pos = pos_p[(int64_t)b * pos_stride];
  if (pos < 0 || pos >= max_pos) return;
  const int slot = slot_of(pos, slots, sinks);
  const int last = (int)min(pos, (int64_t)slots - 1);  // the last slot in use
  const int blk0 = z * nt;
  if (blk0 * kSlotBlock > last) return;
  const int blk1 = min(blk0 + nt, last / kSlotBlock + 1);
  const int nact = last / (kSlotBlock * nt) + 1;
  const int nblk = (slots + kSlotBlock - 1) / kSlotBlock;
  const int64_t head = (int64_t)b * Hkv + j;
  uint8_t* kc = c.kc + head * nblk * (kSlotBlock * D / 2);
  uint16_t* kp = c.kp + head * nblk * (kSlotBlock * NK * 2);
  uint8_t* vc = c.vc + head * nblk * (16 * D);
  uint16_t* vp = c.vp + head * nblk * (NK * 64);
  const int l = ln & 15, r = ln >> 4;
  const bool owner = slot / (kSlotBlock * nt) == z && h0 == 0;  // writes the new row
  const bool holds = slot / (kSlotBlock * nt) == z;

  // a step's loads: whole rows and blocks, in the buffers whatever the step
  struct Step {
    u32x4 k[2], v[ND / 4];
    uint32_t kpar[2], kscale[2];  // (s, m) of (row l, group r % NK) and of (row 4 r + l % 4, group l / 4)
    uint2 vpar;
  };
  const int kr = r * (D / 8);
  auto load = [&](Step& x, int blk) {
    blk = min(blk, nblk - 1);
    const uint8_t* kb = kc + (int64_t)blk * (kSlotBlock * D / 2) + l * (D / 2) + kr;
    const uint16_t* pb = kp + (int64_t)blk * (kSlotBlock * NK * 2) + (l * NK + r % NK) * 2;
    const uint16_t* sb = kp + (int64_t)blk * (kSlotBlock * NK * 2) + ((4 * r + (l & 3)) * NK + (l >> 2) % NK) * 2;
    const uint8_t* vb = vc + (int64_t)blk * (16 * D) + ln * 16;
#pragma unroll
    for (int tt = 0; tt < 2; tt++) {
      if constexpr (D == 128) {
        x.k[tt] = *reinterpret_cast<const u32x4*>(kb + tt * 16 * (D / 2));
      } else {
        const uint2 y = *reinterpret_cast<const uint2*>(kb + tt * 16 * (D / 2));
        x.k[tt] = u32x4{y.x, y.y, 0, 0};
      }
      x.kpar[tt] = *reinterpret_cast<const uint32_t*>(pb + tt * 16 * NK * 2);
      x.kscale[tt] = *reinterpret_cast<const uint32_t*>(sb + tt * 16 * NK * 2);
    }
#pragma unroll
    for (int e = 0; e < ND / 4; e++) x.v[e] = *reinterpret_cast<const u32x4*>(vb + e * 1024);
    x.vpar = *reinterpret_cast<const uint2*>(vp + (int64_t)blk * (NK * 64) + v_param((l >> 2) % NK, r, l & 3));
  };
  // the first rows are on their way while the queries are staged
  Step sa, sb;
  load(sa, blk0 + wave);
  __shared__ __attribute__((aligned(16))) uint16_t qs[kHeads][D];
  __shared__ uint32_t new_k[D / 8], new_v[D / 8], new_kp[NK], new_vp[NK];
  extern __shared__ float res[];  // [nw][kHeads][D + 2]

  const uint16_t* cs = rcos ? rcos + pos * D : nullptr;
  const uint16_t* sn = rsin ? rsin + pos * D : nullptr;
  // eight elements of a row, scaled and rotated; all loads first
  auto prepared = [&](const uint16_t* row, int d, float f, bool rot, uint16_t(&x)[8]) {
    auto half = [](const uint4& w, int i) { return bits_to_h((uint16_t)((&w.x)[i >> 1] >> (16 * (i & 1)))); };
    const uint4 own = *reinterpret_cast<const uint4*>(row + d);
    if (rot) {
      const uint4 other = *reinterpret_cast<const uint4*>(row + (d + D / 2) % D);
      const uint4 cv = *reinterpret_cast<const uint4*>(cs + d), sv = *reinterpret_cast<const uint4*>(sn + d);
#pragma unroll
      for (int i = 0; i < 8; i++)
        x[i] = h_to_bits(turned(rn_h((float)half(own, i) * f), rn_h((float)half(other, i) * f), d < D / 2,
                                h_to_bits(half(cv, i)), h_to_bits(half(sv, i))));
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = h_to_bits(rn_h((float)half(own, i) * f));  // f = 1 is exact
    }
  };
  const uint16_t* qb = q + ((int64_t)b * H + (int64_t)j * G + h0) * D;
  for (int i = t; i < kHeads * (D / 8); i += 64 * nw) {
    const int g = i / (D / 8), d = i % (D / 8) * 8;
    uint16_t x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (g < heads) prepared(qb + g * D, d, q_scale, rcos != nullptr, x);
    uint4 w;
#pragma unroll
    for (int n = 0; n < 4; n++) (&w.x)[n] = (uint32_t)x[2 * n] | (uint32_t)x[2 * n + 1] << 16;
    *reinterpret_cast<uint4*>(&qs[g][d]) = w;
  }
  if (holds && t < 64) {
    // the step's own row, keys in the wave's lower half, values in its upper
    const bool val = t >= 32;
    const int d = (t & 31) * 8;
    if (d < D) {
      uint16_t x[8];
      prepared((val ? v_new : k_new) + head * D, d, 1.0f, !val && rcos, x);
      uint16_t sb, mb;
      const uint32_t w = quantize8(x, &sb, &mb);
      (val ? new_v : new_k)[d / 8] = w;
      if ((t & 3) == 0) (val ? new_vp : new_kp)[d / 32] = (uint32_t)sb | (uint32_t)mb << 16;
    }
  }
  __syncthreads();

  // the queries as the scores' second operand: head l, elements 32 kk +
  // 8 word_of(r) + the order in which pair_of gives a word's nibbles; the sum of the
  // queries over group r, which the keys' minima multiply, in the codes' unit
  half8v qv[NK];
  float qsum = 0.0f;
#pragma unroll
  for (int kk = 0; kk < NK; kk++) {
    half8v ones;
#pragma unroll
    for (int n = 0; n < 8; n++) {
      qv[kk][n] = bits_to_h(qs[l][32 * kk + 8 * word_of<D>(r) + (n >> 1) + 4 * (n & 1)]);
      ones[n] = (f16)1.0f;
    }
    const float b = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, qv[kk], float4v{0, 0, 0, 0}, 0, 0, 0)[0];
    if (r == kk) qsum = b * kCodeUnit;
  }

  float4v o[ND], den;
#pragma unroll
  for (int e = 0; e < ND; e++) o[e] = float4v{0, 0, 0, 0};
  den = float4v{0, 0, 0, 0};
  float m = -INFINITY;
  uint32_t magic = 0x64006400u;
  asm volatile("" : "+v"(magic));
  half8v ones;
#pragma unroll
  for (int n = 0; n < 8; n++) ones[n] = (f16)1.0f;

  auto step = [&](Step& y, int blk) {
    uint2& vpar = y.vpar;
    const int s0 = blk * kSlotBlock;
    if (slot / kSlotBlock == blk) {
      // the step's own row replaces what the slot held, here and in memory
      const int at = slot % kSlotBlock, n = (at >> 4) * 4 + (at & 3);
#pragma unroll
      for (int tt = 0; tt < 2; tt++)
        if (16 * tt + l == at) {
#pragma unroll
          for (int kk = 0; kk < NK; kk++) {
            y.k[tt][kk] = new_k[r * (D / 32) + kk];
            if (owner) *reinterpret_cast<uint32_t*>(kc + (int64_t)slot * (D / 2) + kr + kk * 4) = y.k[tt][kk];
          }
          y.kpar[tt] = new_kp[r % NK];
          if (owner && r < NK) *reinterpret_cast<uint32_t*>(kp + ((int64_t)slot * NK + r) * 2) = y.kpar[tt];
        }
#pragma unroll
      for (int tt = 0; tt < 2; tt++)
        if (16 * tt + 4 * r + (l & 3) == at) y.kscale[tt] = new_kp[(l >> 2) % NK];
      if (r == ((at & 15) >> 2)) {
#pragma unroll
        for (int e = 0; e < ND; e++) {
          const int d = e * 16 + l;
          const uint32_t code = (new_v[d / 8] >> (4 * (d & 7))) & 15;
          const uint32_t w = (y.v[e >> 2][e & 3] & ~(15u << (4 * n))) | code << (4 * n);
          y.v[e >> 2][e & 3] = w;
          if (owner) *reinterpret_cast<uint32_t*>(vc + (int64_t)blk * (16 * D) + (e >> 2) * 1024 + ln * 16 + (e & 3) * 4) = w;
        }
        if ((l & 3) == (at & 3)) {
          const uint32_t p = new_vp[(l >> 2) % NK];
          const int sh = (at >> 4) * 16;
          vpar.x = (vpar.x & ~(0xFFFFu << sh)) | (p & 0xFFFF) << sh;
          vpar.y = (vpar.y & ~(0xFFFFu << sh)) | (p >> 16) << sh;
          if (owner && l < 4 * NK)
            *reinterpret_cast<uint2*>(vp + (int64_t)blk * (NK * 64) + v_param(l >> 2, r, l & 3)) = vpar;
        }
      }
    }
    const bool edge = s0 + kSlotBlock - 1 > last;
    if (edge) {
      // slots past the last in use: whatever they hold, their values count as 0
      const int i = l & 3;
      if (s0 + 4 * r + i > last) vpar.x &= 0xFFFF0000u, vpar.y &= 0xFFFF0000u;
      if (s0 + 16 + 4 * r + i > last) vpar.x &= 0xFFFFu, vpar.y &= 0xFFFFu;
    }
    // q . (s c + m) = sum over groups of s (q . c) + m sum(q): products of whole numbers
    // with q, scaled in f32
    float4v acc[2];
    float s_of[2];
#pragma unroll
    for (int tt = 0; tt < 2; tt++) {
      groups_apart<D>(y.k[tt]);
      s_of[tt] = (float)bits_to_h((uint16_t)y.kscale[tt]);
      acc[tt] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)bits_to_h((uint16_t)(y.kpar[tt] >> 16)), qsum, float4v{0, 0, 0, 0}, 0, 0, 0);
    }
    auto group = [&](auto gc) {
      constexpr int g = decltype(gc)::value;
      float4v d[2];
#pragma unroll
      for (int tt = 0; tt < 2; tt++) {
        u32x4 a;
#pragma unroll
        for (int n = 0; n < 4; n++) a[n] = small_pair_of(y.k[tt][g], n);
        d[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, a), qv[g], float4v{0, 0, 0, 0}, 0, 0, 0);
      }
      auto of_slot = [&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const uint2 p = row16_bcast<4 * g + i>(make_uint2(__builtin_bit_cast(uint32_t, s_of[0]), __builtin_bit_cast(uint32_t, s_of[1])));
        acc[0][i] = fmaf(__builtin_bit_cast(float, p.x), d[0][i], acc[0][i]);
        acc[1][i] = fmaf(__builtin_bit_cast(float, p.y), d[1][i], acc[1][i]);
      };
      of_slot(std::integral_constant<int, 0>{});
      of_slot(std::integral_constant<int, 1>{});
      of_slot(std::integral_constant<int, 2>{});
      of_slot(std::integral_constant<int, 3>{});
    };
    group(std::integral_constant<int, 0>{});
    group(std::integral_constant<int, 1>{});
    if constexpr (NK == 4) {
      group(std::integral_constant<int, 2>{});
      group(std::integral_constant<int, 3>{});
    }
    float x[8];
#pragma unroll
    for (int n = 0; n < 8; n++) x[n] = acc[n >> 2][n & 3];
    if (edge) {
      asm volatile("");  // a branch: few blocks are at the edge
#pragma unroll
      for (int n = 0; n < 8; n++)
        if (s0 + 16 * (n >> 2) + 4 * r + (n & 3) > last) x[n] = -INFINITY;
    }
    float mx = x[0];
#pragma unroll
    for (int n = 1; n < 8; n++) mx = fmaxf(mx, x[n]);
    mx = fmaxf(m, max_quarters(mx) * scale2);
    if (__ballot(mx != m)) {
      const float f = __builtin_amdgcn_exp2f(m - mx);  // every block has a slot in use: mx is a number
#pragma unroll
      for (int e = 0; e < ND; e++) o[e] *= f;
      den *= f;
      m = mx;
    }
    // numerators, slot pairs (t = 0, 1) as pair_of gives the values'
    half8v pv, pl;
#pragma unroll
    for (int n = 0; n < 8; n++) {
      const float p = __builtin_amdgcn_exp2f(fmaf(x[4 * (n & 1) + (n >> 1)], scale2, -m));
      pv[n] = rn_h(p);
      pl[n] = rn_h(p - (float)pv[n]);
    }
    den = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pv, den, 0, 0, 0);
    den = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl, den, 0, 0, 0);
    auto values = [&](auto gc) {
      constexpr int g = decltype(gc)::value;
      half2v s2[4], m2[4];
      auto of_slot = [&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const uint2 p = row16_bcast<4 * g + i>(vpar);
        s2[i] = __builtin_bit_cast(half2v, p.x);
        m2[i] = __builtin_bit_cast(half2v, p.y);
      };
      of_slot(std::integral_constant<int, 0>{});
      of_slot(std::integral_constant<int, 1>{});
      of_slot(std::integral_constant<int, 2>{});
      of_slot(std::integral_constant<int, 3>{});
#pragma unroll
      for (int e = 2 * g; e < 2 * g + 2; e++) {
        half8v a;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const half2v v2 = __builtin_elementwise_fma(pair_of(y.v[e >> 2][e & 3], i, magic), s2[i], m2[i]);
          a[2 * i] = v2.x;
          a[2 * i + 1] = v2.y;
        }
        o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pv, o[e], 0, 0, 0);
        o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, o[e], 0, 0, 0);
      }
    };
    values(std::integral_constant<int, 0>{});
    values(std::integral_constant<int, 1>{});
    if constexpr (NK == 4) {
      values(std::integral_constant<int, 2>{});
      values(std::integral_constant<int, 3>{});
    }
  };
  for (int blk = blk0 + wave; blk < blk1; blk += 2 * nw) {
    load(sb, blk + nw);
    __builtin_amdgcn_sched_barrier(0);
    step(sa, blk);
    load(sa, blk + 2 * nw);
    __builtin_amdgcn_sched_barrier(0);
    if (blk + nw < blk1) step(sb, blk + nw);
  }

  // the waves' sums meet: maximum over the waves, each scaled to it, in order
  constexpr int RS = D + 2;
  if (l < heads) {
    float* w = res + (wave * kHeads + l) * RS;
#pragma unroll
    for (int e = 0; e < ND; e++)
#pragma unroll
      for (int i = 0; i < 4; i++) w[16 * e + 4 * r + i] = o[e][i];
    if (r == 0) {
      w[D] = m;
      w[D + 1] = den[0];
    }
  }
  __syncthreads();
  const int na = min(nw, blk1 - blk0);  // waves that had a block
  uint16_t* ob = out + ((int64_t)b * H + (int64_t)j * G + h0) * D;
  float* sp = part + (((int64_t)b * gridDim.x + blockIdx.x) * ns + z) * (kHeads * D + 2 * kHeads);
  for (int i = t; i < heads * D; i += 64 * nw) {
    const int g = i / D, d = i % D;
    float mx = -INFINITY;
    for (int w = 0; w < na; w++) mx = fmaxf(mx, res[(w * kHeads + g) * RS + D]);
    float num = 0.0f, sum = 0.0f;
    for (int w = 0; w < na; w++) {
      const float* y = res + (w * kHeads + g) * RS;
      const float f = y[D] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(y[D] - mx);
      num = fmaf(y[d], f, num);
      sum = fmaf(y[D + 1], f, sum);
    }
    if (nact == 1) {
      ob[i] = h_to_bits(rn_h(num / sum));
    } else {
      sp[i] = num;
      if (d == 0) {
        sp[kHeads * D + g] = mx;
        sp[kHeads * D + kHeads + g] = sum;
      }
    }
  }
}

// Merges the spans' (maximum, denominator, sum) of one query head: every wave
// has all spans' (m, l), one a lane; 256 / D groups of threads take every
// (256 / D)-th span in order, eight loads in flight, and are added in order.
template <int D>
__global__ __launch_bounds__(256) void kv4_combine_kernel(const int64_t* __restrict__ pos_p, int pos_stride, int H,
                                                          int Hkv, int hb, int slots, int64_t max_pos, int nt, int ns,
                                                          const float* __restrict__ part, uint16_t* __restrict__ out) {
  constexpr int PF = kHeads * D + 2 * kHeads;
  constexpr int NG = 256 / D;
  const int h = blockIdx.x, b = blockIdx.y, t = threadIdx.x, grp = t / D, d = t % D, z = t & 63;
  const int G = H / Hkv, j = h / G, tile = h % G / kHeads, g = h % G % kHeads;
  const int64_t pos = pos_p[(int64_t)b * pos_stride];
  if (pos < 0 || pos >= max_pos) return;
  const int nact = (int)min(pos, (int64_t)slots - 1) / (kSlotBlock * nt) + 1;
  if (nact == 1) return;  // that span wrote out
  const float* pk = part + (((int64_t)b * Hkv + j) * hb + tile) * ns * PF;
  __shared__ float f[kMaxSpans4], sum[NG][D];
  const float m = z < nact ? pk[(int64_t)z * PF + kHeads * D + g] : -INFINITY;
  const float l = z < nact ? pk[(int64_t)z * PF + kHeads * D + kHeads + g] : 0.0f;
  const float mx = wave_group_max_f32<64>(m);
  const float e = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
  const float den = wave_group_sum_f32<64>(l * e);
  if (t < 64) f[z] = e;
  __syncthreads();
  float num = 0.0f;
  for (int z0 = grp; z0 < nact; z0 += 8 * NG) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = z0 + NG * k < nact ? pk[(int64_t)(z0 + NG * k) * PF + g * D + d] : 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (z0 + NG * k < nact) num = fmaf(v[k], f[z0 + NG * k], num);
  }
  sum[grp][d] = num;
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int k = 1; k < NG; k++) num += sum[k][d];
    out[((int64_t)b * H + h) * D + d] = h_to_bits(rn_h(num / den));
  }
}

int check_cache4(const char* what, const void* kc, const void* kp, const void* vc, const void* vp, int64_t B, int64_t Hkv,
                 int64_t D, int64_t slots) {
  AQ_CHECK_ARG(kc && kp && vc && vp, "%s: null pointer", what);
  AQ_CHECK_ARG(D == 64 || D == 128, "%s: head dim %lld (64 or 128 supported)", what, (long long)D);
  AQ_CHECK_ARG(B > 0 && B <= 65535 && Hkv > 0 && Hkv <= 65535 && slots > 0 && slots <= (1 << 24),
               "%s: sizes out of range", what);
  AQ_CHECK_ARG((uintptr_t)kc % 16 == 0 && (uintptr_t)kp % 16 == 0 && (uintptr_t)vc % 16 == 0 && (uintptr_t)vp % 16 == 0,
               "%s: the cache's buffers must be 16-byte aligned", what);
  return AQ_OK;
}

}  // namespace

extern "C" int aq_kv4_store(const void* k, const void* v, int64_t B, int64_t Hkv, int64_t S, int64_t D,
                            const int64_t* k_strides, const int64_t* v_strides, int64_t start, const int64_t* lengths,
                            void* k_codes, void* k_params, void* v_codes, void* v_params, int64_t slots, int64_t sinks,
                            void* stream) {
  AQ_CHECK_ARG(k && v && k_strides && v_strides, "aq_kv4_store: null pointer");
  if (const int rc = check_cache4("aq_kv4_store", k_codes, k_params, v_codes, v_params, B, Hkv, D, slots)) return rc;
  AQ_CHECK_ARG(sinks >= -1 && sinks < slots, "aq_kv4_store: %lld sinks in %lld slots", (long long)sinks, (long long)slots);
  AQ_CHECK_ARG(S > 0 && start >= 0 && S <= INT32_MAX && start <= INT32_MAX - S,
               "aq_kv4_store: positions %lld .. +%lld out of range", (long long)start, (long long)S);
  AQ_CHECK_ARG(sinks >= 0 || start + S <= slots, "aq_kv4_store: positions up to %lld in %lld slots",
               (long long)(start + S), (long long)slots);
  for (int i = 0; i < 3; i++)
    AQ_CHECK_ARG(k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0, "aq_kv4_store: strides must be multiples of 8");
  AQ_CHECK_ARG((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)lengths % 8 == 0,
               "aq_kv4_store: k and v must be 16-byte aligned");
  const int64_t nblk = aq::ceil_div(slots, kSlotBlock);
  // blocks without one of the positions are left out, where no slot is used again
  const int64_t first = start + S <= slots ? start / kSlotBlock : 0;
  const int64_t end = start + S <= slots ? aq::ceil_div(start + S, kSlotBlock) : nblk;
  const Cache4 c = {(uint8_t*)k_codes, (uint16_t*)k_params, (uint8_t*)v_codes, (uint16_t*)v_params};
  const dim3 grid((unsigned)(end - first), (unsigned)Hkv, (unsigned)B);
#define AQ_KV4_STORE(DD)                                                                                              \
  hipLaunchKernelGGL((kv4_store_kernel<DD>), grid, dim3(256), 0, (hipStream_t)stream, (const uint16_t*)k,             \
                     (const uint16_t*)v, k_strides[0], k_strides[1], k_strides[2], v_strides[0], v_strides[1],        \
                     v_strides[2], (int)S, start, lengths, c, (int)Hkv, (int)slots, (int)sinks, (int)first)
  if (D == 64) AQ_KV4_STORE(64);
  else AQ_KV4_STORE(128);
#undef AQ_KV4_STORE
  AQ_LAUNCH_CHECK("aq_kv4_store");
  return AQ_OK;
}

extern "C" int aq_kv4_load(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params,
                           int64_t B, int64_t Hkv, int64_t D, int64_t slots, int64_t count, void* k, void* v,
                           void* stream) {
  AQ_CHECK_ARG(k && v, "aq_kv4_load: null pointer");
  if (const int rc = check_cache4("aq_kv4_load", k_codes, k_params, v_codes, v_params, B, Hkv, D, slots)) return rc;
  AQ_CHECK_ARG(count > 0 && count <= slots, "aq_kv4_load: %lld of %lld slots", (long long)count, (long long)slots);
  AQ_CHECK_ARG((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, "aq_kv4_load: k and v must be 16-byte aligned");
  const Cache4 c = {(uint8_t*)k_codes, (uint16_t*)k_params, (uint8_t*)v_codes, (uint16_t*)v_params};
  const dim3 grid((unsigned)aq::ceil_div(count, kSlotBlock), (unsigned)Hkv, (unsigned)B);
  if (D == 64)
    hipLaunchKernelGGL((kv4_load_kernel<64>), grid, dim3(256), 0, (hipStream_t)stream, c, (int)slots, (int)count, (uint16_t*)k, (uint16_t*)v);
  else
    hipLaunchKernelGGL((kv4_load_kernel<128>), grid, dim3(256), 0, (hipStream_t)stream, c, (int)slots, (int)count, (uint16_t*)k, (uint16_t*)v);
  AQ_LAUNCH_CHECK("aq_kv4_load");
  return AQ_OK;
}

extern "C" int64_t aq_kv4_attention_workspace(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t slots) {
  if (B <= 0 || Hkv <= 0 || H <= 0 || H % Hkv != 0 || (D != 64 && D != 128) || slots <= 0) return -1;
  return split4_of(B, Hkv, H / Hkv, D, slots).bytes;
}

extern "C" int aq_kv4_attention(const void* q, const void* k_new, const void* v_new, void* k_codes, void* k_params,
                                void* v_codes, void* v_params, const int64_t* pos, int64_t pos_stride, int64_t B,
                                int64_t H, int64_t Hkv, int64_t D, int64_t slots, int64_t sinks, float scale,
                                float q_scale, const void* rope_cos, const void* rope_sin, int64_t rope_rows,
                                void* workspace, int64_t ws_bytes, void* out, void* stream) {
  AQ_CHECK_ARG(q && k_new && v_new && pos && out, "aq_kv4_attention: null pointer");
  if (const int rc = check_cache4("aq_kv4_attention", k_codes, k_params, v_codes, v_params, B, Hkv, D, slots)) return rc;
  AQ_CHECK_ARG((rope_cos == nullptr) == (rope_sin == nullptr), "aq_kv4_attention: rope_cos and rope_sin come together");
  AQ_CHECK_ARG(H > 0 && H % Hkv == 0, "aq_kv4_attention: H (%lld) must be a multiple of Hkv (%lld)", (long long)H,
               (long long)Hkv);
  AQ_CHECK_ARG(pos_stride == 0 || pos_stride == 1, "aq_kv4_attention: pos_stride %lld (0 or 1)", (long long)pos_stride);
  AQ_CHECK_ARG(sinks >= -1 && sinks < slots, "aq_kv4_attention: %lld sinks in %lld slots", (long long)sinks,
               (long long)slots);
  AQ_CHECK_ARG(!rope_cos || rope_rows > 0, "aq_kv4_attention: %lld rows of rope_cos", (long long)rope_rows);
  AQ_CHECK_ARG((uintptr_t)q % 16 == 0 && (uintptr_t)k_new % 16 == 0 && (uintptr_t)v_new % 16 == 0 &&
                   (uintptr_t)out % 16 == 0 && (uintptr_t)rope_cos % 16 == 0 && (uintptr_t)rope_sin % 16 == 0 &&
                   (uintptr_t)pos % 8 == 0,
               "aq_kv4_attention: q, k_new, v_new, out and the rotary tables must be 16-byte aligned");
  const Split4 sp = split4_of(B, Hkv, H / Hkv, D, slots);
  AQ_CHECK_ARG(Hkv * sp.hb <= 65535 && H <= 65535, "aq_kv4_attention: sizes out of range");
  AQ_CHECK_ARG(sp.bytes == 0 || (workspace && (uintptr_t)workspace % 16 == 0 && ws_bytes >= sp.bytes),
               "aq_kv4_attention: workspace of %lld bytes, %lld needed, 16-byte aligned", (long long)ws_bytes,
               (long long)sp.bytes);
  // positions past the table, past a cache without sinks, or past 31 bits are not run
  int64_t max_pos = sinks < 0 ? slots : INT32_MAX;
  if (rope_cos) max_pos = std::min(max_pos, rope_rows);
  const Cache4 c = {(uint8_t*)k_codes, (uint16_t*)k_params, (uint8_t*)v_codes, (uint16_t*)v_params};
  // the kernel's is above 0, so that the largest product has the largest score and a
  // masked one, -inf, stays it: a negative scale's sign and a zero go to the queries
  const float scale2 = (scale == 0.0f ? 1.0f : fabsf(scale) * 1.44269504f) / kCodeUnit;
  if (!(scale > 0.0f)) q_scale = scale == 0.0f ? 0.0f : -q_scale;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)(Hkv * sp.hb), (unsigned)B, (unsigned)sp.ns);
  const size_t lds = (size_t)sp.nw * kHeads * (D + 2) * 4;
#define AQ_KV4_LAUNCH(DD)                                                                                             \
  do {                                                                                                                \
    hipLaunchKernelGGL((kv4_attention_kernel<DD>), grid, dim3(64 * (unsigned)sp.nw), lds, s, (const uint16_t*)q,      \
                       (const uint16_t*)k_new, (const uint16_t*)v_new, c, pos, (int)pos_stride, (int)H, (int)Hkv,     \
                       (int)sp.hb, (int)slots, (int)sinks, scale2, q_scale, (const uint16_t*)rope_cos,                \
                       (const uint16_t*)rope_sin, max_pos, (int)sp.nt, (int)sp.ns, (float*)workspace,                 \
                       (uint16_t*)out);                                                                               \
    if (sp.ns > 1)                                                                                                    \
      hipLaunchKernelGGL((kv4_combine_kernel<DD>), dim3((unsigned)H, (unsigned)B), dim3(256), 0, s, pos,               \
                         (int)pos_stride, (int)H, (int)Hkv, (int)sp.hb, (int)slots, max_pos, (int)sp.nt, (int)sp.ns,  \
                         (const float*)workspace, (uint16_t*)out);                                                    \
  } while (0)
  if (D == 64) AQ_KV4_LAUNCH(64);
  else AQ_KV4_LAUNCH(128);
#undef AQ_KV4_LAUNCH
  AQ_LAUNCH_CHECK("aq_kv4_attention");
  return AQ_OK;
}
