// aq_window.hip -- attention of a prompt through a sliding window with sinks.
//
// out = softmax(scale q k^T + mask) v in one pass over the keys a block of
// queries can see: with the running maximum m of a query's scores and the sums
// l = sum e^(s - m), o = sum e^(s - m) v so far, a tile of keys with maximum m'
// scales l and o by e^(m - max(m, m')) and adds its own terms.
#include "aq_common.h"

namespace {

typedef _Float16 half4v __attribute__((ext_vector_type(4)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_s4;

constexpr int kQ = 128;  // queries a workgroup, 32 a wave
constexpr int kK = 64;   // keys a tile
constexpr float kGrow = 8.0f;

struct WindowArgs {
  const uint16_t *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];
  const int* starts;
  uint16_t* out;
  int H, G, M, N, window, sinks, blocks, items, per;
  float c;  // |scale| log2(e), above 0: a masked score, -inf, times it stays that
  uint32_t keep, flip;  // for the queries' bits: none for a scale of 0, the sign of a negative one
};

typedef __attribute__((address_space(3))) uint8_t lds_u8;

// 16 bytes a lane from a buffer's byte `off` straight to LDS, at dst + 16 lane;
// zeros past the buffer's end.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t r, uint8_t* dst, int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (void*)dst, 16, off, 0, 0, 0);
}

// Four rows of 16 fp16 numbers in LDS, 8 bytes given by each of 16 lanes in
// order: lane i gets column i.
__device__ __forceinline__ half4v read_turned(const uint8_t* p) {
  return __builtin_bit_cast(half4v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds_u8*)p));
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The larger of m and the magnitudes of eight fp16 numbers, as pairs of bits:
// from 0x7C00 on one is not finite.
__device__ __forceinline__ u16x2 magnitudes8(u16x2 m, uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
  return m;
}

// A tile's rows lie in LDS one after the other, 16-byte pieces permuted within
// each so that the reads below meet every bank equally: piece c of key r at place
// c ^ (r & 7) of a key row, pairs of pieces c / 2 at (c / 2) ^ (r & 3) of a value row.
template <int D>
__device__ __forceinline__ int k_place(int r, int c) { return r * (D * 2) + (c ^ (r & 7)) * 16; }
template <int D>
__device__ __forceinline__ int v_place(int r, int c) { return r * (D * 2) + ((((c >> 1) ^ (r & 3)) << 1) | (c & 1)) * 16; }

// One workgroup: 128 queries of a head, 32 a wave; tiles of 64 keys and values
// go straight from memory to LDS (direct loads, one tile ahead for D = 128, three
// for 64, whose tiles take half as long as a load; one barrier a tile).
//   scores   transposed, s^T = k q^T (mfma 32 x 32 x 16): a lane has 32 scores of
//            one query, another lane the other 32, so maxima and sums need one
//            exchange
//   softmax  p = e^(s - m) with m the maximum when it last moved: it moves only
//            when a score passes it by 2^8 (p stays below 2^8, exact in range for
//            fp16 and f32 alike), which spares scaling the sums nearly always
//   values   o^T = v^T p^T: the numerators, rounded to fp16, are the operand as
//            they are; the values come out of their rows transposed
//            (ds_read_tr16_b64: four keys of 16 elements for 16 lanes)
//   sums     of the rounded numerators (v_dot2), so that rounding them does not
//            shift the mean
// Bound by the matrix unit and the softmax's exponentials together: 32 heads of 128
// over 8 key/value heads, 8192 positions, a window of 4096 with 4 sinks: 483 us, 854
// TFLOP/s of the two products (the library's fp16 product of 8192^3: 1144); 32 heads
// of 64, 1017 positions, a window of 256: 15 us, one round of workgroups of up to
// seven tiles each, one wave a SIMD.
template <int D>
__global__ __launch_bounds__(256, 2) void window_attention_kernel(WindowArgs a) {
  constexpr int NC = D / 8;                    // 16-byte pieces of a row
  constexpr int TB = kK * D * 2;               // bytes of a tile of keys, or of values
  constexpr int PN = TB / 1024 / 4;            // 1 KiB loads of each a wave
  constexpr int NS = D == 64 ? 4 : 2;          // stages: 64 KiB
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NS * 2 * TB];  // keys and values of each stage
  __shared__ int bad[NS];
  const int t = threadIdx.x, ln = t & 63, c = ln & 31, h = ln >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  // runs of neighbouring items to an XCD (they share keys and values in its L2)
  const int item = (int)(blockIdx.x & 7) * a.per + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= a.per || item >= a.items) return;
  // cleared before any wave may set one, which is before the loop's first barrier
  if (t < NS) bad[t] = 0;
  __syncthreads();
  // heads of a group next to each other, late blocks (more keys) first
  const int g = item % a.G, qb = a.blocks - 1 - item / a.G % a.blocks, u = item / a.G / a.blocks;
  const int hkv = a.H / a.G, b = u / hkv, j = u % hkv, head = j * a.G + g, q0 = qb * kQ;
  const int off = a.N - a.M;
  const int start = a.starts ? max(0, a.starts[b]) : 0;
  const uint16_t* kb = a.k + b * a.ks[0] + j * a.ks[1];
  const uint16_t* vb = a.v + b * a.vs[0] + j * a.vs[1];

  // positions of the workgroup's queries, and the tiles with keys they see
  const int lo = off + q0, hi = off + min(q0 + kQ, a.M) - 1;
  const int near = max(lo - a.window + 1, start);
  const int b0 = near / kK, b1 = hi >= start ? hi / kK : b0 - 1;
  const int sink_end = (int)min((int64_t)start + a.sinks, (int64_t)hi + 1);  // sinks are start .. sink_end - 1
  const int a0 = start / kK;
  const int na = sink_end > start ? max(0, min((sink_end - 1) / kK + 1, b0) - a0) : 0;
  const int tiles = na + max(0, b1 - b0 + 1);
  auto tile_at = [&](int i) { return i < na ? a0 + i : b0 + i - na; };

  const int qi = q0 + wave * 32 + c, qpos = off + qi;  // this lane's query
  half8v qv[D / 16];
  {
    const uint16_t* qp = a.q + b * a.qs[0] + head * a.qs[1] + (int64_t)min(qi, a.M - 1) * a.qs[2] + 8 * h;
#pragma unroll
    for (int s = 0; s < D / 16; s++) {
      uint4 x = *reinterpret_cast<const uint4*>(qp + 16 * s);
#pragma unroll
      for (int i = 0; i < 4; i++) (&x.x)[i] = ((&x.x)[i] & a.keep) ^ a.flip;
      qv[s] = __builtin_bit_cast(half8v, x);
    }
  }
  float16v o[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; e++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[e][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  const int wlo = off + q0 + wave * 32, whi = min(wlo + 31, a.N - 1);  // the wave's positions
  const float grow = kGrow / a.c;

  // this lane's part of the loads: piece n of the wave covers rows of the tile
  int row[PN], ko[PN], vo[PN];
#pragma unroll
  for (int n = 0; n < PN; n++) {
    row[n] = (wave * PN + n) * (64 / NC) + ln / NC;
    const int pc = ln % NC;
    ko[n] = row[n] * (int)a.ks[2] * 2 + (pc ^ (row[n] & 7)) * 16;
    vo[n] = row[n] * (int)a.vs[2] * 2 + ((((pc >> 1) ^ (row[n] & 3)) << 1) | (pc & 1)) * 16;
  }
  auto load = [&](int i) {
    const int k0 = tile_at(i) * kK;
    uint8_t* st = lds + (i & (NS - 1)) * (2 * TB) + wave * PN * 1024;
    // rows past the last read as zeros, values before the start too, whatever is there
    const int rows = min(a.N - k0, kK);
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(kb + (int64_t)k0 * a.ks[2]), (short)0, ((rows - 1) * (int)a.ks[2] + D) * 2, 0x00020000);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(vb + (int64_t)k0 * a.vs[2]), (short)0, ((rows - 1) * (int)a.vs[2] + D) * 2, 0x00020000);
#pragma unroll
    for (int n = 0; n < PN; n++) load_to_lds(kr, st + n * 1024, ko[n]);
    const int first = start - k0;
    if (first > 0) {
#pragma unroll
      for (int n = 0; n < PN; n++)
        load_to_lds(vr, st + TB + n * 1024, row[n] < first ? (int)0x80000000 : vo[n]);
    } else {
#pragma unroll
      for (int n = 0; n < PN; n++) load_to_lds(vr, st + TB + n * 1024, vo[n]);
    }
  };
  // LDS offsets of this lane's fragments: keys of row c, pieces 2 e + h (e & 3;
  // e + 4 lies 128 bytes on); values of keys 4 h + r, 16 elements of 32 e (e & 1)
  int kf[4], vf[2];
#pragma unroll
  for (int e = 0; e < 4; e++) kf[e] = k_place<D>(c, 2 * e + h);
  const int r4 = (ln >> 2) & 3;
#pragma unroll
  for (int e = 0; e < 2; e++) vf[e] = v_place<D>(4 * h + r4, 2 * (2 * e + ((ln >> 4) & 1)) + ((ln & 3) >> 1)) + (ln & 1) * 8;

  for (int i = 0; i < min(NS - 1, tiles); i++) load(i);
  for (int i = 0; i < tiles; i++) {
    const int k0 = tile_at(i) * kK;
    const uint8_t* st = lds + (i & (NS - 1)) * (2 * TB);
    // this wave's part of the tile is there; the NS - 2 tiles after it may be on their way
    if (i + NS - 2 < tiles)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * 2 * PN) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (!(k0 + kK - 1 <= lo && k0 > hi - a.window && k0 >= start)) {
      // a tile that the mask cuts for some query: whether its values are finite
      u16x2 m = 0;
#pragma unroll
      for (int n = 0; n < PN; n++) m = magnitudes8(m, *reinterpret_cast<const uint4*>(st + TB + (wave * PN + n) * 1024 + ln * 16));
      if (__ballot(max(m.x, m.y) >= 0x7C00) && ln == 0) bad[i & (NS - 1)] = i + 1;
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // every wave's part; the tile before is done with
    if (i + NS - 1 < tiles) load(i + NS - 1);
    // whether this wave's queries see none, all or some of the tile
    if (k0 > whi || (k0 + kK - 1 <= wlo - a.window && k0 >= sink_end) || k0 + kK <= start) continue;
    const bool all = k0 + kK - 1 <= wlo && k0 > whi - a.window && k0 >= start;
    float16v x[2];
#pragma unroll
    for (int s = 0; s < 2; s++) {
#pragma unroll
      for (int e = 0; e < 16; e++) x[s][e] = 0.0f;
#pragma unroll
      for (int e = 0; e < D / 16; e++) {
        const half8v f = *reinterpret_cast<const half8v*>(st + kf[e & 3] + (e >> 2) * 128 + s * 32 * (D * 2));
        x[s] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, qv[e], x[s], 0, 0, 0);
      }
    }
    if (!all) {
      // a key is seen when it lies in one of two ranges: near the query, or among
      // the sinks, both up to the query (each a subtraction, an unsigned comparison
      // and a selection: conditions joined as masks would go through the scalar unit
      // and take five times as long)
      const int last = qpos - k0 - 4 * h, from = max(last - a.window + 1, start - k0 - 4 * h);
      const int sink0 = start - k0 - 4 * h;
      const uint32_t near_n = (uint32_t)max(last - from + 1, 0);
      const uint32_t sink_n = (uint32_t)max(min(a.sinks, last - sink0 + 1), 0);
      if (k0 < sink_end) {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const int key = 32 * s + 8 * (e >> 2) + (e & 3);
            const float y = (uint32_t)(key - sink0) < sink_n ? x[s][e] : -INFINITY;
            x[s][e] = (uint32_t)(key - from) < near_n ? x[s][e] : y;
          }
      } else {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const int key = 32 * s + 8 * (e >> 2) + (e & 3);
            x[s][e] = (uint32_t)(key - from) < near_n ? x[s][e] : -INFINITY;
          }
      }
    }
    float mx = fmaxf(x[0][0], x[1][0]);
#pragma unroll
    for (int e = 1; e < 16; e++) mx = fmaxf(fmaxf(mx, x[0][e]), x[1][e]);  // v_max3
    mx = xlane_level_max_f32<6>(mx);
    if (__ballot(mx > m + grow || (m == -INFINITY && mx > m))) {
      const float n = fmaxf(m, mx), f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - n) * a.c);
      l *= f;
#pragma unroll
      for (int e = 0; e < D / 32; e++) o[e] *= f;
      m = n;
    }
    const float base = m == -INFINITY ? 0.0f : -m * a.c;
    uint32_t p[16];  // the numerators in pairs: p[4 n .. 4 n + 3] are the operand of 16 keys
    const half2v one = {(f16)1.0f, (f16)1.0f};
#pragma unroll
    for (int e = 0; e < 16; e++) {
      const int y = 2 * e & 15;
      const float2v w = {__builtin_amdgcn_exp2f(fmaf(x[e >> 3][y], a.c, base)),
                         __builtin_amdgcn_exp2f(fmaf(x[e >> 3][y + 1], a.c, base))};
      const half2v r = __builtin_convertvector(w, half2v);  // one conversion for both, to nearest
      l = __builtin_amdgcn_fdot2(r, one, l, false);
      p[e] = __builtin_bit_cast(uint32_t, r);
    }
    if (!all && bad[i & (NS - 1)] == i + 1) {
      // an infinity or NaN among the values of a tile that the mask cuts: the
      // terms one by one, leaving out those of keys that the query does not see (a
      // weight may also have rounded to zero: times infinity that is NaN, as in the
      // products below)
      // (the sums pass an empty asm here, so that what the compiler does for this
      // loop's sake, copying them, it does here and not on the common path)
#pragma unroll
      for (int e = 0; e < D / 32; e++) asm volatile("" : "+v"(o[e]));
      int from = max(qpos - a.window + 1, start) - k0, sink0 = start - k0;
      uint32_t near_n = (uint32_t)max(qpos - k0 - from + 1, 0), sink_n = (uint32_t)max(min(a.sinks, qpos - start + 1), 0);
      asm volatile("" : "+v"(from), "+v"(sink0), "+v"(near_n), "+v"(sink_n));
#pragma unroll 1
      for (int key = 0; key < kK; key++) {
        const int y = (key >> 2) & 1, n = (key >> 4) * 4 + ((key >> 3) & 1) * 2 + ((key >> 1) & 1);  // its half wave, pair
        uint32_t w = p[0];
#pragma unroll
        for (int e = 1; e < 16; e++) w = e == n ? p[e] : w;
        const bool seen = (uint32_t)(key - from) < near_n || (uint32_t)(key - sink0) < sink_n;
        const float wf = __shfl((float)bits_to_h((uint16_t)(key & 1 ? w >> 16 : w)), c + 32 * y, 64);
#pragma unroll
        for (int e = 0; e < D / 32; e++)
#pragma unroll
          for (int z = 0; z < 16; z++) {
            const int d = 32 * e + 8 * (z >> 2) + 4 * h + (z & 3);
            const uint16_t vd = *reinterpret_cast<const uint16_t*>(st + TB + v_place<D>(key, d >> 3) + (d & 7) * 2);
            if (seen) o[e][z] = fmaf(wf, (float)bits_to_h(vd), o[e][z]);
          }
      }
      continue;
    }
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
      for (int e = 0; e < D / 32; e++) {
        // keys 16 s + 4 h + 0 .. 3, then 8 on: the order in which a lane has the numerators
        const uint8_t* f = st + TB + vf[e & 1] + (e >> 1) * 128 + s * 16 * (D * 2);
        const half8v w = __builtin_shufflevector(read_turned(f), read_turned(f + 8 * (D * 2)), 0, 1, 2, 3, 4, 5, 6, 7);
        o[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w, __builtin_bit_cast(half8v, u32x4{p[4 * s], p[4 * s + 1], p[4 * s + 2], p[4 * s + 3]}), o[e], 0, 0, 0);
      }
  }
  l = xlane_level_sum_f32<6>(l);
  if (qi < a.M) {
    // a query that sees nothing answers zero; one that sees a key, its own among them, and
    // only scores of -inf (l is 0) NaN, as the softmax of these
    const float f = qpos >= start ? (l == 0.0f ? NAN : 1.0f / l) : 0.0f;
    uint16_t* op = a.out + (((int64_t)b * a.M + qi) * a.H + head) * D + 4 * h;
#pragma unroll
    for (int e = 0; e < D / 32; e++)
#pragma unroll
      for (int n = 0; n < 4; n++) {
        uint32_t w[2];
#pragma unroll
        for (int y = 0; y < 2; y++)
          w[y] = (uint32_t)h_to_bits(rn_h(o[e][4 * n + 2 * y] * f)) | (uint32_t)h_to_bits(rn_h(o[e][4 * n + 2 * y + 1] * f)) << 16;
        *reinterpret_cast<uint2*>(op + 32 * e + 8 * n) = make_uint2(w[0], w[1]);
      }
  }
}

}  // namespace

extern "C" int aq_window_attention(const void* q, const void* k, const void* v, int64_t B, int64_t H, int64_t Hkv,
                                   int64_t M, int64_t N, int64_t D, const int64_t* q_strides, const int64_t* k_strides,
                                   const int64_t* v_strides, int64_t window, int64_t sinks, float scale,
                                   const int32_t* starts, void* out, void* stream) {
  AQ_CHECK_ARG(q && k && v && q_strides && k_strides && v_strides && out, "aq_window_attention: null pointer");
  AQ_CHECK_ARG(D == 64 || D == 128, "aq_window_attention: head dim %lld (64 or 128 supported)", (long long)D);
  AQ_CHECK_ARG(B > 0 && B <= 65535 && Hkv > 0 && H > 0 && H <= 65535 && H % Hkv == 0,
               "aq_window_attention: %lld sequences, H (%lld) must be a multiple of Hkv (%lld)", (long long)B,
               (long long)H, (long long)Hkv);
  AQ_CHECK_ARG(M > 0 && M <= N && N < (1 << 24), "aq_window_attention: the last %lld of %lld positions", (long long)M,
               (long long)N);
  AQ_CHECK_ARG(window >= 1 && sinks >= 0, "aq_window_attention: window %lld, %lld sinks", (long long)window,
               (long long)sinks);
  for (int i = 0; i < 3; i++)
    AQ_CHECK_ARG(q_strides[i] % 8 == 0 && k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0,
                 "aq_window_attention: strides must be multiples of 8");
  AQ_CHECK_ARG(k_strides[2] >= 0 && v_strides[2] >= 0 && k_strides[2] <= (1 << 23) && v_strides[2] <= (1 << 23),
               "aq_window_attention: positions of k and v more than 2^23 elements apart");
  AQ_CHECK_ARG((uintptr_t)q % 16 == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)out % 16 == 0 &&
                   (uintptr_t)starts % 4 == 0,
               "aq_window_attention: q, k, v and out must be 16-byte aligned");
  WindowArgs a;
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  for (int i = 0; i < 3; i++) {
    a.qs[i] = q_strides[i];
    a.ks[i] = k_strides[i];
    a.vs[i] = v_strides[i];
  }
  a.starts = starts;
  a.out = (uint16_t*)out;
  a.H = (int)H;
  a.G = (int)(H / Hkv);
  a.M = (int)M;
  a.N = (int)N;
  a.window = (int)std::min<int64_t>(window, N);
  a.sinks = (int)std::min<int64_t>(sinks, N);
  a.c = scale == 0.0f ? 1.0f : fabsf(scale) * 1.44269504f;
  a.keep = scale == 0.0f ? 0u : 0xFFFFFFFFu;
  a.flip = scale < 0.0f ? 0x80008000u : 0u;
  a.blocks = (int)aq::ceil_div(M, kQ);
  const int64_t items = B * H * a.blocks;
  // (a grid has fewer than 2^32 threads)
  AQ_CHECK_ARG(items <= (1 << 24) - 8, "aq_window_attention: %lld blocks of queries", (long long)items);
  a.items = (int)items;
  a.per = (int)aq::ceil_div(items, 8);
  const dim3 grid((unsigned)(8 * a.per));
  if (D == 64)
    hipLaunchKernelGGL((window_attention_kernel<64>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((window_attention_kernel<128>), grid, dim3(256), 0, (hipStream_t)stream, a);
  AQ_LAUNCH_CHECK("aq_window_attention");
  return AQ_OK;
}
