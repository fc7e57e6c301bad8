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
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kQ = 128;  // queries a workgroup, 32 a wave
constexpr int kK = 64;   // keys a tile

struct WindowArgs {
  const uint16_t *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];
  const int* starts;
  uint16_t* out;
  int H, G, M, N, window, sinks;
  float scale2;
};

__device__ __forceinline__ bool not_finite8(uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; i++) bad = bad || (w[i] & 0x7C00u) == 0x7C00u || (w[i] & 0x7C000000u) == 0x7C000000u;
  return bad;
}

// Scores are taken transposed (keys as rows of mfma 32 x 32 x 16), so that a
// lane has 16 scores of one query and its numerators are the second product's
// operand as they are; the values lie transposed in LDS, the keys of each 16 in
// the order in which a lane has them.
template <int D>
__global__ __launch_bounds__(256) void window_attention_kernel(WindowArgs a) {
  constexpr int KS = D + 8;       // LDS row of keys, in fp16
  constexpr int VS = kK + 8;      // LDS row of one element of the values
  constexpr int NC = D / 8;       // 16-byte pieces of a row
  constexpr int KP = kK * NC / 256;  // pieces of keys a thread
  __shared__ uint16_t kl[kK * KS];
  __shared__ uint16_t vl[D * VS];
  __shared__ int bad;
  const int t = threadIdx.x, ln = t & 63, c = ln & 31, h = ln >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int head = blockIdx.y, b = blockIdx.z, q0 = blockIdx.x * kQ;
  const int off = a.N - a.M;
  const int start = a.starts ? max(0, a.starts[b]) : 0;
  const uint16_t* kb = a.k + b * a.ks[0] + (head / a.G) * a.ks[1];
  const uint16_t* vb = a.v + b * a.vs[0] + (head / a.G) * a.vs[1];

  // positions of the workgroup's queries, and the tiles with keys they see
  const int lo = off + q0, hi = off + min(q0 + kQ, a.M) - 1;
  int64_t near64 = (int64_t)lo - a.window + 1;
  const int near = (int)max(near64, (int64_t)start);
  const int b0 = near / kK, b1 = hi >= start ? hi / kK : b0 - 1;
  const int64_t sink_end = min((int64_t)start + a.sinks, (int64_t)hi + 1);  // sinks are start .. sink_end - 1
  const int a0 = start / kK;
  const int na = sink_end > start ? max(0, min((int)((sink_end - 1) / kK) + 1, b0) - a0) : 0;
  const int tiles = na + max(0, b1 - b0 + 1);
  auto tile_at = [&](int i) { return i < na ? a0 + i : b0 + i - na; };

  const int qi = q0 + wave * 32 + c, qpos = off + qi;  // this lane's query
  half8v qv[D / 16];
  {
    const uint16_t* qp = a.q + b * a.qs[0] + head * a.qs[1] + (int64_t)min(qi, a.M - 1) * a.qs[2] + 8 * h;
#pragma unroll
    for (int s = 0; s < D / 16; s++) qv[s] = *reinterpret_cast<const half8v*>(qp + 16 * s);
  }
  float16v o[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; e++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[e][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  const int wlo = off + q0 + wave * 32, whi = min(wlo + 31, a.N - 1);  // the wave's positions

  uint4 kr[KP], vr[4];
  const uint4 zero = make_uint4(0, 0, 0, 0);
  // values: a thread has four keys of one 16-byte piece (D = 64: half of them)
  const int vq = t & 15, vd = t >> 4;
  auto load = [&](int tile) {
    const int k0 = tile * kK;
#pragma unroll
    for (int n = 0; n < KP; n++) {
      const int i = n * 256 + t, r = k0 + i / NC;
      kr[n] = r < a.N ? *reinterpret_cast<const uint4*>(kb + (int64_t)r * a.ks[2] + i % NC * 8) : zero;
    }
#pragma unroll
    for (int n = 0; n < 4; n++) {
      const int r = k0 + 4 * vq + n;  // keys before start or past the end count as zeros whatever is there
      vr[n] = vd < NC && r < a.N && r >= start ? *reinterpret_cast<const uint4*>(vb + (int64_t)r * a.vs[2] + vd * 8) : zero;
    }
  };
  if (t == 0) bad = 0;
  if (tiles > 0) load(tile_at(0));
  for (int i = 0; i < tiles; i++) {
    const int k0 = tile_at(i) * kK;
    __syncthreads();  // the tile before has been read
    if (t == 0) bad = 0;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < KP; n++) {
      const int x = n * 256 + t;
      *reinterpret_cast<uint4*>(kl + x / NC * KS + x % NC * 8) = kr[n];
    }
    if (vd < NC) {
      // key 16 s + 8 x + 4 y + z at place 16 s + 8 y + 4 x + z
      const int place = (vq >> 2) * 16 + (vq & 1) * 8 + ((vq >> 1) & 1) * 4;
      const uint16_t* r0 = reinterpret_cast<const uint16_t*>(vr);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        uint2 w;
        w.x = (uint32_t)r0[e] | (uint32_t)r0[8 + e] << 16;
        w.y = (uint32_t)r0[16 + e] | (uint32_t)r0[24 + e] << 16;
        *reinterpret_cast<uint2*>(vl + (vd * 8 + e) * VS + place) = w;
      }
      if (not_finite8(vr[0]) || not_finite8(vr[1]) || not_finite8(vr[2]) || not_finite8(vr[3])) bad = 1;
    }
    if (i + 1 < tiles) load(tile_at(i + 1));
    __syncthreads();
    // whether this wave's queries see none, all or some of the tile
    const bool none = k0 > whi || (k0 + kK - 1 <= wlo - a.window && k0 >= sink_end) || k0 + kK <= start;
    if (none) continue;
    const bool all = k0 + kK - 1 <= wlo && k0 > whi - a.window && k0 >= start;
    float x[32];
#pragma unroll
    for (int s = 0; s < 2; s++) {
      float16v acc;
#pragma unroll
      for (int e = 0; e < 16; e++) acc[e] = 0.0f;
#pragma unroll
      for (int e = 0; e < D / 16; e++) {
        const half8v kf = *reinterpret_cast<const half8v*>(kl + (s * 32 + c) * KS + e * 16 + 8 * h);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qv[e], acc, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 16; e++) x[16 * s + e] = acc[e] * a.scale2;
    }
    if (!all) {
#pragma unroll
      for (int e = 0; e < 32; e++) {
        const int key = k0 + 32 * (e >> 4) + 8 * ((e >> 2) & 3) + 4 * h + (e & 3);
        const bool sees = key <= qpos && key >= start && (qpos - key < a.window || key - start < a.sinks);
        x[e] = sees ? x[e] : -INFINITY;
      }
    }
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < 32; e++) mx = fmaxf(mx, x[e]);
    mx = fmaxf(m, xlane_level_max_f32<6>(mx));
    if (__ballot(mx != m)) {
      const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
      l *= f;
#pragma unroll
      for (int e = 0; e < D / 32; e++) o[e] *= f;
      m = mx;
    }
    const float base = m == -INFINITY ? 0.0f : m;
    half8v p[4];
#pragma unroll
    for (int e = 0; e < 32; e++) {
      const float w = __builtin_amdgcn_exp2f(x[e] - base);
      l += w;
      p[e >> 3][e & 7] = rn_h(w);
    }
    if (!all && bad) {
      // an infinity or NaN among the values of a tile that the mask cuts: the
      // terms one by one, leaving out those of weight zero
      for (int key = 0; key < kK; key++) {
        const int s = key >> 4, y = (key >> 2) & 1, e8 = ((key >> 3) & 1) * 4 + (key & 3);
        f16 w = (f16)0.0f;
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (n == s && e == e8) w = p[n][e];
        const float wf = __shfl((float)w, c + 32 * y, 64);
        const uint16_t* vp = vl + s * 16 + y * 8 + e8;
#pragma unroll
        for (int e = 0; e < D / 32; e++)
#pragma unroll
          for (int n = 0; n < 16; n++) {
            const int d = 32 * e + 8 * (n >> 2) + 4 * h + (n & 3);
            if (wf != 0.0f) o[e][n] = fmaf(wf, (float)bits_to_h(vp[d * VS]), o[e][n]);
          }
      }
      continue;
    }
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
      for (int e = 0; e < D / 32; e++) {
        const half8v vf = *reinterpret_cast<const half8v*>(vl + (e * 32 + c) * VS + s * 16 + 8 * h);
        o[e] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, p[s], o[e], 0, 0, 0);
      }
  }
  l = xlane_level_sum_f32<6>(l);
  if (qi < a.M) {
    const float f = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // a query that sees nothing answers zero
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
  a.scale2 = scale * 1.44269504f;
  const dim3 grid((unsigned)aq::ceil_div(M, kQ), (unsigned)H, (unsigned)B);
  if (D == 64)
    hipLaunchKernelGGL((window_attention_kernel<64>), grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((window_attention_kernel<128>), grid, dim3(256), 0, (hipStream_t)stream, a);
  AQ_LAUNCH_CHECK("aq_window_attention");
  return AQ_OK;
}
