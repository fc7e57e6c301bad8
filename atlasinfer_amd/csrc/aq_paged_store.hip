// aq_paged_store.hip -- new tokens of several sequences into a paged cache,
// rotary positions on the way.
//
// Pair i of a row at position p turns by the angle a = p f_i:
//   x' = m (x cos a - y sin a),  y' = m (y cos a + x sin a)
// (x, y) elements i and i + R/2 of the head (half layout) or 2 i and 2 i + 1
// (interleaved), m the factor that scaled rotary forms put on both.
#include "aq_paged.h"

namespace {

using namespace paged;

constexpr int kThreads = 256;

struct StoreArgs {
  Batch b;
  const uint16_t *q, *k, *v;
  int64_t qs[2], ks[2], vs[2];  // elements between rows, heads
  uint16_t *q_out, *k_cache, *v_cache;
  const float* freq;
  float factor;
  int H, Hkv, D, R, interleaved;
};

// One workgroup a row.  A unit is 16 elements: the two pieces of 8 whose
// elements turn together (half layout: R/2 apart), or two neighbouring pieces.  The sine
// and cosine of each pair are taken once for all heads.
// Bound by memory: 8191 rows of 3 x 32 heads of 64, 201 MB in 42 us (4.8 TB/s; a copy of
// 2 GiB runs at 4.9); 8 rows 4 us, a launch and the chain of loads from the starts over the
// lengths to the page.
template <class T>
__global__ __launch_bounds__(kThreads) void paged_store_kernel(StoreArgs a) {
  __shared__ float s_cos[64], s_sin[64];
  const int t = blockIdx.x, tid = threadIdx.x;
  const int seq = sequence_of(a.b, t);
  if (seq < 0) return;
  const int n = a.b.scalar_start(seq + 1) - a.b.scalar_start(seq), len = scalar_int(a.b.lengths, seq);
  if (n > len || n > a.b.max_new || len > a.b.max_length) return;
  const int pos = len - (a.b.scalar_start(seq + 1) - t);
  int page = scalar_int(a.b.table, (int64_t)seq * a.b.W + (pos >> a.b.shift));
  if ((unsigned)page >= (unsigned)a.b.pages) page = -1;
  if (tid < a.R / 2) {
    // in turns, in 64 bits: an angle of a far position has lost its fraction in 32
    const double u = (double)pos * (double)a.freq[tid] * 0.15915494309189535;
    float sn, cs;
    sincospif(2.0f * (float)(u - rint(u)), &sn, &cs);
    s_cos[tid] = cs * a.factor;
    s_sin[tid] = sn * a.factor;
  }
  __syncthreads();
  const int slot = pos & ((1 << a.b.shift) - 1);
  const int UH = a.D / 16, RU = a.R / 16;  // units of a head, of its turning part
  const int units = (a.H + 2 * a.Hkv) * UH;
  for (int i = tid; i < units; i += kThreads) {
    const int head = i / UH, u = i % UH;
    const uint16_t* src;
    uint16_t* dst;
    if (head < a.H) {
      src = a.q + t * a.qs[0] + head * a.qs[1];
      dst = a.q_out + ((int64_t)t * a.H + head) * a.D;
    } else {
      if (page < 0) continue;
      const bool key = head < a.H + a.Hkv;
      const int j = head - a.H - (key ? 0 : a.Hkv);
      src = key ? a.k + t * a.ks[0] + j * a.ks[1] : a.v + t * a.vs[0] + j * a.vs[1];
      dst = (key ? a.k_cache : a.v_cache) + ((((int64_t)page * a.Hkv + j) << a.b.shift) + slot) * a.D;
    }
    const bool turns = head < a.H + a.Hkv && u < RU;
    const int first = turns && !a.interleaved ? u * 8 : u * 16;
    const int second = turns && !a.interleaved ? first + a.R / 2 : first + 8;
    uint4 x = *reinterpret_cast<const uint4*>(src + first), y = *reinterpret_cast<const uint4*>(src + second);
    if (turns) {
      uint32_t *xw = &x.x, *yw = &y.x;
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          uint32_t& w = e < 4 ? xw[e] : yw[e - 4];
          const float c = s_cos[u * 8 + e], s = s_sin[u * 8 + e];
          const float p = T::to_f32((uint16_t)w), r = T::to_f32((uint16_t)(w >> 16));
          w = T::pack(fmaf(p, c, -(r * s)), fmaf(r, c, p * s));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float o[2], z[2];
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const float c = s_cos[u * 8 + 2 * e + i], s = s_sin[u * 8 + 2 * e + i];
            const float p = T::to_f32((uint16_t)(xw[e] >> (16 * i))), r = T::to_f32((uint16_t)(yw[e] >> (16 * i)));
            o[i] = fmaf(p, c, -(r * s));
            z[i] = fmaf(r, c, p * s);
          }
          xw[e] = T::pack(o[0], o[1]);
          yw[e] = T::pack(z[0], z[1]);
        }
      }
    }
    *reinterpret_cast<uint4*>(dst + first) = x;
    *reinterpret_cast<uint4*>(dst + second) = y;
  }
}

}  // namespace

extern "C" int aq_paged_store(const void* q, const void* k, const void* v, int dtype, int64_t T, int64_t H, int64_t Hkv,
                              int64_t D, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head, int64_t v_row,
                              int64_t v_head, const int32_t* starts, const int32_t* lengths, int64_t S, const int32_t* table, int64_t W,
                              int64_t max_new, int64_t max_length, const float* frequencies, int64_t rotary,
                              int interleaved, float factor, void* q_out, void* k_cache, void* v_cache, int64_t pages,
                              int64_t page_size, void* stream) {
  const char* me = "aq_paged_store";
  AQ_CHECK_ARG(k && v && starts && lengths && table && k_cache && v_cache, "%s: null pointer", me);
  AQ_CHECK_ARG((q == nullptr) == (H == 0) && (q == nullptr) == (q_out == nullptr), "%s: q and q_out come with H", me);
  AQ_CHECK_ARG(dtype == AQ_F16 || dtype == AQ_BF16, "%s: dtype %d (fp16 and bf16 supported)", me, dtype);
  AQ_CHECK_ARG(D == 64 || D == 128, "%s: head dim %lld (64 or 128 supported)", me, (long long)D);
  AQ_CHECK_ARG(T > 0 && T < (1 << 24) && S > 0 && S <= 65535 && H >= 0 && H <= 1024 && Hkv > 0 && Hkv <= 1024,
               "%s: sizes out of range (%lld rows, %lld sequences)", me, (long long)T, (long long)S);
  AQ_CHECK_ARG(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
               "%s: page size %lld (a power of two from 16 to 1024)", me, (long long)page_size);
  AQ_CHECK_ARG(pages > 0 && pages <= INT32_MAX && W > 0 && W <= INT32_MAX / page_size, "%s: %lld pages, %lld of a sequence", me,
               (long long)pages, (long long)W);
  AQ_CHECK_ARG(max_new > 0 && max_length > 0 && max_length <= W * page_size, "%s: at most %lld new, %lld positions of a sequence", me,
               (long long)max_new, (long long)max_length);
  AQ_CHECK_ARG(rotary >= 0 && rotary <= D && rotary % 16 == 0 && (rotary == 0) == (frequencies == nullptr),
               "%s: %lld rotary elements (a multiple of 16 up to D, with their frequencies)", me, (long long)rotary);
  AQ_CHECK_ARG((q_row | q_head | k_row | k_head | v_row | v_head) % 8 == 0, "%s: strides must be multiples of 8", me);
  AQ_CHECK_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 &&
                   ((uintptr_t)starts | (uintptr_t)lengths | (uintptr_t)table | (uintptr_t)frequencies) % 4 == 0,
               "%s: q, k, v, q_out and the caches must be 16-byte aligned", me);
  StoreArgs a;
  a.b = Batch{starts, lengths, table, (int)T, (int)S, (int)W, (int)pages, __builtin_ctz((unsigned)page_size),
              (int)std::min<int64_t>(max_new, T), (int)max_length};
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.qs[0] = q_row;
  a.qs[1] = q_head;
  a.ks[0] = k_row;
  a.ks[1] = k_head;
  a.vs[0] = v_row;
  a.vs[1] = v_head;
  a.q_out = (uint16_t*)q_out;
  a.k_cache = (uint16_t*)k_cache;
  a.v_cache = (uint16_t*)v_cache;
  a.freq = frequencies;
  a.factor = factor;
  a.H = (int)H;
  a.Hkv = (int)Hkv;
  a.D = (int)D;
  a.R = (int)rotary;
  a.interleaved = interleaved;
  if (dtype == AQ_F16)
    hipLaunchKernelGGL((paged_store_kernel<Half>), dim3((unsigned)T), dim3(kThreads), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL((paged_store_kernel<Bf16>), dim3((unsigned)T), dim3(kThreads), 0, (hipStream_t)stream, a);
  AQ_LAUNCH_CHECK(me);
  return AQ_OK;
}
