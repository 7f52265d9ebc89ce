// What the two attention kernels over the 4-bit K/V cache share: arguments, the conversion of codes and scales, the
// look-up of a key's cache row and the epilogue of a row.
#pragma once
#include <cuda_fp16.h>

#include <climits>

#include "msl_common.cuh"
#include "msl_host.h"

namespace msl {

struct Kv4Args {
  const __nv_bfloat16* q;       // [tokens][hq][D], row pitch ld_q
  int64_t ld_q;
  const uint8_t *k, *ks, *v, *vs;
  const int* page_table;        // [batch][max_pages]
  int max_pages;
  const int* seq_lens;
  const int* cu_seqlens_q;
  const float* k_scale;
  const float* v_scale;
  float softmax_scale;
  int batch, max_q_len, tokens, hq, hkv, page_size, window;
  int64_t cache_rows;
  __nv_bfloat16* out;
  int64_t ld_out;
  const __nv_bfloat16* gate;
  int64_t ld_gate;
  float* part;                  // partial results (workspace)
  int workers;                  // few rows: CTAs that share the key tiles,
  int heads;                    //   KV heads a CTA takes at once,
  int tile_shift;               //   log2 of a tile's keys
  int kv_splits;                // many rows: slices of a query block's keys
  int alternate;                //   up to 128 rows a request: CTAs share the key tiles, their sub-tiles in turn
  int page_shift;               // log2 of the page size, -1: not a power of two
  int* status;
};

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ float kv_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The four bytes of a word, each a pair of e2m1 codes -> f16x2 (low nibble in the low half).
__device__ __forceinline__ void e2m1x8(uint32_t w, __half2 (&h)[4]) {
  uint32_t a, b, c, d;
  asm("{.reg .b8 x, y, z, u;\n\tmov.b32 {x, y, z, u}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, x;\n\tcvt.rn.f16x2.e2m1x2 %1, y;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, z;\n\tcvt.rn.f16x2.e2m1x2 %3, u;}"
      : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(w));
  h[0] = bits_h2(a); h[1] = bits_h2(b); h[2] = bits_h2(c); h[3] = bits_h2(d);
}
// Two e4m3 scales -> f16x2.  The NaN codes (never written by the store) read as 448: a NaN would reach rows that
// do not see the key, as 0 * NaN in P V.
__device__ __forceinline__ __half2 scales_h2(uint32_t two) {
  uint32_t h;
  asm("{.reg .b16 x;\n\tcvt.u16.u32 x, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, x;}" : "=r"(h) : "r"(two));
  return __hmin2(bits_h2(h), __half2half2(__ushort_as_half(0x5F00)));   // 448
}
// A query row's score scale: the softmax's, in log2 units, without the power of two `up` that the row was multiplied
// by.  It stays above zero: a hidden score is -inf, and -inf * 0 would make a row NaN.  (Only a row of nothing but tiny
// values, whose scores weigh all keys alike, has a factor this small.)
__device__ __forceinline__ float kv4_row_scale(float scale_log2, float up) {
  float s = scale_log2 / up;
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(s) : "f"(1.17549435e-38f));   // (a NaN stays one)
  return s;
}
// A request as the schedule sees it: q rows [begin, begin + len), `seq` cached tokens.
struct Kv4Req {
  int begin, len, seq;
  bool over;                    // has rows past max_q_len, which nothing writes
};
__device__ __forceinline__ Kv4Req kv4_request(const Kv4Args& p, int b) {
  Kv4Req r;
  r.begin = max(0, min(p.cu_seqlens_q[b], p.tokens));
  const int end = max(r.begin, min(p.cu_seqlens_q[b + 1], p.tokens));
  r.len = min(end - r.begin, p.max_q_len);
  r.over = end - r.begin > p.max_q_len;
  r.seq = p.seq_lens[b];
  return r;
}
// Key tiles [first, last) that a request's rows can see, 2^tile_shift keys a tile.
struct Kv4Span {
  int first, last;
};
__device__ __forceinline__ Kv4Span kv4_span(const Kv4Args& p, const Kv4Req& r, int tile_shift) {
  // keys past the table's row have no page: they are not walked (the kernel reports them)
  const int hi = static_cast<int>(min(static_cast<int64_t>(r.seq) + r.len,
                                      static_cast<int64_t>(p.max_pages) * p.page_size));
  const int lo = p.window ? max(0, r.seq - p.window + 1) : 0;
  Kv4Span s;
  s.first = lo >> tile_shift;
  s.last = max(s.first + 1, (hi + (1 << tile_shift) - 1) >> tile_shift);   // with nothing to see: zeros are written
  return s;
}
template <int W>
__device__ __forceinline__ int64_t block_sum_i64(int64_t v, int64_t* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  int64_t s = 0;
  for (int w = 0; w < W; ++w) s += scratch[w];
  __syncthreads();
  return s;
}

// Programmatic launch: the next kernel's blocks may start; wait until the kernel before has ended and its writes show.
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A key's page table entry, loaded a step before its row is needed.
struct Kv4Page {
  int page, off;                // page INT_MIN: the key is hidden from every row
};
__device__ __forceinline__ Kv4Page kv4_page(const Kv4Args& p, const int* table, int key, int lo, int hi) {
  Kv4Page x{INT_MIN, 0};
  if (key >= lo && key < hi) {
    const int idx = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
    x.off = key - idx * p.page_size;
    x.page = idx < p.max_pages ? table[idx] : -1;
  }
  return x;
}
__device__ __forceinline__ int kv4_row_of(const Kv4Args& p, const Kv4Page& x) {
  const int64_t row = static_cast<int64_t>(x.page) * p.page_size + x.off;
  if (x.page >= 0 && row < p.cache_rows) return static_cast<int>(row);
  if (x.page != INT_MIN) report_error(p.status, MSL_ERR_CAPACITY);
  return -1;
}

// Rows of a finished block: O / l, v_scale, optional per-head RMS norm * sigmoid(gate), bf16.  One warp per row,
// lane holds channels [D/32 lane, ...).
template <int D>
__device__ __forceinline__ void kv4_write_row(const Kv4Args& p, float (&o)[D / 32], float l, int64_t token, int head,
                                              int lane) {
  constexpr int PER = D / 32;
  const float c = l > 0.f ? *p.v_scale / l : 0.f;          // a row that sees nothing is zero
  // a NaN sum (a NaN query) must stay visible
  const float scale = l != l ? l : c;
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) { o[i] *= scale; ss += o[i] * o[i]; }
  if (p.gate != nullptr) {
    const float r = 1.0f / sqrtf(warp_sum(ss) / D + 1e-5f);
    const __nv_bfloat16* grow = p.gate + token * p.ld_gate + head * D + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] *= __fdividef(r, 1.0f + __expf(-__bfloat162float(grow[i])));
  }
  __nv_bfloat16* orow = p.out + token * p.ld_out + head * D + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; i += 2) *reinterpret_cast<uint32_t*>(orow + i) = pack_bf16x2(o[i], o[i + 1]);
}

// Many query rows per KV head (prefill, chunks): csrc/attention_kv4_tc.cu.
int launch_kv4_tc(const Kv4Args& a, int head_dim, cudaStream_t st);
int64_t kv4_tc_workspace(int slots, int tokens, int hq, int head_dim);
int64_t kv4_tc_shared_workspace(int rows, int tokens, int hq, int head_dim);

}  // namespace msl
