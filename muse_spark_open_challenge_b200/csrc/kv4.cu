// The 4-bit K/V cache: page plan, store (norm + RoPE + quantise) and row read-back.
//
// Cache format (the grid and the nibble order of the reference's NVFP4 weights,
// muse_prefill_layer/nvfp4.py:24-47): channels [16 i, 16 i + 16) of a (row, head) share one E4M3 scale s,
// an element is an E2M1 code c, element 2 i in the low nibble of byte i, and stands for c * s * scale with
// one fp32 scale for the keys and one for the values.  Codes u8 [rows][hkv][D / 2], scales e4m3
// [rows][hkv][D / 16]: 4.5 bits an element against the 8 of the FP8 cache.
#include <cuda_fp16.h>

#include "msl_common.cuh"
#include "msl_host.h"

namespace msl {

// ============================================================================ page plan
// Exclusive prefix sums over the requests of new tokens (cu) and of pages to take (pg), in every block: the
// batch is small next to the tokens, and a block that has both sums in shared memory finds the request of a
// token or of a page by bisection, so one launch does everything.  Bound by latency: one round of loads for
// the lengths, one for the free list, one store.
constexpr int kPlanThreads = 256;
constexpr int kPlanMaxBatch = 16384;     // 2 sums x 4 bytes: 128 KB of shared memory

struct PlanArgs {
  const int* new_lens;          // [batch]
  const int* seq_lens;          // [batch] cached tokens
  int* page_table;              // [batch][max_pages]
  const int* free_pages;        // [n_free]
  const int* free_head;         // index of the first free page
  int* free_head_out;
  int* cu_seqlens_q;            // [batch + 1]
  int64_t* positions;           // [tokens]
  int64_t* cache_loc;           // [tokens]
  int batch, max_pages, n_free, page_size, tokens;
  int* status;
};

__device__ __forceinline__ int pages_of(int64_t len, int page_size, int max_pages) {
  return static_cast<int>(min((len + page_size - 1) / page_size, static_cast<int64_t>(max_pages)));
}

// Largest b with sums[b] <= x (sums ascending, sums[0] = 0, x < sums[n]): the request that x falls into.
__device__ __forceinline__ int owner_of(const int* sums, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(PlanArgs p) {
  extern __shared__ int plan_smem[];
  int* cu = plan_smem;                    // [batch + 1]
  int* pg = plan_smem + p.batch + 1;      // [batch + 1]
  __shared__ long long part[2][kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
  bool bad = false;
  long long sum_t = 0, sum_p = 0;
  auto lengths = [&](int b, int& n, int64_t& seq) {
    n = p.new_lens[b];
    seq = p.seq_lens[b];
    if (n < 0 || seq < 0) { bad = true; n = max(n, 0); seq = seq < 0 ? 0 : seq; }
  };
  for (int b = b0; b < b1; ++b) {
    int n; int64_t seq;
    lengths(b, n, seq);
    sum_t += n;
    sum_p += pages_of(seq + n, p.page_size, p.max_pages) - pages_of(seq, p.page_size, p.max_pages);
    bad |= (seq + n + p.page_size - 1) / p.page_size > p.max_pages;
  }
  // inclusive sums over the threads
  long long inc_t = sum_t, inc_p = sum_p;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, inc_t, o), c = __shfl_up_sync(0xffffffffu, inc_p, o);
    if (lane >= o) { inc_t += a; inc_p += c; }
  }
  if (lane == 31) { part[0][warp] = inc_t; part[1][warp] = inc_p; }
  __syncthreads();
  for (int w = 0; w < warp; ++w) { inc_t += part[0][w]; inc_p += part[1][w]; }
  long long at_t = inc_t - sum_t, at_p = inc_p - sum_p;
  const long long int_max = 0x7fffffff;
  for (int b = b0; b < b1; ++b) {
    cu[b] = static_cast<int>(min(at_t, static_cast<long long>(p.tokens)));
    pg[b] = static_cast<int>(min(at_p, int_max));
    int n; int64_t seq;
    lengths(b, n, seq);
    at_t += n;
    at_p += pages_of(seq + n, p.page_size, p.max_pages) - pages_of(seq, p.page_size, p.max_pages);
  }
  if (tid == kPlanThreads - 1) {          // the last thread's inclusive sums are the totals
    cu[p.batch] = static_cast<int>(min(inc_t, static_cast<long long>(p.tokens)));
    pg[p.batch] = static_cast<int>(min(inc_p, int_max));
    bad |= inc_t > p.tokens;
  }
  __syncthreads();
  const int total = cu[p.batch], taken = pg[p.batch];
  const int head = *p.free_head;
  const int usable = head < 0 ? 0 : max(0, p.n_free - head);
  bad |= taken > usable;
  auto page_at = [&](int j) { return j < usable ? p.free_pages[head + j] : -1; };
  const int step = gridDim.x * kPlanThreads, first = blockIdx.x * kPlanThreads + tid;
  for (int b = first; b <= p.batch; b += step) p.cu_seqlens_q[b] = cu[b];
  if (first == 0) *p.free_head_out = head + min(taken, usable);
  for (int64_t j = first; j < taken; j += step) {
    const int b = owner_of(pg, p.batch, static_cast<int>(j));
    const int have = pages_of(max(p.seq_lens[b], 0), p.page_size, p.max_pages);
    p.page_table[static_cast<int64_t>(b) * p.max_pages + have + (j - pg[b])] = page_at(static_cast<int>(j));
  }
  for (int64_t t = first; t < p.tokens; t += step) {
    int64_t pos = 0, loc = -1;
    if (t < total) {
      const int b = owner_of(cu, p.batch, static_cast<int>(t));
      const int seq = max(p.seq_lens[b], 0);
      pos = static_cast<int64_t>(seq) + (t - cu[b]);
      const int64_t idx = pos / p.page_size;
      const int have = pages_of(seq, p.page_size, p.max_pages);
      int page = -1;
      // a page the request already holds is read from its row (this call writes only entries from `have` on)
      if (idx < have) page = p.page_table[static_cast<int64_t>(b) * p.max_pages + idx];
      else if (idx < p.max_pages) page = page_at(pg[b] + static_cast<int>(idx - have));
      if (page >= 0) loc = static_cast<int64_t>(page) * p.page_size + pos % p.page_size;
      else bad = true;
    }
    p.positions[t] = pos;
    p.cache_loc[t] = loc;
  }
  if (bad) report_error(p.status, MSL_ERR_CAPACITY);
}

// ============================================================================ store
// Lanes own 8 consecutive channels of a head, D / 8 lanes a head; two neighbouring lanes share a block of 16.
// Queries are rounded to bf16 once, so fp32 serves them.  Keys and values end on a coarse grid, where an
// error of one fp32 ulp next to a border moves a value by a whole step: their norm, rotation and borders are
// held in 64 bits (this GPU runs them at half the fp32 rate), and codes come from comparisons with
// border * (s * scale), a product of 24 + 4 + 3 bits that is exact in 64, so that ties are seen as ties.
constexpr int kStoreThreads = 256;

// bf16 bits -> double, exact for finite values; infinities and NaN become finite, +-2^128 and above: the
// format has no code for them, and they saturate like any value beyond its range.
__device__ __forceinline__ double bf16_bits_to_f64(uint32_t b) {
  // the exponent lands in the low bits of a double's: off by the difference of the biases, subnormals too
  const double d = __hiloint2double(static_cast<int>(((b & 0x8000u) << 16) | ((b & 0x7fffu) << 13)), 0);
  return d * __hiloint2double((1023 + 896) << 20, 0);
}

__device__ __forceinline__ double shfl_xor_f64(double v, int o) {
  return __hiloint2double(__shfl_xor_sync(0xffffffffu, __double2hiint(v), o),
                          __shfl_xor_sync(0xffffffffu, __double2loint(v), o));
}

// Nearest E4M3 of x in [0, 448], ties to even: rounding to odd in fp32 first keeps the second rounding right.
__device__ __forceinline__ uint32_t e4m3_of_f64(double x) {
  float f = __double2float_rz(x);
  if (static_cast<double>(f) != x) f = __uint_as_float(__float_as_uint(f) | 1u);
  return __nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(b), __NV_E4M3)));
}

struct StoreArgs {
  const __nv_bfloat16* qkv;
  int64_t ld;
  const int64_t* positions;
  const int64_t* cache_loc;
  const float* inv_freq;        // [D / 2] or NULL
  const float* k_scale;
  const float* v_scale;
  __nv_bfloat16* q;             // [tokens][hq][D]
  uint8_t *k, *ks, *v, *vs;
  int tokens, hq, hkv;
  int64_t cache_rows;
  int* status;
};

template <int D>
__global__ void __launch_bounds__(kStoreThreads)
qk_rope_store_kv4_kernel(StoreArgs p) {
  constexpr int LPH = D / 8;
  __shared__ double2 rot[D / 2];          // (cos, sin) of position * inv_freq[j]
  const int t = blockIdx.x;
  const int lanes = (p.hq + 2 * p.hkv) * LPH;
  const int idx = blockIdx.y * kStoreThreads + threadIdx.x;
  const bool live = idx < lanes;
  const int h = idx / LPH, sub = idx % LPH;
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (live) raw = *reinterpret_cast<const uint4*>(p.qkv + t * p.ld + h * D + sub * 8);
  if (p.inv_freq != nullptr) {
    for (int j = threadIdx.x; j < D / 2; j += kStoreThreads) {
      // the angle's whole turns are taken off in 64 bits: 2 pi as a sum of two doubles
      const double a = static_cast<double>(p.positions[t]) * static_cast<double>(p.inv_freq[j]);
      const double n = rint(a * 0.15915494309189535);
      const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, a));
      double sn, cs;
      sincos(r, &sn, &cs);
      rot[j] = make_double2(cs, sn);
    }
    __syncthreads();
  }
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  const bool is_q = h < p.hq, is_v = h >= p.hq + p.hkv;
  double z[8];
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    z[i] = bf16_bits_to_f64((w[i / 2] >> (16 * (i & 1))) & 0xffffu);
    ss += z[i] * z[i];
  }
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) ss += shfl_xor_f64(ss, o);
  if (!is_v) {
    const double r = 1.0 / sqrt(ss / D + 1e-5);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      double e = z[i] * r, o = z[i + 1] * r;
      if (p.inv_freq != nullptr) {
        const double2 cs = rot[(sub * 8 + i) / 2];
        const double e2 = e * cs.x - o * cs.y;
        o = e * cs.y + o * cs.x;
        e = e2;
      }
      z[i] = e;
      z[i + 1] = o;
    }
  }
  double amax = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmax(amax, fabs(z[i]));
  amax = fmax(amax, shfl_xor_f64(amax, 1));
  if (!live) return;
  if (is_q) {
    uint4 o;
    o.x = pack_bf16x2(static_cast<float>(z[0]), static_cast<float>(z[1]));
    o.y = pack_bf16x2(static_cast<float>(z[2]), static_cast<float>(z[3]));
    o.z = pack_bf16x2(static_cast<float>(z[4]), static_cast<float>(z[5]));
    o.w = pack_bf16x2(static_cast<float>(z[6]), static_cast<float>(z[7]));
    *reinterpret_cast<uint4*>(p.q + (static_cast<int64_t>(t) * p.hq + h) * D + sub * 8) = o;
    return;
  }
  const int64_t row = p.cache_loc[t];
  if (row < 0) return;                                      // a padding token
  if (row >= p.cache_rows) { report_error(p.status, MSL_ERR_CAPACITY); return; }
  const double scale = is_v ? *p.v_scale : *p.k_scale;
  const uint32_t s8 = e4m3_of_f64(fmin(amax / (6.0 * scale), 448.0));
  const double c = static_cast<double>(e4m3_to_f32(s8)) * scale;
  uint32_t packed = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double m = fabs(z[i]);
    uint32_t code = (m > 0.25 * c) + (m >= 0.75 * c) + (m > 1.25 * c) + (m >= 1.75 * c) + (m > 2.5 * c) +
                    (m >= 3.5 * c) + (m > 5.0 * c);
    if (z[i] < 0.0) code |= 8u;
    packed |= code << (4 * i);
  }
  if (s8 == 0) packed = 0;                                  // a block below half the smallest scale
  const int head = is_v ? h - p.hq - p.hkv : h - p.hq;
  uint8_t* codes = is_v ? p.v : p.k;
  uint8_t* scales = is_v ? p.vs : p.ks;
  const int64_t at = row * p.hkv + head;
  *reinterpret_cast<uint32_t*>(codes + at * (D / 2) + sub * 4) = packed;
  if ((sub & 1) == 0) scales[at * (D / 16) + sub / 2] = static_cast<uint8_t>(s8);
}

// ============================================================================ read-back
// out[i] = the values of cache row rows[i] (zeros for a negative index), one lane per 8 codes.
template <typename OUT>
__global__ void __launch_bounds__(256)
kv4_rows_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const float* __restrict__ scale,
                const int64_t* __restrict__ rows, int64_t n, int width, int64_t cache_rows, OUT* __restrict__ out,
                int* status) {
  const int per_row = width / 8;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (idx >= n * per_row) return;
  const int64_t i = idx / per_row;
  const int c = static_cast<int>(idx % per_row);
  const int64_t row = rows[i];
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (row >= cache_rows) report_error(status, MSL_ERR_CAPACITY);
  if (row >= 0 && row < cache_rows) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + row * (width / 2) + c * 4);
    const float s = e4m3_to_f32(scales[row * (width / 16) + c / 2]);
    const float t = *scale;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t code = (w >> (4 * k)) & 15u, m = code & 7u;
      // code * s is exact (2 + 4 bits), so the fp32 product with the tensor's scale rounds once
      const float mag = m < 4 ? 0.5f * m : (m < 6 ? static_cast<float>(m - 2) : 2.0f * m - 8.0f);
      v[k] = ((code & 8u) ? -mag : mag) * s * t;
    }
  }
  if constexpr (sizeof(OUT) == 2) {
    *reinterpret_cast<uint4*>(out + idx * 8) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                          pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
    float4* dst = reinterpret_cast<float4*>(out + idx * 8);
    dst[0] = make_float4(v[0], v[1], v[2], v[3]);
    dst[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

static bool misaligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

}  // namespace msl

using namespace msl;

extern "C" int msl_page_plan(const int* new_lens, const int* seq_lens, int* page_table, int max_pages,
                             const int* free_pages, int n_free, const int* free_head, int* free_head_out, int batch,
                             int page_size, int tokens, int* cu_seqlens_q, int64_t* positions, int64_t* cache_loc,
                             int* status, void* stream) {
  if (batch <= 0 || page_size <= 0 || max_pages <= 0 || n_free < 0 || tokens < 0) return MSL_ERR_ARG;
  if (!new_lens || !seq_lens || !page_table || !free_head || !free_head_out || !cu_seqlens_q ||
      (n_free > 0 && !free_pages) || (tokens > 0 && (!positions || !cache_loc)))
    return MSL_ERR_ARG;
  if (free_head == free_head_out) return MSL_ERR_ARG;       // every block reads the old head
  if (batch > kPlanMaxBatch) return MSL_ERR_UNSUPPORTED;
  static SmemConfig config;
  if (int rc = config.ensure(page_plan_kernel, 2 * (kPlanMaxBatch + 1) * 4)) return rc;
  const PlanArgs a{new_lens, seq_lens, page_table, free_pages, free_head, free_head_out, cu_seqlens_q, positions,
                   cache_loc, batch, max_pages, n_free, page_size, tokens, status};
  // a block per 1024 tokens (four a thread): the sums are repeated in every block, the bisections are not
  const int64_t want = (static_cast<int64_t>(std::max(tokens, batch)) + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
  const int grid = static_cast<int>(std::min<int64_t>(want, 4 * sm_count()));
  page_plan_kernel<<<grid, kPlanThreads, 2 * (batch + 1) * 4, static_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? MSL_OK : MSL_ERR_CUDA;
}

extern "C" int msl_qk_rope_store_kv4(const void* qkv, int64_t ld, const int64_t* positions, const int64_t* cache_loc,
                                     const float* inv_freq, const float* k_scale, const float* v_scale, void* q,
                                     void* k_cache, void* k_sf, void* v_cache, void* v_sf, int tokens, int hq, int hkv,
                                     int head_dim, int64_t cache_rows, int* status, void* stream) {
  if (tokens < 0 || hq <= 0 || hkv <= 0 || cache_rows <= 0) return MSL_ERR_ARG;
  if (head_dim != 64 && head_dim != 128) return MSL_ERR_UNSUPPORTED;
  if (tokens == 0) return MSL_OK;
  if (!qkv || !positions || !cache_loc || !k_scale || !v_scale || !q || !k_cache || !k_sf || !v_cache || !v_sf)
    return MSL_ERR_ARG;
  if (ld < static_cast<int64_t>(hq + 2 * hkv) * head_dim) return MSL_ERR_ARG;
  if (misaligned(qkv, 16) || misaligned(q, 16) || (ld & 7) || misaligned(k_cache, 16) || misaligned(v_cache, 16))
    return MSL_ERR_ALIGN;
  const StoreArgs a{static_cast<const __nv_bfloat16*>(qkv), ld, positions, cache_loc, inv_freq, k_scale, v_scale,
                    static_cast<__nv_bfloat16*>(q), static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(k_sf),
                    static_cast<uint8_t*>(v_cache), static_cast<uint8_t*>(v_sf), tokens, hq, hkv, cache_rows, status};
  const int lanes = (hq + 2 * hkv) * (head_dim / 8);
  const dim3 grid(tokens, (lanes + kStoreThreads - 1) / kStoreThreads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) qk_rope_store_kv4_kernel<128><<<grid, kStoreThreads, 0, st>>>(a);
  else qk_rope_store_kv4_kernel<64><<<grid, kStoreThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? MSL_OK : MSL_ERR_CUDA;
}

extern "C" int msl_kv4_rows(const void* codes, const void* scales, const float* scale, const int64_t* rows, int64_t n,
                            int width, int64_t cache_rows, int out_mode, void* out, int* status, void* stream) {
  if (n < 0 || width <= 0 || cache_rows <= 0 || (out_mode != MSL_OUT_BF16 && out_mode != MSL_OUT_F32)) return MSL_ERR_ARG;
  if (n == 0) return MSL_OK;
  if (!codes || !scales || !scale || !rows || !out) return MSL_ERR_ARG;
  if ((width & 15) || misaligned(codes, 16) || misaligned(out, 16)) return MSL_ERR_ALIGN;
  const int64_t blocks = (n * (width / 8) + 255) / 256;
  if (blocks > 0x7fffffff) return MSL_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto* c = static_cast<const uint8_t*>(codes);
  const auto* s = static_cast<const uint8_t*>(scales);
  if (out_mode == MSL_OUT_BF16)
    kv4_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(c, s, scale, rows, n, width, cache_rows,
                                                                  static_cast<__nv_bfloat16*>(out), status);
  else
    kv4_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(c, s, scale, rows, n, width, cache_rows,
                                                                  static_cast<float*>(out), status);
  return cudaGetLastError() == cudaSuccess ? MSL_OK : MSL_ERR_CUDA;
}
