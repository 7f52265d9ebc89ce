// The 4-bit K/V cache: page plan, store (norm + RoPE + quantise) and row read-back.
//
// Cache format (the grid and the nibble order of the reference's NVFP4 weights,
// muse_prefill_layer/nvfp4.py:24-47): channels [16 i, 16 i + 16) of a (row, head) share one E4M3 scale s,
// an element is an E2M1 code c, element 2 i in the low nibble of byte i, and stands for c * s * scale with
// one fp32 scale for the keys and one for the values.  Codes u8 [rows][hkv][D / 2], scales e4m3
// [rows][hkv][D / 16]: 4.5 bits an element against the 8 of the FP8 cache.
#include "kv4_common.cuh"

namespace msl {

// ============================================================================ page plan
// Exclusive prefix sums over the requests of new tokens (cu) and of pages to take (pg), in every block: the
// batch is small next to the tokens, and a block that has both sums in shared memory finds the request of a
// token or of a page by bisection, so one launch does everything.  Bound by latency: one round of loads for
// the lengths, one for the free list, one store.  64 requests 6 us, 256 with 131072 tokens 10, 1000 with pages of one
// token 14.
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
// A lane owns a block of 16 consecutive channels, D / 16 lanes a head: 32 bytes in, 8 bytes of codes and a scale out.
// Queries are rounded to bf16 once, so fp32 serves them.  Keys and values end on a coarse grid, where an error of one
// fp32 ulp next to a border moves a value by a whole step.  So fp32 only proposes: scale and codes are formed from the value
// nudged up and down by more than the fp32 error (below), and where the two disagree 64 bits decide: a value against
// border * (s * scale), 3 + 4 + 24 bits and exact, so that ties are seen as ties; a key (its norm and rotation are not
// exact in fp32) by doing its heads again in 64 bits, which one warp in a hundred has to.
// What it is bound by is issue slots, then HBM: 16384 tokens of 32 + 8 + 8 heads x 128 (354 MB) took 190 us with
// everything in 64 bits, 116 with the queries in fp32, 100 with the keys' proposal in fp32, 85 with a block of 16
// channels a lane (4.2 TB/s of the measured 6.55).  Counted: 0.75 instructions issued per cycle and scheduler with two
// more warps ready for each one, DRAM 48 % busy, ALU 46 %.  64 registers for four blocks an SM cost 24 to 32 bytes of spill
// stores a thread (up to 60 in key_codes_f64).
// A key channel that is exactly zero, or a block of keys whose scale is below 2^-6 (a row of zeros, so a padding token),
// takes the 64-bit way too, and the whole warp with it.
constexpr int kStoreThreads = 256, kStoreWarps = kStoreThreads / 32;
constexpr int kStoreTok = 4;               // most tokens of a block

// bf16 bits -> double, exact for finite values; infinities and NaN become finite, +-2^128 and above: the
// format has no code for them, and they saturate like any value beyond its range.
__device__ __forceinline__ double bf16_bits_to_f64(uint32_t b) {
  // the exponent lands in the low bits of a double's: off by the difference of the biases, subnormals too
  const double d = __hiloint2double(static_cast<int>(((b & 0x8000u) << 16) | ((b & 0x7fffu) << 13)), 0);
  return d * __hiloint2double((1023 + 896) << 20, 0);
}

__device__ __forceinline__ double shfl_xor_f64(uint32_t mask, double v, int o) {
  return __hiloint2double(__shfl_xor_sync(mask, __double2hiint(v), o), __shfl_xor_sync(mask, __double2loint(v), o));
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

// Nearest E2M1 codes (saturating) of eight values, element i in nibble i.
__device__ __forceinline__ uint32_t e2m1_pack(const float* v) {
  uint32_t w;
  asm("{.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};}"
      : "=r"(w)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return w;
}
// Codes of u[i] * f; + 0 keeps a zero's code 0 whatever its sign.
__device__ __forceinline__ uint2 e2m1_of_16(const float (&u)[16], float f) {
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = fmaf(u[i], f, 0.0f);
  return make_uint2(e2m1_pack(v), e2m1_pack(v + 8));
}
// ... with the magnitude moved up or down by `nudge`.  A value within it of zero changes its sign when it is moved down,
// and a zero does in one of the two (-0 when it is moved up): the codes then differ and 64 bits decide.
template <bool UP>
__device__ __forceinline__ uint2 e2m1_of_16(const float (&u)[16], float f, float nudge) {
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = UP ? fmaf(u[i], f, copysignf(nudge, u[i])) : fmaf(u[i], f, -copysignf(nudge, u[i]));
  return make_uint2(e2m1_pack(v), e2m1_pack(v + 8));
}
// 32 bytes at once where the rows allow it (`wide`: base and pitch multiples of 32), else as two halves.
__device__ __forceinline__ void load_32(uint32_t (&w)[8], const void* src, bool wide) {
  if (wide) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(src));
  } else {
    const uint4 a = reinterpret_cast<const uint4*>(src)[0], b = reinterpret_cast<const uint4*>(src)[1];
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  }
}
__device__ __forceinline__ void store_32(void* dst, const uint32_t (&w)[8], bool wide) {
  if (wide) {
    st_global_v8(dst, w);
  } else {
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// The angle is formed in 64 bits (csrc/elementwise.cu forms it in fp32): in fp32 it would be off by up to 2^-24 of itself,
// 0.03 rad at position 500000, a hundred times and more the error of the rest (below).
// (cos, sin) of an angle of any size: quarter turns are taken off in 64 bits (pi / 2 as a sum of two doubles), what is
// left has at most pi / 4, where a Taylor series serves: to r^14, good to about 1e-14, or in fp32 to r^10.
__device__ __forceinline__ double2 cos_sin_f64(double a) {
  const double n = rint(a * 0.63661977236758134);
  const double r = fma(-n, 6.123233995736766e-17, fma(-n, 1.5707963267948966, a));
  const double q = r * r;
  double s = 1.0 / 6227020800.0, c = -1.0 / 87178291200.0;
  s = fma(s, q, -1.0 / 39916800.0); c = fma(c, q, 1.0 / 479001600.0);
  s = fma(s, q, 1.0 / 362880.0); c = fma(c, q, -1.0 / 3628800.0);
  s = fma(s, q, -1.0 / 5040.0); c = fma(c, q, 1.0 / 40320.0);
  s = fma(s, q, 1.0 / 120.0); c = fma(c, q, -1.0 / 720.0);
  s = fma(s, q, -1.0 / 6.0); c = fma(c, q, 1.0 / 24.0);
  c = fma(c, q, -0.5);
  s = fma(s * q, r, r);
  c = fma(c, q, 1.0);
  // n mod 4 from the low bits of n + 1.5 * 2^52
  const int k = __double2loint(n + 6755399441055744.0) & 3;
  const double x = (k & 1) ? s : c, y = (k & 1) ? c : s;
  return make_double2((k == 1 || k == 2) ? -x : x, (k & 2) ? -y : y);
}

__device__ __forceinline__ float2 cos_sin_f32(double a) {
  const double n = rint(a * 0.63661977236758134);
  const float r = static_cast<float>(fma(-n, 6.123233995736766e-17, fma(-n, 1.5707963267948966, a)));
  const float q = r * r;
  float s = 2.7557319e-6f, c = -2.7557319e-7f;             // 1 / 9!, -1 / 10!
  s = fmaf(s, q, -1.9841270e-4f); c = fmaf(c, q, 2.4801587e-5f);
  s = fmaf(s, q, 8.3333333e-3f); c = fmaf(c, q, -1.3888889e-3f);
  s = fmaf(s, q, -1.6666667e-1f); c = fmaf(c, q, 4.1666667e-2f);
  c = fmaf(c, q, -0.5f);
  s = fmaf(s * q, r, r);
  c = fmaf(c, q, 1.0f);
  const int k = __double2loint(n + 6755399441055744.0) & 3;
  const float x = (k & 1) ? s : c, y = (k & 1) ? c : s;
  return make_float2((k == 1 || k == 2) ? -x : x, (k & 2) ? -y : y);
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
  int per_block;                // tokens of a block
  bool wide_in, wide_out;       // rows of qkv / q start on 32 bytes
  int64_t cache_rows;
  int* status;
};

// The E4M3 scale of a block from its largest magnitude in fp32, relative error below 2^-18; `sure` is false near a
// midpoint of E4M3 and among its subnormals.
__device__ __forceinline__ uint32_t block_scale(float amax, float inv_scale, bool& sure) {
  const float want = fminf(amax * (inv_scale * (1.0f / 6.0f)), 448.0f);
  const int from_mid = static_cast<int>(__float_as_uint(want) & 0xfffffu) - 0x80000;
  sure = want >= 0.015625f && (from_mid < -64 || from_mid > 64);
  return __nv_cvt_float_to_fp8(want, __NV_SATFINITE, __NV_E4M3);
}

// A key head's 16 channels of this lane in 64 bits, start to end; the whole warp takes part.
template <int D, bool ROPE>
__device__ __noinline__ uint2 key_codes_f64(const __nv_bfloat16* src, bool in, double position, const float* inv_freq,
                                            double scale, uint32_t& s8) {
  constexpr int LPH = D / 16;
  const int sub = threadIdx.x % LPH;
  double z[16], ss = 0.0, top = 0.0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    z[i] = in ? bf16_bits_to_f64(reinterpret_cast<const uint16_t*>(src)[i]) : 0.0;
    ss = fma(z[i], z[i], ss);
  }
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) ss += shfl_xor_f64(0xffffffffu, ss, o);
  const double r = 1.0 / sqrt(ss / D + 1e-5);
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    double e = z[i] * r, o = z[i + 1] * r;
    if (ROPE) {
      const double2 cs = cos_sin_f64(position * static_cast<double>(inv_freq[sub * 8 + i / 2]));
      const double e2 = e * cs.x - o * cs.y;
      o = e * cs.y + o * cs.x;
      e = e2;
    }
    z[i] = e;
    z[i + 1] = o;
    top = fmax(top, fmax(fabs(e), fabs(o)));
  }
  s8 = e4m3_of_f64(fmin(top / (6.0 * scale), 448.0));
  const double c = static_cast<double>(e4m3_to_f32(s8)) * scale;
  uint32_t packed[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const double m = fabs(z[i]);
    uint32_t code = (m > 0.25 * c) + (m >= 0.75 * c) + (m > 1.25 * c) + (m >= 1.75 * c) + (m > 2.5 * c) +
                    (m >= 3.5 * c) + (m > 5.0 * c);
    if (z[i] < 0.0) code |= 8u;
    packed[i / 8] |= code << (4 * (i % 8));
  }
  // a block below half the smallest scale has zero codes
  return s8 == 0 ? make_uint2(0, 0) : make_uint2(packed[0], packed[1]);
}

// A block takes p.per_block tokens with all their heads: their rotations first (a thread an angle), then the lanes of
// their queries, keys and values in units of 32, dealt out to the warps in turn; a unit's heads have one role.
template <int D, bool ROPE>
__global__ void __launch_bounds__(kStoreThreads, 4)
qk_rope_store_kv4_kernel(StoreArgs p) {
  constexpr int LPH = D / 16;
  // (cos, sin) of position * inv_freq[8 lane + i] at [i][lane]: a warp's reads are contiguous
  __shared__ float2 rot[kStoreTok][8][LPH];
  const int t0 = blockIdx.x * p.per_block, nt = min(p.per_block, p.tokens - t0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = threadIdx.x % LPH;
  const __nv_bfloat16* src = p.qkv + t0 * p.ld;
  const int q_lanes = p.hq * LPH, kv_lanes = p.hkv * LPH;
  const int q_units = (q_lanes + 31) / 32, kv_units = (kv_lanes + 31) / 32, units = q_units + 2 * kv_units;
  // unit u: this lane's place in its role, the role's first lane among the token's lanes, its number of lanes
  const auto role_of = [&](int u, int& at, int& first, int& count) {
    const int kv = u - q_units;
    first = kv < 0 ? 0 : kv < kv_units ? q_lanes : q_lanes + kv_lanes;
    count = kv < 0 ? q_lanes : kv_lanes;
    at = 32 * (kv < 0 ? u : kv < kv_units ? kv : kv - kv_units) + lane;
    return kv;
  };
  uint32_t next[8];
  const auto fetch = [&](int tt, int u) {                   // lanes past the role's end go through the motions
    int at, first, count;
    role_of(u, at, first, count);
#pragma unroll
    for (int i = 0; i < 8; ++i) next[i] = 0;
    if (at < count) load_32(next, src + tt * p.ld + (first + at) * 16, p.wide_in);
  };
  int u = warp, tt = 0;
  const auto settle = [&]() {                               // on to the token that unit u falls into
    while (u >= units) { u -= units; ++tt; }
  };
  settle();
  if (tt < nt) fetch(tt, u);
  if (ROPE) {
    for (int x = threadIdx.x; x < nt * (D / 2); x += kStoreThreads) {
      const int t = x / (D / 2), j = x % (D / 2);
      rot[t][j % 8][j / 8] = cos_sin_f32(static_cast<double>(p.positions[t0 + t]) * static_cast<double>(p.inv_freq[j]));
    }
    __syncthreads();
  }
  const float k_scale = *p.k_scale, v_scale = *p.v_scale, inv_k = 1.0f / k_scale, inv_v = 1.0f / v_scale;
  while (tt < nt) {
    const int now = tt, unit = u;
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = next[i];
    u += kStoreWarps;
    settle();
    if (tt < nt) fetch(tt, u);
    int at, first, count;
    const int kv = role_of(unit, at, first, count);
    const bool in = at < count;
    float v[16];
    if (kv < kv_units) {
      // ---- a query or a key: norm and rotation
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        v[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        ss = fmaf(v[i], v[i], ss);
      }
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss * (1.0f / D) + 1e-5f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float e = v[2 * i] * r, o = v[2 * i + 1] * r;
        if (ROPE) {
          const float2 cs = rot[now][i][sub];
          const float e2 = e * cs.x - o * cs.y;
          o = e * cs.y + o * cs.x;
          e = e2;
        }
        v[2 * i] = e;
        v[2 * i + 1] = o;
      }
      if (kv < 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
        if (in) store_32(p.q + static_cast<int64_t>(t0 + now) * p.hq * D + at * 16, w, p.wide_out);
        continue;
      }
      // fp32 errors, in half steps of 2^-24: 14 in r (16 products and 3 sums of shuffles, halved by the root; the root
      // 4), 1 in e, 3 in cosine and sine, 2 in the rotation, so 20 (|e| + |o|) <= 40 largest magnitudes of the block:
      // 2^-18.6 of it.  That magnitude is at most 6.4 of a code's units, so 1.6e-5 of one; the nudge is 3e-5.  (Where the
      // scale saturates at 448 the block reaches further: 64 bits.)
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(v[i]));
      bool sure;
      uint32_t s8 = block_scale(amax, inv_k, sure);
      const float inv = __fdividef(inv_k, e4m3_to_f32(s8));
      uint2 packed = e2m1_of_16<true>(v, inv, 3.0517578125e-5f);
      const uint2 below = e2m1_of_16<false>(v, inv, 3.0517578125e-5f);
      sure &= packed.x == below.x && packed.y == below.y && ss < 1e38f && amax * inv < 6.5f;
      if (__any_sync(0xffffffffu, in && !sure))
        packed = key_codes_f64<D, ROPE>(src + now * p.ld + (first + at) * 16, in,
                                        static_cast<double>(p.positions[t0 + now]), p.inv_freq, k_scale, s8);
      const int64_t row = p.cache_loc[t0 + now];
      if (row >= p.cache_rows) report_error(p.status, MSL_ERR_CAPACITY);
      if (in && row >= 0 && row < p.cache_rows) {           // negative: a padding token
        const int64_t to = row * kv_lanes + at;             // 8 bytes of codes and a scale a lane
        *reinterpret_cast<uint2*>(p.k + to * 8) = packed;
        p.ks[to] = static_cast<uint8_t>(s8);
      }
      continue;
    }
    // ---- a value: exact in fp32; infinities and NaN, which have no code, count as the largest finite magnitude
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t mag = __vminu2(w[i] & 0x7fff7fffu, 0x7f7f7f7fu);
      top = __vmaxu2(top, mag);
      w[i] = mag | (w[i] & 0x80008000u);
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    const float amax = bf16_bits_to_f32(max(top & 0xffffu, top >> 16));
    bool sure;
    uint32_t s8 = block_scale(amax, inv_v, sure);
    if (!sure) s8 = e4m3_of_f64(fmin(static_cast<double>(amax) / (6.0 * static_cast<double>(v_scale)), 448.0));
    const float s = e4m3_to_f32(s8), inv = __fdividef(inv_v, s);   // good to 2^-21 or better, the nudge is 2^-20
    uint2 packed = e2m1_of_16(v, inv * (1.0f + 9.5367431640625e-7f));
    const uint2 below = e2m1_of_16(v, inv * (1.0f - 9.5367431640625e-7f));
    if (s8 == 0) {                                          // a block below half the smallest scale
      packed = make_uint2(0, 0);
    } else if (packed.x != below.x || packed.y != below.y) {
      const double c = static_cast<double>(s) * static_cast<double>(v_scale);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t& mine = half ? packed.y : packed.x;
        const uint32_t unsure = mine ^ (half ? below.y : below.x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if ((unsure >> (4 * i)) & 15u) {
            // `mine` has the upper code; 4 x the border below it: 1 3 5 7 10 14 20
            const uint32_t up = (mine >> (4 * i)) & 7u;
            const uint32_t border4 = static_cast<uint32_t>(0x140e0a0705030100ull >> (8 * up)) & 255u;
            const double d = fma(-0.25 * border4, c, static_cast<double>(fabsf(v[8 * half + i])));
            if (d < 0.0 || (d == 0.0 && (up & 1u))) mine -= 1u << (4 * i);   // a tie goes to the even code
          }
        }
      }
    }
    const int64_t row = p.cache_loc[t0 + now];
    if (row >= p.cache_rows) report_error(p.status, MSL_ERR_CAPACITY);
    if (in && row >= 0 && row < p.cache_rows) {
      const int64_t to = row * kv_lanes + at;
      *reinterpret_cast<uint2*>(p.v + to * 8) = packed;
      p.vs[to] = static_cast<uint8_t>(s8);
    }
  }
}

// ============================================================================ read-back
// out[i] = the values of cache row rows[i] (zeros for a negative index), one lane per block of 16: 8 bytes of codes and
// a scale in, 32 or 64 bytes out.
constexpr int kRowsThreads = 256;
template <typename OUT>
__global__ void __launch_bounds__(kRowsThreads)
kv4_rows_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const float* __restrict__ scale,
                const int64_t* __restrict__ rows, int64_t n, int blocks, int rows_per_cta, int64_t cache_rows,
                OUT* __restrict__ out, int* status) {
  const float t = *scale;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * rows_per_cta;
  for (int x = threadIdx.x; x < rows_per_cta * blocks; x += kRowsThreads) {
    const int64_t i = first + x / blocks;
    if (i >= n) return;
    const int64_t row = rows[i];
    uint2 w = make_uint2(0, 0);
    float s = 0.f;
    if (row >= cache_rows) {
      report_error(status, MSL_ERR_CAPACITY);
    } else if (row >= 0) {
      const int64_t at = row * blocks + x % blocks;
      w = *reinterpret_cast<const uint2*>(codes + at * 8);
      s = fminf(e4m3_to_f32(scales[at]), 448.f);            // the NaN codes too, as the attention reads them
    }
    // code * s is exact (2 + 4 bits), so the fp32 product with the tensor's scale rounds once
    float v[16];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __half2 h[4];
      e2m1x8(k ? w.y : w.x, h);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(h[j]);
        v[8 * k + 2 * j] = f.x * s * t;
        v[8 * k + 2 * j + 1] = f.y * s * t;
      }
    }
    OUT* dst = out + (first * blocks + x) * 16;
    if constexpr (sizeof(OUT) == 2) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        reinterpret_cast<uint4*>(dst)[k] =
            make_uint4(pack_bf16x2(v[8 * k], v[8 * k + 1]), pack_bf16x2(v[8 * k + 2], v[8 * k + 3]),
                       pack_bf16x2(v[8 * k + 4], v[8 * k + 5]), pack_bf16x2(v[8 * k + 6], v[8 * k + 7]));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        reinterpret_cast<float4*>(dst)[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    }
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
  // four tokens a block once that still fills the GPU, one before: their heads are then spread over more SMs
  const int per_block = tokens >= 4 * kStoreTok * sm_count() ? kStoreTok : 1;
  const StoreArgs a{static_cast<const __nv_bfloat16*>(qkv), ld, positions, cache_loc, inv_freq, k_scale, v_scale,
                    static_cast<__nv_bfloat16*>(q), static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(k_sf),
                    static_cast<uint8_t*>(v_cache), static_cast<uint8_t*>(v_sf), tokens, hq, hkv, per_block,
                    !misaligned(qkv, 32) && (ld & 15) == 0, !misaligned(q, 32), cache_rows, status};
  const int grid = (tokens + per_block - 1) / per_block;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) {
    if (inv_freq) qk_rope_store_kv4_kernel<128, true><<<grid, kStoreThreads, 0, st>>>(a);
    else qk_rope_store_kv4_kernel<128, false><<<grid, kStoreThreads, 0, st>>>(a);
  } else {
    if (inv_freq) qk_rope_store_kv4_kernel<64, true><<<grid, kStoreThreads, 0, st>>>(a);
    else qk_rope_store_kv4_kernel<64, false><<<grid, kStoreThreads, 0, st>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? MSL_OK : MSL_ERR_CUDA;
}

extern "C" int msl_kv4_rows(const void* codes, const void* scales, const float* scale, const int64_t* rows, int64_t n,
                            int width, int64_t cache_rows, int out_mode, void* out, int* status, void* stream) {
  if (n < 0 || width <= 0 || cache_rows <= 0 || (out_mode != MSL_OUT_BF16 && out_mode != MSL_OUT_F32)) return MSL_ERR_ARG;
  if (n == 0) return MSL_OK;
  if (!codes || !scales || !scale || !rows || !out) return MSL_ERR_ARG;
  if ((width & 15) || misaligned(codes, 16) || misaligned(out, 16)) return MSL_ERR_ALIGN;
  const int blocks = width / 16;
  const int per = std::max(1, kRowsThreads / blocks);       // whole rows a CTA
  const int64_t grid = (n + per - 1) / per;
  if (grid > 0x7fffffff) return MSL_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto* c = static_cast<const uint8_t*>(codes);
  const auto* s = static_cast<const uint8_t*>(scales);
  if (out_mode == MSL_OUT_BF16)
    kv4_rows_kernel<<<static_cast<unsigned>(grid), kRowsThreads, 0, st>>>(
        c, s, scale, rows, n, blocks, per, cache_rows, static_cast<__nv_bfloat16*>(out), status);
  else
    kv4_rows_kernel<<<static_cast<unsigned>(grid), kRowsThreads, 0, st>>>(c, s, scale, rows, n, blocks, per, cache_rows,
                                                                         static_cast<float*>(out), status);
  return cudaGetLastError() == cudaSuccess ? MSL_OK : MSL_ERR_CUDA;
}
