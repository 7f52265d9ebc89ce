// Causal varlen attention over the paged 4-bit K/V cache, many query rows per KV head (prefill, chunks), on tcgen05.
//
// A block of work is (request, KV head, 2 * floor(128 / G) query tokens[, key slice]); two 128-row query sub-tiles
// (rows are (token, head in group) pairs) share every K/V tile.  One CTA per SM takes blocks one after another; requests
// of up to 128 rows share out all their key tiles equally instead (TcWalk below).  512 threads:
//   warps 0-3, 4-7  softmax groups of sub-tile 0 / 1, one thread per row, as in the FP8 kernel (csrc/attention_fp8.cu):
//                   the row of S in registers, maximum, exponentials, P written back to tensor memory over the first
//                   64 columns of the sub-tile's own S, in two halves; arithmetic on pairs of fp32.
//                   Before that each thread brings its query row into shared memory: scaled by a power of two to f16
//                   (largest magnitude in [2^14, 2^15)), so that one operand type serves both products.  The next
//                   block's queries come before this one's results, whose stores its first Q K^T then covers
//   warp  8         tensor memory and tcgen05.mma issue: S_s = Q_s K^T, O_s += P_s V (kind::f16, fp32 accumulators)
//   warps 12-15     producers: thread = key of the tile.  Codes and scales go from global memory to registers a tile
//                   ahead, become f16 (e2m1 conversion times the block scale: exact) and are stored as K-major (K) and
//                   N-major (V) swizzled operand tiles of a ring
//   warps 9-11      round the warpgroup up whose registers the others use; warp 9 looks for requests over max_q_len
// Registers are split 184 (softmax) / 56 / 88 (producers): 128 x (184 + 184 + 56 + 88) = 65536, the launch's total.
// P is f16 (half a step 2^-11) times 2^6, which with a lag of the running maximum of at most 2^8 stays below 2^15.
// A key whose page is missing is hidden: producers leave one bit per key, and the mask pass takes it with the causal
// limits.  Every wait is bounded.
//
// What bounds it: neither a pipe nor memory, but the chain S -> maximum -> exponentials -> P -> P V of each sub-tile,
// which two of them hide only in part, and instruction fetch.  4 x 2048 causal, 32 + 8 heads x 128: tensor pipe 34 %
// active, exponential unit 35 %, ALU 32 %, issue 38 %.  4 x 4096 (0.55 TFLOP) as the layer calls it, scores of a
// deviation near 5 and the norm and gate: 787 us = 699 TFLOP/s.  Where the scores are that wide the running maxima move
// often, and O is rescaled: without the gate 730 us, against 650 for scores of a deviation near 1 (715 with the gate; 592
// without the producers' loads, 616 without their conversion).
// Registers are short: at 128 a thread at launch the compiler spills 92 bytes of stores and 136 of loads (head_dim 128),
// 48 and 60 (head_dim 64), and 196 and 300 (196 and 296) where ranges are shared.
// Kept on the way, 4 x 4096, narrow scores: 1170 us -> 717 packed fp32 arithmetic, O rescaled before the exponentials, no turns at the
// exponential unit -> 665 MMAs issued four to a block in a rolled loop (a smaller loop for the fetch) -> 651 masks by
// bits; with the gate 832 -> 708 its division by a fast reciprocal.  753-token chunks over 80000 keys, page 1: 262 -> 230
// persistent CTAs, page entries a tile further ahead -> 216.
// Measured and not kept: turns at the exponential unit; a cubic in place of some exponentials (4 x 4096 767 us and more
// against 739 then); registers 176/56/104 (722 against 710); four lanes to a row in the epilogue (755 against 655); S read
// in pieces; separate warps for the queries; L2 prefetch of the keys two or three tiles ahead (no difference); for wide
// scores, O rescaled 32 columns at a time (no difference), two pieces in flight (763 against 723, registers), a lag of up
// to 2^9.75 (3 us).
#include "kv4_common.cuh"

namespace msl {

constexpr int kTM = 128;        // rows of a query sub-tile
constexpr int kTN = 128;        // keys of a tile
constexpr int kTcThreads = 512;
constexpr float kTcTau = 8.0f;
constexpr float kTcShift = 6.0f;

template <int D>
struct TcSmem {
  static constexpr int kTile = kTN * D * 2;                // bytes of one K, V or Q tile
  static constexpr int kStages = D == 128 ? 5 : 8;         // ring of K and V tiles in turn
  static constexpr int kQ = 0;                             // 2 sub-tiles
  static constexpr int kRing = 2 * kTile;
  static constexpr int kHeld = kRing + kStages * kTile;    // 8 x 4 words: the keys of a tile that have a page
  static constexpr int kBar = kHeld + 8 * 16;
  // q_full[2], full[stages], empty[stages], s_full[2], p_lo[2], p_hi[2], pv_done[2]
  static constexpr int kNumBars = 2 + 2 * kStages + 8;
  static constexpr int kTotal = kBar + kNumBars * 8 + 16;
};

template <int N>
__device__ __forceinline__ void reg_alloc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dealloc() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&o)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]),
      "r"(o[8]), "r"(o[9]), "r"(o[10]), "r"(o[11]), "r"(o[12]), "r"(o[13]), "r"(o[14]), "r"(o[15]), "r"(o[16]),
      "r"(o[17]), "r"(o[18]), "r"(o[19]), "r"(o[20]), "r"(o[21]), "r"(o[22]), "r"(o[23]), "r"(o[24]), "r"(o[25]),
      "r"(o[26]), "r"(o[27]), "r"(o[28]), "r"(o[29]), "r"(o[30]), "r"(o[31])
      : "memory");
}

__device__ __forceinline__ float tc_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float tc_row_max(const uint32_t (&s0)[32], const uint32_t (&s1)[32], float m) {
  float acc[4] = {m, -INFINITY, -INFINITY, -INFINITY};     // independent chains
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i & 3] = tc_max3(acc[i & 3], __uint_as_float(s0[i]), __uint_as_float(s1[i]));
  return fmaxf(fmaxf(acc[0], acc[1]), fmaxf(acc[2], acc[3]));
}
// Scores of keys that this row does not see become -inf: of the 32 columns from col0 on, lim_lo < column <= lim_hi and a
// cache row are needed.
__device__ __forceinline__ void tc_mask(uint32_t (&s)[32], int col0, int lim_hi, int lim_lo, uint32_t held) {
  const int hi = lim_hi - col0, lo = lim_lo - col0;         // columns in (lo, hi]
  uint32_t seen = held & (hi >= 31 ? 0xffffffffu : hi < 0 ? 0u : (2u << hi) - 1u);
  seen &= lo >= 31 ? 0u : lo < 0 ? 0xffffffffu : ~((2u << lo) - 1u);
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (!(seen & (1u << i))) s[i] = 0xff800000u;
}
// Two fp32 values an instruction: the FMA pipe takes half the issue slots.
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 unpack_f32x2(uint64_t v) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
  return d;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 32 columns of a row of S: exponentials summed (four chains) and packed as f16 pairs in key order.
__device__ __forceinline__ void tc_exp32(const uint32_t (&s)[32], uint64_t scale, uint64_t neg_m, uint64_t (&sum)[2],
                                         uint32_t* packed) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const float2 x = unpack_f32x2(fma_f32x2(f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), scale, neg_m));
    const float a = kv_ex2(x.x), b = kv_ex2(x.y);
    sum[(i / 2) & 1] = add_f32x2(sum[(i / 2) & 1], f32x2(a, b));
    packed[i / 2] = h2_bits(__floats2half2_rn(a, b));
  }
}

// Four K = 16 steps of S += Q K^T: both operands advance 32 bytes within a 128-byte swizzled row (descriptors count 16
// bytes).  One asm block, so that the issuing warp's loop stays small: it is fetched over and over between the softmax
// warps' (the issue of each instruction by itself, unrolled over the sub-tiles: 711 against 665 us for 4 x 4096).
__device__ __forceinline__ void tc_mma4_qk(uint32_t on, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "setp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.u64 a1, %1, 2;\n\tadd.u64 a2, %1, 4;\n\tadd.u64 a3, %1, 6;\n\t"
      "add.u64 b1, %2, 2;\n\tadd.u64 b2, %2, 4;\n\tadd.u64 b3, %2, 6;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(on)
      : "memory");
}
// Four K = 16 steps of O += P V: P advances 8 TMEM columns, V 16 rows of 128 bytes.
__device__ __forceinline__ void tc_mma4_pv(uint32_t on, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q, t;\n\t.reg .b64 b1, b2, b3;\n\t.reg .b32 a1, a2, a3;\n\t"
      "setp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\t"
      "add.u64 b1, %2, 128;\n\tadd.u64 b2, %2, 256;\n\tadd.u64 b3, %2, 384;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(on)
      : "memory");
}

// A key row's codes and scales as loaded.
template <int D>
struct TcRow {
  uint32_t c[D / 8];
  uint32_t s[D / 64];
};
template <int D>
__device__ __forceinline__ void tc_load_row(TcRow<D>& x, const uint8_t* codes, const uint8_t* scales, int row, int hkv,
                                            int kvh) {
#pragma unroll
  for (int i = 0; i < D / 8; ++i) x.c[i] = 0;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) x.s[i] = 0;
  if (row >= 0) {
    const int64_t at = static_cast<int64_t>(row) * hkv + kvh;
    const uint4* src = reinterpret_cast<const uint4*>(codes + at * (D / 2));
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint4 v = src[i];
      x.c[4 * i] = v.x; x.c[4 * i + 1] = v.y; x.c[4 * i + 2] = v.z; x.c[4 * i + 3] = v.w;
    }
    if constexpr (D == 128) {
      const uint2 v = *reinterpret_cast<const uint2*>(scales + at * 8);
      x.s[0] = v.x; x.s[1] = v.y;
    } else {
      x.s[0] = *reinterpret_cast<const uint32_t*>(scales + at * 4);
    }
  }
}
// ... as f16 into row r of a tile of 64-channel slabs [128 rows][128 bytes], 128-byte swizzle.
template <int D>
__device__ __forceinline__ void tc_store_row(const TcRow<D>& x, uint8_t* tile, int r) {
#pragma unroll
  for (int b = 0; b < D / 16; b += 2) {                     // two scale blocks of 16 channels
    const __half2 s2 = scales_h2((x.s[b / 4] >> (8 * (b & 3))) & 0xffffu);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const __half2 s = e ? __high2half2(s2) : __low2half2(s2);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int chunk = 2 * (b + e) + w;                  // 8 channels = 16 bytes
        __half2 h[4];
        e2m1x8(x.c[chunk], h);
        *reinterpret_cast<uint4*>(tile + (chunk / 8) * (kTN * 128) + swz128(r, chunk % 8)) =
            make_uint4(h2_bits(__hmul2(h[0], s)), h2_bits(__hmul2(h[1], s)), h2_bits(__hmul2(h[2], s)),
                       h2_bits(__hmul2(h[3], s)));
      }
    }
  }
}

// A block of work: up to 2 TQ query tokens of one request and KV head, and a slice of their key tiles.  Every role of a
// CTA walks the same list, block i, i + gridDim.x, ...; longest key ranges first (later query blocks see more keys).
struct TcItem {
  int b, kvh, split, q_begin, q_len, seq, kt_begin, key_lo, last_qpos, n_tiles;
  int first_tok[2], rows_valid[2], max_qpos[2], n_sub[2];  // per sub-tile: rows, last position, number of key tiles
};
__device__ __forceinline__ bool tc_item(const Kv4Args& p, int i, TcItem& it) {
  const int G = p.hq / p.hkv, TQ = kTM / G;
  it.split = i % p.kv_splits;
  i /= p.kv_splits;
  it.kvh = i % p.hkv;
  i /= p.hkv;
  it.b = i % p.batch;
  const int rank = i / p.batch;
  it.q_begin = max(0, min(p.cu_seqlens_q[it.b], p.tokens));
  it.q_len = min(max(0, min(p.cu_seqlens_q[it.b + 1], p.tokens) - it.q_begin), p.max_q_len);
  const int qblk = (it.q_len + 2 * TQ - 1) / (2 * TQ) - 1 - rank;
  if (qblk < 0) return false;
  const int q0 = qblk * 2 * TQ;
  it.seq = p.seq_lens[it.b];
  const int64_t table_keys = static_cast<int64_t>(p.max_pages) * p.page_size;
  it.key_lo = p.window ? max(0, it.seq + q0 - p.window + 1) : 0;
  it.kt_begin = it.key_lo / kTN;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    it.first_tok[s] = q0 + s * TQ;
    const int cnt = max(0, min(TQ, it.q_len - it.first_tok[s]));
    it.rows_valid[s] = cnt * G;
    it.max_qpos[s] = it.seq + it.first_tok[s] + cnt - 1;
    const int last_key = static_cast<int>(min(static_cast<int64_t>(it.max_qpos[s]), table_keys - 1));
    // one tile at least: a row that sees nothing is still written
    it.n_sub[s] = cnt > 0 ? max(1, last_key / kTN + 1 - it.kt_begin) : 0;
  }
  it.last_qpos = max(it.rows_valid[0] ? it.max_qpos[0] : -1, it.rows_valid[1] ? it.max_qpos[1] : -1);
  it.n_tiles = max(it.n_sub[0], it.n_sub[1]);
  if (p.kv_splits > 1) {                                    // a slice may be empty for one or both sub-tiles
    const int chunk = (it.n_tiles + p.kv_splits - 1) / p.kv_splits;
    const int lo = it.split * chunk, hi = min(it.n_tiles, lo + chunk);
#pragma unroll
    for (int s = 0; s < 2; ++s) it.n_sub[s] = max(0, min(it.n_sub[s], hi) - lo);
    it.kt_begin += lo;
    it.n_tiles = max(it.n_sub[0], it.n_sub[1]);
  }
  return true;
}
// What a CTA works on, item by item; every role of it makes the same walk.
//   SHARED = false  block i, i + gridDim.x, ... of the list above
//   SHARED = true   up to 128 rows a request (verify blocks): the key tiles of all requests and KV heads, laid end to
//                   end, are cut into equal ranges, one a CTA, as in csrc/attention_kv4.cu; the two sub-tiles hold the same
//                   rows and take the tiles of an item in turn.  Producers that load two tiles ahead, in registers taken
//                   from the softmax warps (168/56/120), need 99 us for 16 x 8 x 4096 against 78.  16 requests x 8 tokens after 500 .. 8192: 94 us
//                   against 125 with the requests' own slices.
template <bool SHARED>
struct TcWalk;
template <>
struct TcWalk<false> {
  int i;                                                    // next block
};
template <>
struct TcWalk<true> {
  int b;                                                    // request
  int64_t skip, at, end;                                    // its tiles before; the range that is left
};
__device__ __forceinline__ bool tc_next(const Kv4Args& p, int n_items, TcWalk<false>& w, TcItem& it) {
  for (; w.i < n_items; w.i += gridDim.x)
    if (tc_item(p, w.i, it)) return true;
  return false;
}
__device__ __forceinline__ void tc_step(TcWalk<false>& w) { w.i += gridDim.x; }
__device__ __forceinline__ void tc_step(TcWalk<true>&) {}
__device__ __forceinline__ bool tc_next(const Kv4Args& p, int, TcWalk<true>& w, TcItem& it) {
  while (w.at < w.end && w.b < p.batch) {
    const Kv4Req r = kv4_request(p, w.b);
    if (r.len <= 0) { ++w.b; continue; }
    const Kv4Span span = kv4_span(p, r, 7);
    const int n_span = span.last - span.first, off = static_cast<int>(w.skip % n_span);
    it.b = w.b;
    it.kvh = static_cast<int>(w.skip / n_span);
    it.q_begin = r.begin;
    it.q_len = r.len;
    it.seq = r.seq;
    it.key_lo = p.window ? max(0, r.seq - p.window + 1) : 0;
    it.kt_begin = span.first + off;
    it.last_qpos = r.seq + r.len - 1;
    it.n_tiles = static_cast<int>(min(w.end - w.at, static_cast<int64_t>(n_span - off)));
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      it.first_tok[s] = 0;
      it.rows_valid[s] = r.len * (p.hq / p.hkv);
      it.max_qpos[s] = it.last_qpos;
      it.n_sub[s] = (it.n_tiles + 1 - s) / 2;
    }
    // where its result goes: an item has one beginning (-1), a CTA at most one rest of an item that an earlier one began
    it.split = off == 0 ? -1 : static_cast<int>(blockIdx.x);
    w.at += it.n_tiles;
    w.skip += it.n_tiles;
    if (w.skip == static_cast<int64_t>(n_span) * p.hkv) { w.skip = 0; ++w.b; }
    return true;
  }
  return false;
}

// Place of the tiles of an item with n tiles in the order in which the ring carries them: `lag` K tiles first, then V(j)
// and K(j + lag) in turn.
__device__ __forceinline__ int tc_place_k(int j, int lag) { return j < lag ? j : 2 * j - lag + 1; }
__device__ __forceinline__ int tc_place_v(int j, int n, int lag) { return min(lag, n) + j + min(j, max(n - lag, 0)); }

// Rows of partial results of shared ranges: two sub-tiles' beginnings of each query row, and `ctas` CTAs' rests.
__host__ __device__ __forceinline__ int64_t kv4_tc_shared_parts(int tokens, int hq, int ctas, int max_rows) {
  return 2 * (static_cast<int64_t>(tokens) * hq + static_cast<int64_t>(ctas) * max_rows);
}

template <int D, bool SHARED>
__global__ void __launch_bounds__(kTcThreads, 1)
attention_kv4_tc_kernel(Kv4Args p, int n_items) {
  using S = TcSmem<D>;
  constexpr int kSt = S::kStages;
  constexpr int kSlab = kTN * 128;                         // 128 rows x 64 f16 channels
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBar);
  uint64_t* q_full = bars;
  uint64_t* full = bars + 2;
  uint64_t* empty = full + kSt;
  uint64_t* s_full = empty + kSt;
  uint64_t* p_lo = s_full + 2;
  uint64_t* p_hi = p_lo + 2;
  uint64_t* pv_done = p_hi + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S::kNumBars);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  uint32_t* held = reinterpret_cast<uint32_t*>(smem + S::kHeld);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int lag = SHARED ? 2 : 1;
  TcWalk<SHARED> walk0;
  if constexpr (!SHARED) {
    walk0.i = blockIdx.x;
  } else {
    pdl_launch_dependents();
    __shared__ int64_t scratch[kTcThreads / 32];
    __shared__ TcWalk<true> found;
    const auto tiles_of = [&](int b) {
      const Kv4Req r = kv4_request(p, b);
      const Kv4Span span = kv4_span(p, r, 7);
      return r.len > 0 ? static_cast<int64_t>(span.last - span.first) * p.hkv : 0;
    };
    const int per = (p.batch + kTcThreads - 1) / kTcThreads;
    const int b0 = min(static_cast<int>(threadIdx.x) * per, p.batch), b1 = min(b0 + per, p.batch);
    int64_t mine = 0, total = 0;
    for (int b = b0; b < b1; ++b) {
      if (blockIdx.x == 0 && kv4_request(p, b).over) report_error(p.status, MSL_ERR_CAPACITY);
      mine += tiles_of(b);
    }
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    for (int w = 0; w < kTcThreads / 32; ++w) {
      if (w < warp) inc += scratch[w];
      total += scratch[w];
    }
    const int64_t workers = min(static_cast<int64_t>(gridDim.x), total);   // no empty range in between
    if (blockIdx.x >= workers) return;                      // uniform, before any barrier of the roles
    const int64_t at = total * blockIdx.x / workers;
    if (inc - mine <= at && at < inc) {                     // one thread: walk its few requests
      int64_t base = inc - mine;
      int b = b0;
      for (; b < b1 - 1 && at >= base + tiles_of(b); ++b) base += tiles_of(b);
      found = TcWalk<true>{b, at - base, at, total * (blockIdx.x + 1) / workers};
    }
    __syncthreads();
    walk0 = found;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSt; ++i) { mbar_init(&full[i], 4); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_lo[i], 4);
      mbar_init(&p_hi[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 8) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp >= 12) {
    // ------------------------------------------------------------------ producers: thread = key of the tile
    reg_dealloc<88>();
    const int r = (warp - 12) * 32 + lane;
    bool ok = true;
    int pos = 0, tiles = 0;                                 // ring places and tiles of the items before
    TcWalk<SHARED> walk = walk0;
    TcItem it;
    for (; ok && tc_next(p, n_items, walk, it); tc_step(walk)) {
      if (it.n_tiles == 0) continue;
      const int n = it.n_tiles;
      const int* table = p.page_table + static_cast<int64_t>(it.b) * p.max_pages;
      const int first_key = it.kt_begin * kTN + r, hi = it.last_qpos + 1;
      if (r == 0 && hi > static_cast<int64_t>(p.max_pages) * p.page_size) report_error(p.status, MSL_ERR_CAPACITY);
      const auto page_of = [&](int j) {
        return j < n ? kv4_page(p, table, first_key + j * kTN, it.key_lo, hi) : Kv4Page{INT_MIN, 0};
      };
      // this thread's key in tiles j .. j + 3: its cache rows, and the table entry of the next, on its way
      Kv4Page ahead = page_of(0), ahead1 = page_of(1), ahead2 = page_of(2), ahead3 = page_of(3);
      int row0 = kv4_row_of(p, ahead), row1 = kv4_row_of(p, ahead1), row2 = kv4_row_of(p, ahead2),
          row3 = kv4_row_of(p, ahead3);
      ahead = page_of(4);
      TcRow<D> k, v;
      tc_load_row<D>(k, p.k, p.ks, row0, p.hkv, it.kvh);
      tc_load_row<D>(v, p.v, p.vs, row0, p.hkv, it.kvh);
      const auto put = [&](const TcRow<D>& x, int place) {  // into the ring; false: the wait ran out
        const int st = (pos + place) % kSt;
        if (*abort_flag || !mbar_wait(&empty[st], (((pos + place) / kSt) & 1) ^ 1, true)) return false;
        tc_store_row<D>(x, smem + S::kRing + st * S::kTile, r);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
        return true;
      };
      const auto put_k = [&](int j, int row, int row_next) {
        const uint32_t mask = __ballot_sync(0xffffffffu, row >= 0);
        if (lane == 0) held[((tiles + j) & 7) * 4 + warp - 12] = mask;
        if (!put(k, tc_place_k(j, lag))) return false;
        if (j + 1 < n) tc_load_row<D>(k, p.k, p.ks, row_next, p.hkv, it.kvh);
        return true;
      };
      ok = put_k(0, row0, row1);
      if (ok && lag == 2 && n > 1) ok = put_k(1, row1, row2);
      for (int j = 0; j < n && ok; ++j) {
        const int row4 = kv4_row_of(p, ahead);
        ahead = page_of(j + 5);
        if (!put(v, tc_place_v(j, n, lag))) { ok = false; break; }
        if (j + 1 < n) tc_load_row<D>(v, p.v, p.vs, row1, p.hkv, it.kvh);
        if (j + lag < n) ok = put_k(j + lag, lag == 2 ? row2 : row1, lag == 2 ? row3 : row2);
        row0 = row1; row1 = row2; row2 = row3; row3 = row4;
      }
      pos += 2 * n;
      tiles += n;
    }
    if (!ok && lane == 0) { *abort_flag = 1; report_error(p.status, MSL_ERR_DEVICE_TIMEOUT); }
  } else if (warp >= 8) {
    reg_dealloc<56>();
    if (warp == 8) {
      // ---------------------------------------------------------------- MMA issuer (warp-uniform, one elected lane)
      const uint32_t on = elect_one();
      constexpr uint32_t idesc_qk = make_idesc(0, 0, kTM, kTN);
      constexpr uint32_t idesc_pv = make_idesc(0, 0, kTM, D, 0, 1);     // A = P from TMEM (K-major), B = V, N-major
      const uint32_t sq = smem_u32(smem + S::kQ), ring = smem_u32(smem + S::kRing);
      const auto issue_qk = [&](int s, uint32_t sk) {
        const uint64_t a = make_sdesc(sq + s * S::kTile, 16, 1024, 2), b = make_sdesc(sk, 16, 1024, 2);
#pragma unroll
        for (int k = 0; k < D / 64; ++k)                   // a slab of 64 channels each
          tc_mma4_qk(on, tmem_base + s * kTN, a + k * (kSlab >> 4), b + k * (kSlab >> 4), idesc_qk, k != 0);
        tc_commit_if(on, &s_full[s]);
      };
      // keys [64 half, 64 half + 64) of the tile: P columns [32 half, +32) of the sub-tile's S
      const auto issue_pv_half = [&](int s, uint32_t sv, int half, bool first) {
        tc_mma4_pv(on, tmem_base + 2 * kTN + s * kTN, tmem_base + s * kTN + 32 * half,
                   make_sdesc(sv + half * 64 * 128, kSlab, 1024, 2), idesc_pv, !(first && half == 0));
      };
      bool ok = true;
      int pos = 0, taken0 = 0, taken1 = 0;                  // ring places of, and items with tiles for, the sub-tiles before
      int done0 = 0, done1 = 0;                             // their tiles
      TcWalk<SHARED> walk = walk0;
      TcItem it;
      for (; ok && tc_next(p, n_items, walk, it); tc_step(walk)) {
        if (it.n_tiles == 0) continue;
        const int n = it.n_tiles;
        const auto wait_full = [&](int place) {
          const bool got = !*abort_flag && mbar_wait(&full[place % kSt], (place / kSt) & 1);
          tc_fence_after();
          return got;
        };
        // a sub-tile's queries, where it has any tiles (the groups may be items apart where it has none)
        if (it.n_sub[0] > 0) ok = !*abort_flag && mbar_wait(&q_full[0], taken0++ & 1);
        if (it.n_sub[1] > 0) ok = ok && !*abort_flag && mbar_wait(&q_full[1], taken1++ & 1);
        for (int j = 0; j < min(lag, n) && ok; ++j) {
          const int place = pos + tc_place_k(j, lag);
          ok = wait_full(place);
          if (!ok) break;
          const uint32_t sk = ring + (place % kSt) * S::kTile;
#pragma unroll 1
          for (int s = 0; s < 2; ++s)
            if (SHARED ? s == j : (s ? it.n_sub[1] : it.n_sub[0]) > 0) issue_qk(s, sk);
          tc_commit_if(on, &empty[place % kSt]);
        }
        for (int j = 0; j < n && ok; ++j) {
          const int pv = pos + tc_place_v(j, n, lag), pk = pos + tc_place_k(j + lag, lag);
          const uint32_t sv = ring + (pv % kSt) * S::kTile, sk = ring + (pk % kSt) * S::kTile;
          const int local = SHARED ? j >> 1 : j;       // this tile's number among the sub-tile's own
          bool v_ready = false, k_ready = false;
#pragma unroll 1
          for (int s = 0; s < 2; ++s) {
            const int mine = s ? it.n_sub[1] : it.n_sub[0];
            if (!(SHARED ? (j & 1) == s : j < mine)) continue;
            const uint32_t ph = ((s ? done1 : done0) + local) & 1;
            if (!v_ready) {
              if (!wait_full(pv)) { ok = false; break; }
              v_ready = true;
            }
            if (*abort_flag || !mbar_wait(&p_lo[s], ph)) { ok = false; break; }
            tc_fence_after();
            issue_pv_half(s, sv, 0, local == 0);
            if (*abort_flag || !mbar_wait(&p_hi[s], ph)) { ok = false; break; }
            tc_fence_after();
            issue_pv_half(s, sv, 1, false);
            if (local == mine - 1) tc_commit_if(on, &pv_done[s]);
            if (local + 1 < mine) {
              if (!k_ready) {
                if (!wait_full(pk)) { ok = false; break; }
                k_ready = true;
              }
              issue_qk(s, sk);
            }
          }
          if (!ok) break;
          tc_commit_if(on, &empty[pv % kSt]);
          if (k_ready) tc_commit_if(on, &empty[pk % kSt]);
        }
        pos += 2 * n;
        done0 += it.n_sub[0];
        done1 += it.n_sub[1];
      }
      if (!ok && lane == 0) { *abort_flag = 1; report_error(p.status, MSL_ERR_DEVICE_TIMEOUT); }
    } else if (!SHARED && warp == 9 && blockIdx.x == 0) {
      for (int b = lane; b < p.batch; b += 32)
        if (kv4_request(p, b).over) report_error(p.status, MSL_ERR_CAPACITY);
    }
  } else {
    // ------------------------------------------------------------------ softmax / correction / epilogue
    reg_alloc<184>();
    const int G = p.hq / p.hkv;
    const int sub = warp >> 2;                             // query sub-tile of this group
    const int r = (warp & 3) * 32 + lane;                  // row = TMEM lane
    const int tq = r / G, g = r - tq * G;
    const float scale0 = p.softmax_scale * (*p.k_scale) * 1.4426950408889634f;
    const uint32_t lane_sel = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tmem_s = tmem_base + sub * kTN + lane_sel;
    const uint32_t tmem_o = tmem_base + 2 * kTN + sub * kTN + lane_sel;
    // Partial results: slices of a query block's keys by (slice, token, head); of shared ranges the beginnings of items by
    // (sub-tile, token, head), then the rests by (CTA, sub-tile, row).  Without any a row is written at once.
    const bool partial = SHARED || p.kv_splits > 1;
    const int max_rows = p.max_q_len * G;
    float* part_ml = p.part + (SHARED ? kv4_tc_shared_parts(p.tokens, p.hq, gridDim.x, max_rows)
                                      : static_cast<int64_t>(p.kv_splits) * p.tokens * p.hq) * D;
    const auto part_index = [&](const TcItem& it, int64_t token) {
      if (SHARED && it.split >= 0)
        return kv4_tc_shared_parts(p.tokens, p.hq, it.split, max_rows) + static_cast<int64_t>(sub) * max_rows + r;
      return (static_cast<int64_t>(SHARED ? sub : it.split) * p.tokens + token) * p.hq + it.kvh * G + g;
    };
    // What the main loop needs of an item; the rest is formed again for the results.
    struct Mine {
      int n_tiles, n, kt_begin, qpos, min_qpos, max_qpos;
      float scale_log2;
    };
    // The next item with tiles from i on; where this sub-tile has some, its query rows go to shared memory (every
    // Q K^T of the sub-tile before has finished: its last S has been waited for).  Empty slices are dealt with here.
    const auto take = [&](TcWalk<SHARED>& walk, TcWalk<SHARED>& before, Mine& m) {
      for (;; tc_step(walk)) {
        TcItem it;
        if constexpr (SHARED) before = walk;
        if (!tc_next(p, n_items, walk, it)) return false;
        const int first_tok = sub ? it.first_tok[1] : it.first_tok[0];
        const bool valid = r < (sub ? it.rows_valid[1] : it.rows_valid[0]);
        const int64_t token = static_cast<int64_t>(it.q_begin) + first_tok + tq;
        if (it.n_tiles == 0) {
          if (valid) {
            const int64_t idx = part_index(it, token);
            part_ml[2 * idx] = -INFINITY;
            part_ml[2 * idx + 1] = 0.f;
          }
          continue;
        }
        m.n_tiles = it.n_tiles;
        m.n = sub ? it.n_sub[1] : it.n_sub[0];
        m.kt_begin = it.kt_begin;
        m.qpos = it.seq + min(first_tok + tq, max(it.q_len - 1, 0));
        m.min_qpos = it.seq + first_tok;
        m.max_qpos = sub ? it.max_qpos[1] : it.max_qpos[0];
        if (m.n == 0) return true;
        // f16 with the largest magnitude in [2^14, 2^15)
        const uint4* src = reinterpret_cast<const uint4*>(p.q + token * p.ld_q + (it.kvh * G + g) * D);
        uint8_t* dst = smem + S::kQ + sub * S::kTile;
        uint32_t w[D / 2];
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
          uint4 u = make_uint4(0, 0, 0, 0);
          if (valid) u = src[x];
          w[4 * x] = u.x; w[4 * x + 1] = u.y; w[4 * x + 2] = u.z; w[4 * x + 3] = u.w;
        }
        uint32_t mx = 0;
#pragma unroll
        for (int x = 0; x < D / 2; ++x) mx = max(mx, max(w[x] & 0x7fffu, (w[x] >> 16) & 0x7fffu));
        const int e = min(max(static_cast<int>(mx >> 7), 16), 254);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 141 - e) << 23);
        m.scale_log2 = kv4_row_scale(scale0, up);
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
          uint32_t h[4];
#pragma unroll
          for (int y = 0; y < 4; ++y)
            h[y] = h2_bits(__floats2half2_rn(bf16_bits_to_f32(w[4 * x + y] & 0xffffu) * up,
                                             bf16_bits_to_f32(w[4 * x + y] >> 16) * up));
          *reinterpret_cast<uint4*>(dst + (x / 8) * kSlab + swz128(r, x % 8)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[sub]);
        return true;
      }
    };

    bool ok = true;
    int done = 0, tiles = 0, outs = 0;                      // of this sub-tile, of the CTA, results: items before
    TcWalk<SHARED> walk = walk0, before, at;
    Mine next;
    next.scale_log2 = 0.f;
    bool more = take(walk, before, next);
    while (more && ok) {
      const Mine m = next;
      if constexpr (SHARED) at = before;
      else at = walk;
      const float scale_log2 = m.scale_log2;
      float m_run = -INFINITY, l_run = 0.f;                // l accumulates 2^kTcShift * sum of exponentials
      for (int j = 0; j < m.n && ok; ++j) {
        const int tile = SHARED ? 2 * j + sub : j;
        const int key0 = (m.kt_begin + tile) * kTN;
        if (*abort_flag || !mbar_wait(&s_full[sub], (done + j) & 1)) { ok = false; break; }
        tc_fence_after();
        const uint4 hm = *reinterpret_cast<const uint4*>(held + ((tiles + tile) & 7) * 4);
        const bool full_tile = (key0 + kTN - 1 <= m.min_qpos) && (!p.window || key0 > m.max_qpos - p.window) &&
                               (hm.x & hm.y & hm.z & hm.w) == 0xffffffffu;
        const int lim_hi = m.qpos - key0;                   // visible columns: lim_lo < col <= lim_hi
        const int lim_lo = p.window ? m.qpos - p.window - key0 : -1;
        uint32_t sa[32], sb[32], sc[32], sd[32];
        tmem_ld32(tmem_s, sa);
        tmem_ld32(tmem_s + 32, sb);
        tmem_ld32(tmem_s + 64, sc);
        tmem_ld32(tmem_s + 96, sd);
        tmem_ld_wait();
        if (!full_tile) {
          tc_mask(sa, 0, lim_hi, lim_lo, hm.x);
          tc_mask(sb, 32, lim_hi, lim_lo, hm.y);
          tc_mask(sc, 64, lim_hi, lim_lo, hm.z);
          tc_mask(sd, 96, lim_hi, lim_lo, hm.w);
        }
        const float m_cand = tc_row_max(sc, sd, tc_row_max(sa, sb, -INFINITY)) * scale_log2;
        // A row's reference maximum moves when the row exceeds it by more than tau, or finds its first visible key.
        // Each row decides for itself, so that its bits do not depend on its neighbours; the warp rescales together.
        const bool move = m_cand > m_run + kTcTau || (m_run == -INFINITY && m_cand > -INFINITY);
        float corr = 1.0f;
        if (__any_sync(0xffffffffu, move)) {
          if (move) {
            corr = kv_ex2(m_run - m_cand);                  // 0 when m_run = -inf
            m_run = m_cand;
          }
          if (j > 0) {
            // O moves to the new maximum before any of this tile's P is used.  S was ready only after the P V before
            // had finished (the tensor pipe ran it first), so O is quiet.  Small pieces: the scores hold the registers.
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t oa[16];
              tmem_ld16(tmem_o + c, oa);
              tmem_ld_wait();
#pragma unroll
              for (int x = 0; x < 16; ++x) oa[x] = __float_as_uint(__uint_as_float(oa[x]) * corr);
              tmem_st16(tmem_o + c, oa);
            }
          }
        }
        const float m_use = (m_run == -INFINITY) ? 0.f : m_run;
        const uint64_t scale2 = f32x2(scale_log2, scale_log2), neg_m2 = f32x2(kTcShift - m_use, kTcShift - m_use);
        uint64_t sum[2] = {0, 0};                           // two pairs of +0
        {
          uint32_t pk[32];
          tc_exp32(sa, scale2, neg_m2, sum, pk);
          tc_exp32(sb, scale2, neg_m2, sum, pk + 16);
          tc_st32(tmem_s, pk);
        }
        uint32_t pk[32];
        tc_exp32(sc, scale2, neg_m2, sum, pk);              // the first half's stores land meanwhile
        tmem_st_wait();                                     // P's first half and a rescaled O
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_lo[sub]);
        tc_exp32(sd, scale2, neg_m2, sum, pk + 16);
        tc_st32(tmem_s + 32, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_hi[sub]);
        const float2 total = unpack_f32x2(add_f32x2(sum[0], sum[1]));
        l_run = l_run * corr + (total.x + total.y);
      }
      if (!ok) break;
      done += m.n;
      tiles += m.n_tiles;
      // The next item's queries before this one's results: its first Q K^T runs behind the last P V.
      tc_step(walk);
      more = take(walk, before, next);

      // -------------------------------------------------------------- epilogue
      TcItem it;
      if constexpr (SHARED) tc_next(p, n_items, at, it);
      else tc_item(p, at.i, it);
      const int n_mine = m.n;
      const bool row_valid = r < (sub ? it.rows_valid[1] : it.rows_valid[0]);
      const int64_t token = static_cast<int64_t>(it.q_begin) + (sub ? it.first_tok[1] : it.first_tok[0]) + tq;
      const int head = it.kvh * G + g;
      if (n_mine > 0) {
        if (*abort_flag || !mbar_wait(&pv_done[sub], outs & 1)) { ok = false; break; }   // behind the last P V
        ++outs;
        tc_fence_after();
      }
      if (partial) {
        // partial result of these key tiles: O as it stands in TMEM, with the maximum and sum it refers to
        const int64_t idx = part_index(it, token);
        if (row_valid) {
          part_ml[2 * idx] = m_run;
          part_ml[2 * idx + 1] = l_run;
        }
        if (n_mine > 0) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(tmem_o + c, o);
            tmem_ld_wait();
            if (row_valid) {
              float4* dst = reinterpret_cast<float4*>(p.part + idx * D + c);
#pragma unroll
              for (int x = 0; x < 8; ++x)
                dst[x] = make_float4(__uint_as_float(o[4 * x]), __uint_as_float(o[4 * x + 1]),
                                     __uint_as_float(o[4 * x + 2]), __uint_as_float(o[4 * x + 3]));
            }
          }
        }
      } else if (n_mine > 0) {
        // l carries the same power of two as P; a row that sees nothing is zero, a NaN sum (a NaN query) stays visible
        const float c_out = l_run > 0.f ? (*p.v_scale) / l_run : (l_run != l_run ? l_run : 0.f);
        float r_norm = 1.0f;
        if (p.gate != nullptr) {
          float ss = 0.f;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(tmem_o + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 32; ++x) { const float y = __uint_as_float(o[x]) * c_out; ss += y * y; }
          }
          r_norm = 1.0f / sqrtf(ss / D + 1e-5f);
        }
        __nv_bfloat16* orow = p.out + token * p.ld_out + head * D;
        const __nv_bfloat16* grow = p.gate ? p.gate + token * p.ld_gate + head * D : nullptr;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld32(tmem_o + c, o);
          tmem_ld_wait();
          if (row_valid) {
            float v[32];
#pragma unroll
            for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(o[x]) * c_out * r_norm;
            if (grow != nullptr) {
#pragma unroll
              for (int x = 0; x < 32; x += 8) {
                const uint4 gq = *reinterpret_cast<const uint4*>(grow + c + x);
                const uint32_t gw[4] = {gq.x, gq.y, gq.z, gq.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  v[x + 2 * e] *= __fdividef(1.0f, 1.0f + __expf(-bf16_bits_to_f32(gw[e] & 0xffffu)));
                  v[x + 2 * e + 1] *= __fdividef(1.0f, 1.0f + __expf(-bf16_bits_to_f32(gw[e] >> 16)));
                }
              }
            }
#pragma unroll
            for (int x = 0; x < 32; x += 8)
              *reinterpret_cast<uint4*>(orow + c + x) =
                  make_uint4(pack_bf16x2(v[x], v[x + 1]), pack_bf16x2(v[x + 2], v[x + 3]),
                             pack_bf16x2(v[x + 4], v[x + 5]), pack_bf16x2(v[x + 6], v[x + 7]));
          }
        }
      }
    }
    if (!ok && lane == 0) { *abort_flag = 1; report_error(p.status, MSL_ERR_DEVICE_TIMEOUT); }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    tmem_dealloc(tmem_base, 512);
  }
}

// Joins the key slices: one warp per (token, head); slice s holds O and l relative to its own maximum.  Rows that no
// request owns are left as they are, so the request of a row is looked up first.
template <int D>
__global__ void __launch_bounds__(256)
kv4_tc_merge_kernel(Kv4Args p) {
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  const int q_begin = max(0, min(p.cu_seqlens_q[b], p.tokens));
  const int q_len = min(max(0, min(p.cu_seqlens_q[b + 1], p.tokens) - q_begin), p.max_q_len);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (item >= static_cast<int64_t>(q_len) * p.hq) return;
  const int64_t token = q_begin + item / p.hq;
  const int head = static_cast<int>(item % p.hq);
  const int slots = p.kv_splits;
  const float* part_ml = p.part + static_cast<int64_t>(slots) * p.tokens * p.hq * D;
  const int64_t stride = static_cast<int64_t>(p.tokens) * p.hq, base = token * p.hq + head;
  float mx = -INFINITY;
  for (int s = 0; s < slots; ++s) mx = fmaxf(mx, part_ml[2 * (s * stride + base)]);
  float acc[PER], sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = 0.f;
  for (int s = 0; s < slots; ++s) {
    const int64_t at = s * stride + base;
    const float l = part_ml[2 * at + 1];
    if (l == 0.f) continue;                                 // an empty slice wrote no O
    const float w = kv_ex2(part_ml[2 * at] - (mx == -INFINITY ? 0.f : mx));
    sum += l * w;
    const float* o = p.part + at * D + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] += o[i] * w;
  }
  kv4_write_row<D>(p, acc, sum, token, head, lane);
}

// Joins the partial results of shared ranges: one CTA per (KV head, request, eight rows), a warp a row.
template <int D>
__global__ void __launch_bounds__(256)
kv4_tc_shared_merge_kernel(Kv4Args p, int ctas) {
  constexpr int PER = D / 32;
  __shared__ int64_t scratch[8];
  const int lane = threadIdx.x & 31, b = blockIdx.y, kvh = blockIdx.x, G = p.hq / p.hkv;
  const int row = blockIdx.z * 8 + (threadIdx.x >> 5);
  int64_t before = 0, all = 0;
  for (int x = threadIdx.x; x < p.batch; x += blockDim.x) {
    const Kv4Req r = kv4_request(p, x);
    const Kv4Span span = kv4_span(p, r, 7);
    const int64_t n = r.len > 0 ? static_cast<int64_t>(span.last - span.first) * p.hkv : 0;
    all += n;
    if (x < b) before += n;
  }
  before = block_sum_i64<8>(before, scratch);
  all = block_sum_i64<8>(all, scratch);
  const Kv4Req r = kv4_request(p, b);
  pdl_wait();                               // in every block: this grid ends only after the one before it
  if (row >= r.len * G) return;
  const Kv4Span span = kv4_span(p, r, 7);
  const int n_span = span.last - span.first;
  const int64_t t0 = before + static_cast<int64_t>(kvh) * n_span, t1 = t0 + n_span;   // this item's tiles
  // tile t belongs to the largest w with floor(all * w / workers) <= t
  const int64_t workers = min(static_cast<int64_t>(ctas), all);
  const int w0 = static_cast<int>(((t0 + 1) * workers - 1) / all), w1 = static_cast<int>((t1 * workers - 1) / all);
  const int max_rows = p.max_q_len * G, n = 2 * (w1 - w0 + 1);
  const int64_t token = static_cast<int64_t>(r.begin) + row / G;
  const int head = kvh * G + row % G;
  const float* part_ml = p.part + kv4_tc_shared_parts(p.tokens, p.hq, ctas, max_rows) * D;
  // the i-th partial result: sub-tile i % 2 of CTA w0 + i / 2, the first CTA's the beginning
  const auto index = [&](int i) {
    return i < 2 ? (static_cast<int64_t>(i) * p.tokens + token) * p.hq + head
                 : kv4_tc_shared_parts(p.tokens, p.hq, w0 + i / 2, max_rows) + static_cast<int64_t>(i & 1) * max_rows + row;
  };
  float mx = -INFINITY;
  for (int i = lane; i < n; i += 32) mx = fmaxf(mx, part_ml[2 * index(i)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float ref = mx == -INFINITY ? 0.f : mx;
  float acc[PER], sum = 0.f;
#pragma unroll
  for (int x = 0; x < PER; ++x) acc[x] = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const int64_t at = index(i);
    const float l = part_ml[2 * at + 1];
    if (l == 0.f) continue;                                 // a sub-tile without tiles wrote no O
    const float c = kv_ex2(part_ml[2 * at] - ref);
    sum += l * c;
    const float* o = p.part + at * D + lane * PER;
#pragma unroll
    for (int x = 0; x < PER; ++x) acc[x] += o[x] * c;
  }
  kv4_write_row<D>(p, acc, sum, token, head, lane);
}

template <int D, bool SHARED>
static int launch_tc(const Kv4Args& a, cudaStream_t st) {
  const int smem = TcSmem<D>::kTotal + 1024;
  static SmemConfig config;
  if (int rc = config.ensure(attention_kv4_tc_kernel<D, SHARED>, smem)) return rc;
  if constexpr (SHARED) {
    const int ctas = sm_count();
    attention_kv4_tc_kernel<D, true><<<ctas, kTcThreads, smem, st>>>(a, 0);
    if (cudaGetLastError() != cudaSuccess) return MSL_ERR_CUDA;
    // The merge forms its schedule while the attention runs and waits for it on the device (programmatic launch).
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.hkv, a.batch, (a.max_q_len * (a.hq / a.hkv) + 7) / 8);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_tc_shared_merge_kernel<D>, a, ctas) == cudaSuccess ? MSL_OK : MSL_ERR_CUDA;
  }
  const int tq2 = 2 * (kTM / (a.hq / a.hkv));
  const int64_t items = static_cast<int64_t>((a.max_q_len + tq2 - 1) / tq2) * a.kv_splits * a.hkv * a.batch;
  if (items > 0x7fffffff) return MSL_ERR_UNSUPPORTED;
  attention_kv4_tc_kernel<D, false><<<static_cast<int>(std::min<int64_t>(items, sm_count())), kTcThreads, smem, st>>>(
      a, static_cast<int>(items));
  if (a.kv_splits > 1) {
    const int64_t rows = static_cast<int64_t>(a.max_q_len) * a.hq;
    kv4_tc_merge_kernel<D><<<dim3(static_cast<unsigned>((rows + 7) / 8), a.batch), 256, 0, st>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? MSL_OK : MSL_ERR_CUDA;
}

int launch_kv4_tc(const Kv4Args& a, int head_dim, cudaStream_t st) {
  if (a.alternate) return head_dim == 128 ? launch_tc<128, true>(a, st) : launch_tc<64, true>(a, st);
  return head_dim == 128 ? launch_tc<128, false>(a, st) : launch_tc<64, false>(a, st);
}

// Two partial results of two sub-tiles a CTA.
int64_t kv4_tc_shared_workspace(int rows, int tokens, int hq, int head_dim) {
  return kv4_tc_shared_parts(tokens, hq, sm_count(), rows) * (head_dim + 2) * 4;
}

int64_t kv4_tc_workspace(int slots, int tokens, int hq, int head_dim) {
  return slots <= 1 ? 0 : static_cast<int64_t>(slots) * tokens * hq * (head_dim + 2) * 4;
}

}  // namespace msl
