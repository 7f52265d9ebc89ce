// Causal varlen attention over the paged 4-bit K/V cache (format: csrc/kv4.cu), up to 16 query rows per KV head: decode
// steps.  More rows: csrc/attention_kv4_tc.cu.
//
// A worker (one CTA) owns an equal share of all key tiles of the batch: the tiles of every request and group of KV heads
// are laid end to end and cut into equal ranges, so ragged lengths cost nothing.  A range that covers all tiles of a
// work item writes its rows; the others leave (O, maximum, sum) in the workspace and kv4_merge_kernel joins them.
// The ranges follow from the lengths, which live on the device: both kernels form the same sums, no host knows them.
//
// A warp takes 32 keys of one KV head at a time, from a ring of cp.async stages in shared memory into registers, in
// the layout of the MMA operands (mma.sync: the operands change hands in registers, and a decode step has far too few
// rows for the 128 of a tcgen05 tile).  The contraction index of Q K^T and the row index of O^T may be permuted
// freely, and the permutation is chosen so that a lane's share is contiguous in memory:
//   S^T[key][q] = K Q^T   lane (g, t) holds channels [D/4 t, D/4 (t+1)) of keys g and g + 8: one 16-byte load
//                         (8 at head_dim 64), whose elements lie in at most two scale blocks
//   O^T[d][q]  += V^T P^T lane (g, t) holds channels [D/8 g, D/8 (g+1)) of keys 2t, 2t+1, 2t+8, 2t+9: one
//                         8-byte load a key (4), which lies in one scale block; the low nibbles are MMA row g,
//                         the high ones row g + 8
// Codes become f16 by the e2m1 conversion, times their block scale: exact (2 + 4 significant bits).  P^T moves
// from the accumulator's layout to the operand's by one 8 x 8 transpose in registers.  Queries (bf16) are scaled by
// a power of two per row so that the largest magnitude lies in [2^14, 2^15) and held in f16: exact for every
// element within 2^28 of the row's largest.  P is f16 (half a step 2^-11) times 2^6, which keeps the weights of a long
// context behind one dominating key out of f16's subnormals down to 2^-20; statistics and O are fp32.
//
// What bounds it: the chain of a warp's step (copies, conversion, MMA, maximum, exponentials, MMA), which four warps a
// scheduler cover in part; no unit is at its limit.  64 requests x 4096 keys, 8 heads x 128: 0.59 instructions issued per
// cycle and scheduler, ALU 50 % and DRAM 44 % busy, 718 warp instructions per 32 keys of a head; for each one issued, 1.1
// warps wait out a fixed latency, 0.9 for a math pipe and 0.9 for memory.  64 requests x 8192 keys (604 MB): 146 us = 4.1 TB/s
// of the measured 6.55, with DRAM traffic equal to the bytes needed.  On the way: codes straight from global memory into
// registers 330 us (one ragged batch), the ring 263 us, the heads of a cache row fetched together 171 us.
//
// The ranges follow from the sum of all lengths, so where a request is cut, whether heads are taken together, and with
// that the order of its sums and its last bits, depend on the rest of its batch.  The same call gives the same bits.
#include "kv4_common.cuh"

namespace msl {

constexpr float kKvTau = 8.0f;             // the running maximum may lag by 2^8,
constexpr float kKvShift = 6.0f;           // so P 2^6 stays below 2^15, within f16

// Tiles of a request, all its KV heads, when a CTA takes `heads` of them at once.
__device__ __forceinline__ int64_t kv4_tiles(const Kv4Args& p, const Kv4Req& r, int heads, int tile_shift) {
  if (r.len <= 0) return 0;
  const Kv4Span s = kv4_span(p, r, tile_shift);
  return static_cast<int64_t>(s.last - s.first) * (p.hkv / heads);
}
// A CTA takes p.heads KV heads of 32 W / p.heads keys at once where every worker has at least kKvLong tiles (below), and
// one head of 32 W keys otherwise: the heads of a cache row lie side by side, so taking them together fetches whole rows
// (a 64-byte piece of one costs as much DRAM time as 128 bytes), but it also leaves p.heads times as many partial
// results per item to join, which a short step cannot hide.  When the choice was made, 64 requests x 8192 keys, 8 heads:
// 291 -> 174 us with all heads at once (146 since); 1 x 4096: 18 -> 40 us.
constexpr int kKvLong = 8;

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t o;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(o) : "r"(v));
  return o;
}

// A warp's ring of 32-key stages in shared memory: K codes, V codes, their scales, one word with a bit per key that has
// a cache row.  Filled by cp.async straight from the pages; kStages - 1 of them are in flight while one is computed.
// A lane's V words (one per key, keys 2 apart) would fall into the same banks: within each 128 bytes the 16-byte units
// are permuted by the row.
template <int D>
struct Kv4Ring {
  static constexpr int kRowBytes = D / 2, kChunks = D / 32, kSfBytes = D / 16;
  static constexpr int kV = 32 * kRowBytes, kKs = 2 * kV, kVs = kKs + 32 * kSfBytes, kHeld = kVs + 32 * kSfBytes;
  static constexpr int kStage = kHeld + 16;
  static constexpr int kStages = 3;
  static constexpr int kWarp = kStages * kStage;
};
template <int D>
__device__ __forceinline__ uint32_t kv4_v_offset(int row, int byte) {   // byte < D / 2 of a V row
  constexpr int kPer = D == 128 ? 2 : 4;                    // rows per 128 bytes
  constexpr int kShift = D == 128 ? 1 : 2;
  const int unit = (row & (kPer - 1)) * Kv4Ring<D>::kChunks + (byte >> 4);
  return (row >> kShift) * 128 + ((unit ^ (2 * ((row >> kShift) & (D == 128 ? 3 : 1)))) << 4) + (byte & 15);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {   // fewer bytes: zeros behind them
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Where a lane's copies start: the KV head's bytes of cache row 0, and the lane's 16-byte unit of them.
struct Kv4Source {
  const uint8_t *k, *v, *ks, *vs;
  int pitch, sf_pitch;                      // bytes of a cache row (all heads)
};
template <int D>
__device__ __forceinline__ Kv4Source kv4_source(const Kv4Args& p, int kvh, int lane) {
  using S = Kv4Ring<D>;
  const int at = kvh * S::kRowBytes + (lane % S::kChunks) * 16;
  return {p.k + at, p.v + at, p.ks + kvh * S::kSfBytes, p.vs + kvh * S::kSfBytes,
          p.hkv * S::kRowBytes, p.hkv * S::kSfBytes};
}

// Start copying the 32 keys whose cache rows the lanes hold (-1: zeros).
template <int D>
__device__ __forceinline__ void kv4_issue(const Kv4Source& src, uint8_t* stage, int row, int lane) {
  using S = Kv4Ring<D>;
  const uint32_t base = smem_u32(stage);
  const uint32_t mask = __ballot_sync(0xffffffffu, row >= 0);
  constexpr int kRows = 32 / S::kChunks;                    // rows a round covers
  const int c = lane % S::kChunks;
  if (mask == 0xffffffffu) {
#pragma unroll
    for (int i = 0; i < S::kChunks; ++i) {
      const int r = kRows * i + lane / S::kChunks;
      const int64_t from = __shfl_sync(0xffffffffu, row, r);
      cp_async16(base + r * S::kRowBytes + c * 16, src.k + from * src.pitch, 16);
      cp_async16(base + S::kV + kv4_v_offset<D>(r, c * 16), src.v + from * src.pitch, 16);
    }
    const int64_t from = row;
    cp_async_small<S::kSfBytes>(base + S::kKs + lane * S::kSfBytes, src.ks + from * src.sf_pitch, S::kSfBytes);
    cp_async_small<S::kSfBytes>(base + S::kVs + lane * S::kSfBytes, src.vs + from * src.sf_pitch, S::kSfBytes);
  } else {
#pragma unroll
    for (int i = 0; i < S::kChunks; ++i) {
      const int r = kRows * i + lane / S::kChunks;
      const int got = __shfl_sync(0xffffffffu, row, r);
      const int64_t from = max(got, 0);
      const int bytes = got >= 0 ? 16 : 0;
      cp_async16(base + r * S::kRowBytes + c * 16, src.k + from * src.pitch, bytes);
      cp_async16(base + S::kV + kv4_v_offset<D>(r, c * 16), src.v + from * src.pitch, bytes);
    }
    const int64_t from = max(row, 0);
    const int bytes = row >= 0 ? S::kSfBytes : 0;
    cp_async_small<S::kSfBytes>(base + S::kKs + lane * S::kSfBytes, src.ks + from * src.sf_pitch, bytes);
    cp_async_small<S::kSfBytes>(base + S::kVs + lane * S::kSfBytes, src.vs + from * src.sf_pitch, bytes);
  }
  if (lane == 0) *reinterpret_cast<uint32_t*>(stage + S::kHeld) = mask;
}

// Shared-memory layout of a warp's O [R][D]: channel d of the lane group D/8 at pitch D/8 + 2, so that the float2
// stores of a warp (8 groups x 4 row pairs) fall into different banks.
template <int D>
struct Kv4Merge {
  static constexpr int kGroup = D / 8 + 2;
  static constexpr int kRow = 8 * kGroup + 8;
};

// W warps a CTA.  p.heads of them (a power of two) take one KV head each, the W / p.heads groups of them 32 keys each:
// a cache row's heads lie side by side, and fetching them together is what keeps DRAM traffic at the bytes needed.
template <int D, int NB>
struct Kv4Shape {
  static constexpr bool kSlim = D == 64 || NB == 1;        // fits 128 registers
  static constexpr int kWarps = kSlim ? 8 : 4;
  static constexpr int kCtas = kSlim ? 2 : 3;              // per SM
};

template <int D, int NB, int W>
__global__ void __launch_bounds__(32 * W, Kv4Shape<D, NB>::kCtas)
attention_kv4_kernel(Kv4Args p) {
  constexpr int R = 8 * NB;
  constexpr int KS = D / 16;               // MMA steps of Q K^T, and 16-row tiles of O^T
  using M = Kv4Merge<D>;
  using S = Kv4Ring<D>;
  static_assert(R * M::kRow * 4 <= S::kWarp, "a warp's O takes the place of its ring");
  extern __shared__ __align__(128) uint8_t kv4_smem[];
  const auto sm_o = [&](int w, int row) { return reinterpret_cast<float*>(kv4_smem + w * S::kWarp) + row * M::kRow; };
  __shared__ float sm_m[W][R], sm_l[W][R];
  __shared__ int64_t scratch[W];
  __shared__ int sm_b;
  __shared__ int64_t sm_at;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = p.hq / p.hkv;
  uint8_t* ring = kv4_smem + warp * S::kWarp;
  pdl_launch_dependents();

  // ---- this worker's range of tiles
  const int per = (p.batch + blockDim.x - 1) / blockDim.x;
  const int b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
  constexpr int kWide = W == 8 ? 8 : 7;                     // log2 of a one-head tile's keys, 32 W
  int64_t mine_all = 0, mine = 0;                           // tiles with p.heads heads a CTA, and with one
  for (int b = b0; b < b1; ++b) {
    const Kv4Req r = kv4_request(p, b);
    if (r.over && blockIdx.x == 0) report_error(p.status, MSL_ERR_CAPACITY);
    mine_all += kv4_tiles(p, r, p.heads, p.tile_shift);
    mine += kv4_tiles(p, r, 1, kWide);
  }
  const bool together = block_sum_i64<W>(mine_all, scratch) >= static_cast<int64_t>(kKvLong) * p.workers;
  const int heads = together ? p.heads : 1, tile_shift = together ? p.tile_shift : kWide;
  if (together) mine = mine_all;
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t a = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += a;
  }
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < W; ++w) {
    if (w < warp) inc += scratch[w];
    total += scratch[w];
  }
  const int64_t workers = min(static_cast<int64_t>(p.workers), total);   // no empty range in between
  if (blockIdx.x >= workers) return;                        // uniform
  int64_t at = total * blockIdx.x / workers;
  const int64_t end = total * (blockIdx.x + 1) / workers;
  if (inc - mine <= at && at < inc) {                       // one thread: walk its few requests
    int64_t base = inc - mine;
    int b = b0;
    for (; b < b1 - 1; ++b) {
      const int64_t n = kv4_tiles(p, kv4_request(p, b), heads, tile_shift);
      if (at < base + n) break;
      base += n;
    }
    sm_b = b;
    sm_at = base;
  }
  __syncthreads();
  int b = sm_b;
  int64_t skip = at - sm_at;                                // tiles of request b before this range
  const float scale_log2 = p.softmax_scale * (*p.k_scale) * 1.4426950408889634f;

  const int groups = p.hkv / heads, my_head = warp & (heads - 1), n_sub = W / heads;

  for (; at < end && b < p.batch; ++b) {
    const Kv4Req r = kv4_request(p, b);
    if (r.len <= 0) continue;
    const int* table = p.page_table + static_cast<int64_t>(b) * p.max_pages;
    const Kv4Span span = kv4_span(p, r, tile_shift);
    const int n_span = span.last - span.first;
    for (int group = static_cast<int>(skip / n_span); group < groups && at < end; ++group) {
      const int kvh = group * heads + my_head;
      const int off = static_cast<int>(skip % n_span);
      skip = 0;
      const int n = static_cast<int>(min(end - at, static_cast<int64_t>(n_span - off)));
      // ---- rows of the block: row = token * G + head in group
      const int rows = min(R, r.len * G);                 // (the launch takes care that R is enough)
      const int last_tok = r.len - 1;
      const int hi = r.seq + last_tok + 1;                // keys [lo, hi) are visible to some row
      const int lo = p.window ? max(0, r.seq - p.window + 1) : 0;
      if (tid == 0 && hi > static_cast<int64_t>(p.max_pages) * p.page_size) report_error(p.status, MSL_ERR_CAPACITY);
      const int all_lo = p.window ? max(0, r.seq + last_tok - p.window + 1) : 0;   // keys [all_lo, all_hi) to all
      const int all_hi = r.seq + 1;
      uint32_t qf[NB][KS][2];
      float qs[NB][2];                                    // log2 scale of columns 2t, 2t + 1
      int qpos[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int row = nb * 8 + g;
        uint32_t raw[KS * 2];
#pragma unroll
        for (int w = 0; w < KS * 2; ++w) raw[w] = 0;
        if (row < rows) {
          const int tok = row / G, head = kvh * G + row % G;
          const uint4* src = reinterpret_cast<const uint4*>(p.q + (static_cast<int64_t>(r.begin) + tok) * p.ld_q +
                                                            head * D + t * (D / 4));
#pragma unroll
          for (int w = 0; w < KS / 2; ++w) {
            const uint4 x = src[w];
            raw[4 * w] = x.x; raw[4 * w + 1] = x.y; raw[4 * w + 2] = x.z; raw[4 * w + 3] = x.w;
          }
        }
        uint32_t mx = 0;                                  // largest magnitude as bits (NaN and infinity on top)
#pragma unroll
        for (int w = 0; w < KS * 2; ++w) mx = max(mx, max(raw[w] & 0x7fffu, (raw[w] >> 16) & 0x7fffu));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // 2^(141 - e) takes the exponent e to 141 = 127 + 14; its inverse goes into the row's score scale
        const int e = min(max(static_cast<int>(mx >> 7), 16), 254);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 141 - e) << 23);
        const float down = kv4_row_scale(scale_log2, up);
#pragma unroll
        for (int w = 0; w < KS * 2; ++w)
          qf[nb][w / 2][w & 1] = h2_bits(__floats2half2_rn(bf16_bits_to_f32(raw[w] & 0xffffu) * up,
                                                           bf16_bits_to_f32(raw[w] >> 16) * up));
        qs[nb][0] = __shfl_sync(0xffffffffu, down, 8 * t);         // lane (g = 2t, 0) holds row 2t
        qs[nb][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
#pragma unroll
        for (int c = 0; c < 2; ++c) qpos[nb][c] = r.seq + (nb * 8 + 2 * t + c) / G;
      }
      float o[NB][KS][4], m[NB][2], l[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int c = 0; c < 2; ++c) { m[nb][c] = -INFINITY; l[nb][c] = 0.f; }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[nb][k][c] = 0.f;
      }
      // ---- the keys, 32 a step
      const int tile = 1 << tile_shift;
      const int key_first = (span.first + off) * tile + (warp / heads) * 32;
      const auto page_of = [&](int j) {
        return j < n ? kv4_page(p, table, key_first + j * tile + lane, lo, hi) : Kv4Page{INT_MIN, 0};
      };
      const Kv4Source source = kv4_source<D>(p, kvh, lane);
      Kv4Page ahead[S::kStages];
#pragma unroll
      for (int j = 0; j < S::kStages; ++j) ahead[j] = page_of(j);
#pragma unroll
      for (int j = 0; j < S::kStages - 1; ++j) {
        if (j < n) kv4_issue<D>(source, ring + j * S::kStage, kv4_row_of(p, ahead[j]), lane);
        cp_async_commit();
      }
      Kv4Page page_next = ahead[S::kStages - 1];          // of step j + kStages - 1
      int slot = 0;
      for (int j = 0; j < n; ++j) {
        const int key0 = key_first + j * tile;
        uint8_t* stage = ring + slot * S::kStage;
        cp_async_wait<S::kStages - 2>();
        __syncwarp();                                     // every lane's copies are in, and the last slot is free
        if (j + S::kStages - 1 < n)
          kv4_issue<D>(source, ring + (slot == 0 ? S::kStages - 1 : slot - 1) * S::kStage, kv4_row_of(p, page_next), lane);
        cp_async_commit();
        page_next = page_of(j + S::kStages);
        slot = slot + 1 == S::kStages ? 0 : slot + 1;
        const uint32_t held = *reinterpret_cast<const uint32_t*>(stage + S::kHeld);
        const bool partial = held != 0xffffffffu || key0 < all_lo || key0 + 32 > all_hi;
        float s[2][NB][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[h][nb][c] = 0.f;
          uint32_t k[2][D / 32];
          __half2 sc[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int row = 16 * h + 8 * x + g;
            if constexpr (D == 128) {
              const uint4 v = *reinterpret_cast<const uint4*>(stage + row * 64 + t * 16);
              k[x][0] = v.x; k[x][1] = v.y; k[x][2] = v.z; k[x][3] = v.w;
              sc[x] = scales_h2(*reinterpret_cast<const uint16_t*>(stage + S::kKs + row * 8 + t * 2));
            } else {
              const uint2 v = *reinterpret_cast<const uint2*>(stage + row * 32 + t * 8);
              k[x][0] = v.x; k[x][1] = v.y;
              sc[x] = scales_h2(stage[S::kKs + row * 4 + t]);
            }
          }
#pragma unroll
          for (int w = 0; w < D / 32; ++w) {              // one word = two MMA steps
            __half2 a[4], c[4];
            e2m1x8(k[0][w], a);
            e2m1x8(k[1][w], c);
            const bool second = D == 128 && w >= 2;       // which of the lane's two scale blocks
            const __half2 s0 = second ? __high2half2(sc[0]) : __low2half2(sc[0]);
            const __half2 s1 = second ? __high2half2(sc[1]) : __low2half2(sc[1]);
#pragma unroll
            for (int x = 0; x < 4; ++x) { a[x] = __hmul2(a[x], s0); c[x] = __hmul2(c[x], s1); }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              mma_16816(s[h][nb], h2_bits(a[0]), h2_bits(c[0]), h2_bits(a[1]), h2_bits(c[1]), qf[nb][2 * w][0],
                        qf[nb][2 * w][1]);
              mma_16816(s[h][nb], h2_bits(a[2]), h2_bits(c[2]), h2_bits(a[3]), h2_bits(c[3]), qf[nb][2 * w + 1][0],
                        qf[nb][2 * w + 1][1]);
            }
          }
        }
        // ---- mask where some row does not see a key
        if (partial) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int kk = 16 * h + g + 8 * x;
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  const int key = key0 + kk;
                  const bool seen = ((held >> kk) & 1u) && key <= qpos[nb][c] && (!p.window || key > qpos[nb][c] - p.window);
                  if (!seen) s[h][nb][2 * x + c] = -INFINITY;
                }
            }
        }
        // ---- running maximum: it moves when a row of the warp exceeds it by more than 2^tau
        float top[NB][2];
        bool move = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            // in log2 units (the scale is positive)
            const float x = fmaxf(fmaxf(s[0][nb][c], s[0][nb][2 + c]), fmaxf(s[1][nb][c], s[1][nb][2 + c])) * qs[nb][c];
            top[nb][c] = x;
            move |= x > m[nb][c] + kKvTau || (m[nb][c] == -INFINITY && x > -INFINITY);
          }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x = top[nb][c];
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
              // each column (query row) decides for itself: its bits do not depend on its neighbours
              const float new_m = (x > m[nb][c] + kKvTau || m[nb][c] == -INFINITY) ? x : m[nb][c];
              const float corr = kv_ex2(m[nb][c] - (new_m == -INFINITY ? 0.f : new_m));
              m[nb][c] = new_m;
              l[nb][c] *= corr;
#pragma unroll
              for (int k = 0; k < KS; ++k) { o[nb][k][c] *= corr; o[nb][k][2 + c] *= corr; }
            }
        }
        uint32_t pf[2][NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          // l and O carry P's 2^shift alike, here and in the partial results
          const float n0 = m[nb][0] == -INFINITY ? 0.f : m[nb][0] - kKvShift;
          const float n1 = m[nb][1] == -INFINITY ? 0.f : m[nb][1] - kKvShift;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float e0 = kv_ex2(fmaf(s[h][nb][2 * x], qs[nb][0], -n0));
              const float e1 = kv_ex2(fmaf(s[h][nb][2 * x + 1], qs[nb][1], -n1));
              l[nb][0] += e0;
              l[nb][1] += e1;
              pf[h][nb][x] = transpose8x8(h2_bits(__floats2half2_rn(e0, e1)));
            }
        }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t v[4][D / 64];
          uint32_t vs[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int row = 16 * h + 2 * t + (x & 1) + 8 * (x >> 1);
            const uint8_t* src = stage + S::kV + kv4_v_offset<D>(row, g * (D / 16));
            if constexpr (D == 128) {
              const uint2 u = *reinterpret_cast<const uint2*>(src);
              v[x][0] = u.x; v[x][1] = u.y;
              vs[x] = stage[S::kVs + row * 8 + g];
            } else {
              v[x][0] = *reinterpret_cast<const uint32_t*>(src);
              vs[x] = stage[S::kVs + row * 4 + g / 2];
            }
          }
          const __half2 s01 = scales_h2(vs[0] | (vs[1] << 8));
          const __half2 s23 = scales_h2(vs[2] | (vs[3] << 8));
#pragma unroll
          for (int w = 0; w < D / 64; ++w) {              // one word a key = four 16-row tiles
            // pairs along the keys: low nibbles (even channels, MMA rows g) and high ones (odd, g + 8)
            const uint32_t lo01 = (v[0][w] & 0x0f0f0f0fu) | ((v[1][w] << 4) & 0xf0f0f0f0u);
            const uint32_t hi01 = ((v[0][w] >> 4) & 0x0f0f0f0fu) | (v[1][w] & 0xf0f0f0f0u);
            const uint32_t lo23 = (v[2][w] & 0x0f0f0f0fu) | ((v[3][w] << 4) & 0xf0f0f0f0u);
            const uint32_t hi23 = ((v[2][w] >> 4) & 0x0f0f0f0fu) | (v[3][w] & 0xf0f0f0f0u);
            __half2 a0[4], a1[4], a2[4], a3[4];
            e2m1x8(lo01, a0);
            e2m1x8(hi01, a1);
            e2m1x8(lo23, a2);
            e2m1x8(hi23, a3);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint32_t u0 = h2_bits(__hmul2(a0[x], s01)), u1 = h2_bits(__hmul2(a1[x], s01));
              const uint32_t u2 = h2_bits(__hmul2(a2[x], s23)), u3 = h2_bits(__hmul2(a3[x], s23));
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
                mma_16816(o[nb][4 * w + x], u0, u1, u2, u3, pf[h][nb][0], pf[h][nb][1]);
            }
          }
        }
      }
      __syncwarp();                                       // the ring is read; O takes its place
      // ---- join the warps of a head
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = l[nb][c];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
          const int row = nb * 8 + 2 * t + c;
          if (g == 0) { sm_m[warp][row] = m[nb][c]; sm_l[warp][row] = x; }
#pragma unroll
          for (int k = 0; k < KS; ++k)
            *reinterpret_cast<float2*>(sm_o(warp, row) + g * M::kGroup + 2 * k) =
                make_float2(o[nb][k][c], o[nb][k][2 + c]);
        }
      }
      __syncthreads();
      const bool whole = n == n_span;
      // a worker has at most two partial results: the rest of an item that an earlier worker began (slot 0) and
      // the beginning of one that a later worker ends (slot 1)
      float* part = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + (off == 0 ? 1 : 0)) * p.heads * R * (D + 2);
      for (int job = warp; job < heads * rows; job += W) {
        const int h = job & (heads - 1), row = job / heads;
        float mx = -INFINITY;
        for (int x = 0; x < n_sub; ++x) mx = fmaxf(mx, sm_m[x * heads + h][row]);
        float acc[D / 32], sum = 0.f;
#pragma unroll
        for (int x = 0; x < D / 32; ++x) acc[x] = 0.f;
        for (int y = 0; y < n_sub; ++y) {
          const int w = y * heads + h;
          const float c = kv_ex2(sm_m[w][row] - (mx == -INFINITY ? 0.f : mx));
          sum += sm_l[w][row] * c;
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            const int d = lane * (D / 32) + x;
            acc[x] += sm_o(w, row)[(d / (D / 8)) * M::kGroup + d % (D / 8)] * c;
          }
        }
        if (whole) {
          const int tok = row / G, head = (group * heads + h) * G + row % G;
          kv4_write_row<D>(p, acc, sum, static_cast<int64_t>(r.begin) + tok, head, lane);
        } else {
          float* dst = part + (h * R + row) * (D + 2);
          if (lane == 0) { dst[0] = mx; dst[1] = sum; }
#pragma unroll
          for (int x = 0; x < D / 32; x += 2)
            *reinterpret_cast<float2*>(dst + 2 + lane * (D / 32) + x) = make_float2(acc[x], acc[x + 1]);
        }
      }
      __syncthreads();
      at += n;
    }
    // `skip` is below request b's tiles when the range starts in it, and zero from then on
  }
}

// Joins the partial results of work items that several workers share; items that one worker covered are final already.
// One CTA per (KV head, request, and, where there are few of them, row).  Its warps share out the rows
// and, with warps to spare, the partial results of a row.
constexpr int kMergeWarps = 8;
template <int D, int NB, int W>
__global__ void __launch_bounds__(32 * kMergeWarps)
kv4_merge_kernel(Kv4Args p) {
  constexpr int R = 8 * NB, PER = D / 32;
  __shared__ int64_t scratch[kMergeWarps];
  __shared__ float sm_o[kMergeWarps][D], sm_l[kMergeWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.hq / p.hkv;
  const int b = blockIdx.y, kvh = blockIdx.x;
  constexpr int kWide = W == 8 ? 8 : 7;
  int64_t before = 0, all = 0, before_all = 0, all_all = 0;
  for (int x = tid; x < p.batch; x += blockDim.x) {
    const Kv4Req r = kv4_request(p, x);
    const int64_t n = kv4_tiles(p, r, 1, kWide), m = kv4_tiles(p, r, p.heads, p.tile_shift);
    all += n;
    all_all += m;
    if (x < b) { before += n; before_all += m; }
  }
  all_all = block_sum_i64<kMergeWarps>(all_all, scratch);
  const bool together = all_all >= static_cast<int64_t>(kKvLong) * p.workers;   // the attention kernel's choice
  const int heads = together ? p.heads : 1, tile_shift = together ? p.tile_shift : kWide;
  all = together ? all_all : block_sum_i64<kMergeWarps>(all, scratch);
  before = block_sum_i64<kMergeWarps>(together ? before_all : before, scratch);
  const Kv4Req r = kv4_request(p, b);
  pdl_wait();                               // in every block: this grid ends only after the one before it
  if (r.len <= 0) return;
  const Kv4Span span = kv4_span(p, r, tile_shift);
  const int n_span = span.last - span.first;
  const int64_t t0 = before + static_cast<int64_t>(kvh / heads) * n_span, t1 = t0 + n_span;   // this item's tiles
  // tile t belongs to the largest w with floor(all * w / workers) <= t
  const int64_t workers = min(static_cast<int64_t>(p.workers), all);
  const int w0 = static_cast<int>(((t0 + 1) * workers - 1) / all), w1 = static_cast<int>((t1 * workers - 1) / all);
  if (w0 == w1) return;
  const int rows = min(R, r.len * G);
  // rows_par rows at a time, `share` warps a row
  const int here = gridDim.z == 1 ? rows : 1;
  const int rows_par = here > 4 ? 8 : here > 2 ? 4 : here, share = kMergeWarps / rows_par;
  const int mine = warp % share;
  for (int row0 = blockIdx.z; row0 < rows; row0 += gridDim.z * rows_par) {
    const int row = row0 + warp / share;
    const bool live = row < rows;
    const auto at = [&](int w) {
      return p.part + ((static_cast<int64_t>(w * 2 + (w == w0 ? 1 : 0)) * p.heads + (kvh & (heads - 1))) * R + row) * (D + 2);
    };
    float sum = 0.f, acc[PER];
#pragma unroll
    for (int x = 0; x < PER; ++x) acc[x] = 0.f;
    if (live) {
      float mx = -INFINITY;
      for (int w = w0 + lane; w <= w1; w += 32) mx = fmaxf(mx, at(w)[0]);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll 8
      for (int w = w0 + mine; w <= w1; w += share) {
        const float* src = at(w);
        const float c = kv_ex2(src[0] - ref);
        sum += src[1] * c;
#pragma unroll
        for (int x = 0; x < PER; x += 2) {
          const float2 v = *reinterpret_cast<const float2*>(src + 2 + lane * PER + x);
          acc[x] += v.x * c;
          acc[x + 1] += v.y * c;
        }
      }
    }
    if (share > 1) {                                        // uniform
#pragma unroll
      for (int x = 0; x < PER; ++x) sm_o[warp][lane * PER + x] = acc[x];
      if (lane == 0) sm_l[warp] = sum;
      __syncthreads();
      if (mine == 0) {
        for (int y = 1; y < share; ++y) {                   // all relative to the same maximum
          sum += sm_l[warp + y];
#pragma unroll
          for (int x = 0; x < PER; ++x) acc[x] += sm_o[warp + y][lane * PER + x];
        }
      }
      __syncthreads();
    }
    if (live && mine == 0) {
      const int tok = row / G, head = kvh * G + row % G;
      kv4_write_row<D>(p, acc, sum, static_cast<int64_t>(r.begin) + tok, head, lane);
    }
  }
}

// KV heads a CTA of `warps` warps takes at once: the largest power of two that divides them.
static int kv4_heads(int hkv, int warps) {
  int h = 1;
  while (h < warps && hkv % (2 * h) == 0) h *= 2;
  return h;
}

template <int D, int NB>
static int64_t kv4_few_workspace(int hkv) {
  using Shape = Kv4Shape<D, NB>;
  return static_cast<int64_t>(sm_count()) * Shape::kCtas * 2 * kv4_heads(hkv, Shape::kWarps) * 8 * NB * (D + 2) * 4;
}

template <int D, int NB>
static int launch_kv4(Kv4Args a, cudaStream_t st) {
  using Shape = Kv4Shape<D, NB>;
  constexpr int R = 8 * NB, W = Shape::kWarps;
  constexpr int smem = W * Kv4Ring<D>::kWarp;
  static SmemConfig config;
  if (int rc = config.ensure(attention_kv4_kernel<D, NB, W>, smem)) return rc;
  a.workers = sm_count() * Shape::kCtas;
  a.heads = kv4_heads(a.hkv, W);
  a.tile_shift = 5;
  while ((1 << a.tile_shift) < 32 * (W / a.heads)) ++a.tile_shift;
  attention_kv4_kernel<D, NB, W><<<a.workers, 32 * W, smem, st>>>(a);
  if (cudaGetLastError() != cudaSuccess) return MSL_ERR_CUDA;
  // The merge forms its schedule while the attention runs and waits for it on the device (programmatic launch).
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  // few items: a CTA a row, whose warps share its many partial results
  const int64_t items = static_cast<int64_t>(a.hkv) * a.batch;
  cfg.gridDim = dim3(a.hkv, a.batch, items <= sm_count() / 2 ? R : 1);
  cfg.blockDim = dim3(32 * kMergeWarps);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_merge_kernel<D, NB, W>, a) == cudaSuccess ? MSL_OK : MSL_ERR_CUDA;
}

// Query rows a CTA holds: one MMA column block of 8 where the group's rows fit, else two.
static int kv4_row_blocks(int64_t rows) { return rows <= 8 ? 1 : 2; }

// Up to this many query rows per KV head, the two column blocks that fit its registers, the mma.sync kernel above is
// used; beyond it the tcgen05 kernel, whose 128 rows cost the same however few are used.  8 heads x 128, this kernel
// against tcgen05: 16 rows, 16 requests of 4096 keys 57 us against 73, 64 of 1024 51 against 123, 1 of 30000 32 against
// 49.  Beyond 16 rows this kernel would stream the keys again for every 16: 16 requests of 4096 keys, launch included,
// 32 rows 101 against 94, 64 rows 141 against 94 (2 requests, 32 rows: 54 against 56).
constexpr int kKvFewRows = 16;

struct Kv4Plan {
  bool few;
  int splits, alternate;
  int64_t bytes;
};
static Kv4Plan kv4_plan(int batch, int max_q_len, int tokens, int hq, int hkv, int head_dim, int max_pages, int page_size,
                        int window) {
  Kv4Plan plan{true, 1, 0, 0};
  const int64_t rows = static_cast<int64_t>(max_q_len) * (hq / hkv);
  plan.few = rows <= kKvFewRows;
  if (plan.few) {
    const bool one = kv4_row_blocks(rows) == 1;
    plan.bytes = head_dim == 128 ? (one ? kv4_few_workspace<128, 1>(hkv) : kv4_few_workspace<128, 2>(hkv))
                                 : (one ? kv4_few_workspace<64, 1>(hkv) : kv4_few_workspace<64, 2>(hkv));
  } else {
    plan.splits = msl_attention_split_plan(batch, max_q_len, hq, hkv, max_pages, page_size, window);
    plan.alternate = rows <= 128;
    if (plan.alternate) plan.splits = 1;
    plan.bytes = plan.alternate ? kv4_tc_shared_workspace(static_cast<int>(rows), tokens, hq, head_dim)
                                : kv4_tc_workspace(plan.splits, tokens, hq, head_dim);
  }
  return plan;
}

static bool misaligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

}  // namespace msl

using namespace msl;

extern "C" int64_t msl_attention_kv4_workspace(int batch, int max_q_len, int tokens, int hq, int hkv, int head_dim,
                                               int max_pages, int page_size, int window) {
  if (batch <= 0 || max_q_len <= 0 || tokens <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || hq / hkv > 128 ||
      max_pages <= 0 || page_size <= 0 || window < 0)
    return 0;
  return kv4_plan(batch, max_q_len, tokens, hq, hkv, head_dim, max_pages, page_size, window).bytes;
}

extern "C" int msl_attention_kv4(const void* q, int64_t ld_q, const void* k_cache, const void* k_sf,
                                 const void* v_cache, const void* v_sf, const int* page_table, int max_pages,
                                 const int* seq_lens, const int* cu_seqlens_q, const float* k_scale,
                                 const float* v_scale, float softmax_scale, int batch, int max_q_len, int tokens,
                                 int hq, int hkv, int head_dim, int page_size, int window, int64_t cache_rows,
                                 void* out, int64_t ld_out, const void* gate, int64_t ld_gate, void* workspace,
                                 int64_t workspace_bytes, int* status, void* stream) {
  if (batch <= 0 || max_q_len <= 0 || tokens < 0 || hq <= 0 || hkv <= 0 || hq % hkv || page_size <= 0 || window < 0 ||
      max_pages <= 0 || cache_rows <= 0 || cache_rows > 0x7fffffff || !(softmax_scale > 0.f))
    return MSL_ERR_ARG;
  if (head_dim != 64 && head_dim != 128) return MSL_ERR_UNSUPPORTED;
  const int G = hq / hkv;
  if (G > 128 || batch > 65535) return MSL_ERR_UNSUPPORTED;
  if (tokens == 0) return MSL_OK;
  if (!q || !k_cache || !k_sf || !v_cache || !v_sf || !page_table || !seq_lens || !cu_seqlens_q || !k_scale ||
      !v_scale || !out)
    return MSL_ERR_ARG;
  const Kv4Plan plan = kv4_plan(batch, max_q_len, tokens, hq, hkv, head_dim, max_pages, page_size, window);
  if (plan.bytes > 0 && !workspace) return MSL_ERR_ARG;
  const int64_t cols = static_cast<int64_t>(hq) * head_dim;
  if (ld_q < cols || ld_out < cols || (gate && ld_gate < cols)) return MSL_ERR_ARG;
  if (misaligned(q, 16) || (ld_q & 7) || misaligned(k_cache, 16) || misaligned(v_cache, 16) || misaligned(k_sf, 8) ||
      misaligned(v_sf, 8) || misaligned(out, 16) || (ld_out & 7) || (gate && (misaligned(gate, 16) || (ld_gate & 7))) ||
      misaligned(workspace, 16))
    return MSL_ERR_ALIGN;
  if (workspace_bytes < plan.bytes) return MSL_ERR_CAPACITY;
  const auto u8 = [](const void* x) { return static_cast<const uint8_t*>(x); };
  int page_shift = -1;
  if ((page_size & (page_size - 1)) == 0)
    for (page_shift = 0; (1 << page_shift) < page_size; ++page_shift) {}
  const Kv4Args a{static_cast<const __nv_bfloat16*>(q), ld_q, u8(k_cache), u8(k_sf), u8(v_cache), u8(v_sf),
                  page_table, max_pages, seq_lens, cu_seqlens_q, k_scale, v_scale, softmax_scale, batch, max_q_len,
                  tokens, hq, hkv, page_size, window, cache_rows, static_cast<__nv_bfloat16*>(out), ld_out,
                  static_cast<const __nv_bfloat16*>(gate), ld_gate, static_cast<float*>(workspace),
                  0, 0, 0, plan.splits, plan.alternate, page_shift, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!plan.few) return launch_kv4_tc(a, head_dim, st);
  if (kv4_row_blocks(static_cast<int64_t>(max_q_len) * G) == 1)
    return head_dim == 128 ? launch_kv4<128, 1>(a, st) : launch_kv4<64, 1>(a, st);
  return head_dim == 128 ? launch_kv4<128, 2>(a, st) : launch_kv4<64, 2>(a, st);
}
