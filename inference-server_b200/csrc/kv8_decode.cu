// Paged decode attention over the 8-bit page cache (kv8.cuh) for sm_100a: the counterpart of paged_attn.cu, which reads 16-bit pools,
// and so of the same steps of the reference (src/inference_server/kv_cache/hf_format.py:21-45 and
// src/inference_server/backends/torch_backend.py:305-322).
//
// Mathematics.  A page and kv head has scales 2^ek (keys) and 2^ev (values).  With scores s_t = scale * log2(e) * 2^ek (q . k_t) of the
// e4m3 numbers k_t, the output is  sum_t 2^(s_t + ev) v_t / sum_t 2^s_t.  A value's scale is taken into its weight's exponent:
// p_t = 2^(s_t + ev - m), where m follows the maximum of s_t + ev, so the largest weight sees the largest product and not the largest
// score.  The denominator is sum_t p_t 2^-ev.  Everything that has a scale in it is an fp32 exponent; e4m3 numbers become f16 exactly, and
// weights are f16, whose 11 bits leave them an eighth of the error of bf16.  Weights are taken so that the largest is between 2^6 and
// 2^14; those below 2^-14 lose bits.  A head's query is multiplied by a power of two that brings its largest number to 2^14 and becomes
// f16: what loses bits is 2^-28 of the largest.  (One power for a kv group would let a head that is 2^30 times larger than its neighbours, or
// not finite, take their bits.)  Sums are fp32.  With |ev| <= 32 the sums p_t 2^-ev stay below 2^14 * 2^32 * tokens.
//
// Bound by memory: 2 D bytes per token and kv head, one scale byte per 16 D of them.  256 rows of 512 to 4096 tokens, 32 / 4 heads of
// 128, 623 MB: 109 us with the join in a graph of calls, 5.7 TB/s.  The rest is a chain that no call is without - lengths, table, the first pages, the
// last pages' arithmetic, partials, the join -: one row of 777 tokens 6.5 us, 131001 tokens 31.6 us (134 MB).  More than 16 query heads of a kv head
// read its pages again for every 16: 128 rows, 40 heads on one 68 us, 128 on one 162.
//
//   work   The pages of all rows, one row after the other, are cut into equal runs, one per CTA (kv8_ctas_per_sm), wherever
//          that falls in a row: every CTA streams the same number of bytes without a break, whatever the rows' lengths, and there are no
//          waves.  Each CTA finds its run by itself from the lengths (a scan of at most a few KB).  It meets at most one row that began in a
//          run before and one that goes on in the next; those give fp32 partials (o, m, l), all others are written at once.
//          (Splits of 512 tokens, a CTA each, took 113 us and their join 9 for 256 rows of 512 to 4096 tokens; the last wave was a
//          seventh of it.)
//   grid   (runs, groups of kv heads x slices of 16 query heads); block = one consumer warp per kv head + a producer warp.
//   load   The kv heads of a page are adjacent, so a page is one contiguous read of 16 * HKV * D bytes for the keys and one for the values:
//          TMA boxes of 128-byte rows with 128-byte swizzle into a ring of stages of PPS pages.  The producer also brings the pages' scales
//          and, a row ahead, the queries.
//   math   transposed: S^T = K Q^T and O^T = V^T P^T with mma.sync m16n8k16, so that the 16 rows of the tile are tokens, or columns of V,
//          and not the few heads of a group: 16 MMAs per page, half of what the other orientation needs, and 32 accumulators a thread.
//          The order of head_dim in the products is free, so a thread's A operands come from its own 16-byte pieces of K rows without a
//          transposition; those of V^T take bytes of two tokens and one column together with one byte permutation per four bytes of
//          each.  P^T comes from S^T by one movmatrix per 8 x 8 tile.
//   max    lazy, against 2^8: whether any score of the page outgrew its row's reference is one vote; only then are there shuffles.
//   join   A second kernel joins the parts of the rows that lie in more than one run, in their order.  (Joining in here by the warp that is last
//          to finish a row - a fence, a counter, and the parts from L2 in code that runs once - took 5 us for two parts and 10 for 13;
//          the second kernel, launched ahead, takes 1 to 1.5.)
//
// Bank conflicts: a token's row is 128 bytes, its 16-byte pieces XORed with the row number.  A quarter warp reads K pieces of two
// neighbouring g = lane / 4, so their rows must differ in bit 2; it reads V pieces of four tq = lane % 4, whose rows must differ in
// bits 1 and 2.  Row g of a tile is therefore token g ^ 4 (g & 1) of its eight.

#include <algorithm>

#include "host.h"
#include "kv8.cuh"

namespace b200 {

constexpr float kKv8RefSlack = 8.f;    // a score may pass its reference by 2^8 before the reference moves
constexpr float kKv8Lift = 6.f;        // weights are taken times 2^6: at most 2^14 in f16
constexpr int kKv8QueryTop = 14;       // exponent that the largest number of a head's query is brought to

// D(16x8, f32) += A(16x16, f16, row) * B(16x8, f16, col)
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// CTAs that an SM holds: as many as leave each enough of the ring, and of the registers, to keep its share of the memory busy.  More of
// them cut more rows.  us for 128 rows of 512 to 4096 tokens: head_dim 128, 4 kv heads (256 rows) one 126, two 106; 2 kv heads of 8 queries
// two 39.8, three 33.6, four 35.1, of 16 two 47.5, three 42.5; 1 kv head of 8 queries four 20.6, six 19.5, of 16 four 31.5, five 31.0.
// head_dim 64, 4 kv heads of 8 two 36.6, three 34.1, of 16 two 40.1, three 39.0; 2 kv heads of 8 four 22.5, five 21.1, of 16 three 27.7,
// four 24.2; 1 kv head of 8 four 17.0, six 15.5, eight 16.1, of 16 five 21.9, six 19.9.  (With one power of two for the queries of a kv head; one for
// each query head makes those of 16 one or two percent longer.)
constexpr int kv8_ctas_per_sm(int head_dim, int hkv, int nt) {
  if (head_dim == 64) return hkv == 1 ? 6 : hkv == 2 ? (nt == 1 ? 5 : 4) : 3;
  return hkv == 1 ? (nt == 1 ? 6 : 5) : hkv == 2 ? 3 : hkv == 4 ? 2 : 1;
}
// Kv heads of a CTA.  Eight of head_dim 64 leave an SM room for one CTA, which fills it less well than three of four heads: 128 rows of 512 to 4096
// tokens, 64 / 8 heads 64.3 us, 58.3; of head_dim 128, 32 / 8 heads, 96.8 us and two of four 100.8.
constexpr int kv8_heads_per_cta(int head_dim, int hkv) {
  return hkv % 8 == 0 && head_dim == 128 ? 8 : hkv % 4 == 0 ? 4 : hkv % 2 == 0 ? 2 : 1;
}

// Workspace: the status word, per row where its parts are, then the parts: (m, l) and the unnormalised output per (run, which of its two
// open rows, query head).
struct Kv8Workspace {
  int* err;
  int2* rows;  // first part as run * 2 + (is it the run's second open row?), number of parts
  float2* ml;
  float* o;
  size_t bytes;
};
static Kv8Workspace carve_kv8(void* ws, int batch, int runs, int hq, int D) {
  Kv8Workspace w;
  uint8_t* p = static_cast<uint8_t*>(ws);
  w.err = reinterpret_cast<int*>(p);
  size_t off = 256;
  w.rows = reinterpret_cast<int2*>(p + off);
  off += (static_cast<size_t>(batch) * sizeof(int2) + 255) & ~size_t(255);
  w.ml = reinterpret_cast<float2*>(p + off);
  off += (static_cast<size_t>(runs) * 2 * hq * sizeof(float2) + 255) & ~size_t(255);
  w.o = reinterpret_cast<float*>(p + off);
  off += static_cast<size_t>(runs) * 2 * hq * D * sizeof(float);
  w.bytes = off;
  return w;
}

__device__ __forceinline__ int kv8_length(int L, int max_pages) { return min(max(L, 0), max_pages * kKvPage); }
__device__ __forceinline__ int kv8_pages(int L, int max_pages) { return (kv8_length(L, max_pages) + kKvPage - 1) / kKvPage; }
// D: head_dim.  HKV: kv heads = consumer warps.  NT: tiles of 8 query heads per kv head.  PPS: pages per stage.
template <int D, int HKV, int NT, int PPS, int STAGES>
struct Kv8Cfg {
  static constexpr int kThreads = (HKV + 1) * 32;
  static constexpr int kHeadBytes = kKvPage * D;
  static constexpr int kPageBytes = HKV * kHeadBytes;      // keys, or values, of a page's kv heads
  static constexpr int kStageBytes = PPS * 2 * kPageBytes;  // page by page: keys, values
  static constexpr int kQ = STAGES * kStageBytes;
  static constexpr int kScales = kQ + HKV * 8 * NT * D * 2;    // [stages][PPS][keys, values][8] bytes
  static constexpr int kBars = kScales + STAGES * PPS * 2 * 8;
  static constexpr int kSmemBytes = kBars + 16 * (STAGES + 1) + 1024 /* alignment slack */;
};
template <int BYTES> struct Kv8Word { using T = uint32_t; };
template <> struct Kv8Word<1> { using T = uint8_t; };
template <> struct Kv8Word<2> { using T = uint16_t; };
template <> struct Kv8Word<8> { using T = uint2; };

// A warp's walk over the rows of its CTA's run.  The lengths of 32 rows at a time are held by the lanes.
struct Kv8Walk {
  const int* ctx_lens;
  int batch, max_pages, base, held;  // held: length of row base + lane
  int total, per, begin, end;        // all pages; pages of a run; the run
  int at, row, off;                  // the cursor: the row and the page of it that it is at

  // Finds the run: every lane sums the pages of neighbouring rows, then a scan over the lanes.
  __device__ __forceinline__ void start(const int* lens, int rows, int table_pages, int min_run, int lane, int* err) {
    ctx_lens = lens;
    batch = rows;
    max_pages = table_pages;
    const int each = (batch + 31) / 32, lo = min(lane * each, batch), hi = min(lo + each, batch);
    int mine = 0;
#pragma unroll 8
    for (int b = lo; b < hi; ++b) {
      const int L = ctx_lens[b];
      if (L < 0 || L > max_pages * kKvPage) set_error(err, kErrDevBadCtxLen);
      mine += kv8_pages(L, max_pages);
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    total = __shfl_sync(0xffffffffu, upto, 31);  // < 2^31: no more than entries of the table
    per = max(min_run, static_cast<int>((static_cast<unsigned>(total) + gridDim.x - 1) / gridDim.x));
    const long long first = static_cast<long long>(blockIdx.x) * per;
    begin = at = static_cast<int>(min(first, static_cast<long long>(total)));
    end = static_cast<int>(min(first + per, static_cast<long long>(total)));
    const unsigned past = __ballot_sync(0xffffffffu, begin < upto);  // the first of these lanes has the row
    int before = upto - mine, b = lo;
    if (begin >= before && begin < upto)
      for (int pages; before + (pages = kv8_pages(ctx_lens[b], max_pages)) <= begin; ++b) before += pages;
    const int from = past ? __ffs(past) - 1 : 0;
    row = __shfl_sync(0xffffffffu, b, from);
    off = begin - __shfl_sync(0xffffffffu, before, from);
  }
  __device__ __forceinline__ void fetch(int lane) {
    base = row;
    held = row + lane < batch ? ctx_lens[row + lane] : 0;
  }
  // The next part: row, its length L, first page off, number of pages n; false at the end of the run.
  __device__ __forceinline__ bool next(int lane, int& L, int& n) {
    while (at < end && row < batch) {
      if (row - base >= 32) fetch(lane);
      L = kv8_length(__shfl_sync(0xffffffffu, held, row - base), max_pages);
      const int pages = (L + kKvPage - 1) / kKvPage;
      n = min(pages - off, end - at);
      if (n > 0) return true;
      ++row;
      off = 0;
    }
    return false;
  }
  __device__ __forceinline__ void advance(int n) {
    at += n;
    ++row;
    off = 0;
  }
};

template <int D, int HKV, int NT, int PPS, int STAGES, int CTAS>
__global__ void __launch_bounds__((HKV + 1) * 32, CTAS)
kv8_attn_decode_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                       const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale,
                       const int* __restrict__ block_table, const int* __restrict__ ctx_lens, float* __restrict__ part_o,
                       float2* __restrict__ part_ml, int2* __restrict__ rows, __nv_bfloat16* __restrict__ out, int* __restrict__ err, int batch,
                       int num_q_heads, int num_kv_heads, int num_blocks, int max_pages, int min_run, float scale_log2) {
#ifdef B200_DEVICE_OK
  using Cfg = Kv8Cfg<D, HKV, NT, PPS, STAGES>;
  using Word = typename Kv8Word<HKV>::T;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_sm = ring + Cfg::kQ, scale_sm = ring + Cfg::kScales;
  const uint32_t bars = ring + Cfg::kBars;  // full[STAGES], empty[STAGES], queries there, queries read
  const uint32_t bar_q = bars + 16 * STAGES;

  const int lane = threadIdx.x & 31;
  int warp = threadIdx.x >> 5;
  const int head_groups = num_kv_heads / HKV;
  const int kv0 = static_cast<int>(blockIdx.y) % head_groups * HKV;   // first kv head of this CTA
  const int q0 = static_cast<int>(blockIdx.y) / head_groups * (8 * NT);  // first query head of the group
  const int group = num_q_heads / num_kv_heads;
  const int heads = min(group - q0, 8 * NT);  // query heads of a kv head here

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bars + 8 * s, 1);
      mbar_init(bars + 8 * (STAGES + s), HKV);
    }
    mbar_init(bar_q, 1);
    mbar_init(bar_q + 8, HKV);
    fence_mbar_init();
    fence_proxy_async();
  }
  if (warp == HKV && lane == 0) {
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
  }
  // Blocks of two warps would have all consumers on schedulers 0 and 2: every second pair of warps of the SM swaps its roles, whichever warps the
  // hardware took (23.5 -> 19.5 us for 128 rows of 512 to 4096 tokens, 8 / 1 heads of 128).
  if constexpr (HKV == 1) {
    __shared__ int swap_roles;
    int hardware_warp;
    asm volatile("mov.u32 %0, %%warpid;" : "=r"(hardware_warp));
    if (threadIdx.x == 0) swap_roles = (hardware_warp >> 2) & 1;
    __syncthreads();
    warp ^= swap_roles;
  } else {
    __syncthreads();
  }
  grid_dep_wait();  // lengths, queries and the new tokens' pages come from the kernels before
  grid_dep_launch();

  // Rows with no context attend to nothing: zeros, from the producer warp once it has nothing left to ask for.
  auto zero_rows = [&]() {
    if (blockIdx.y != 0) return;
    for (int b = blockIdx.x; b < batch; b += gridDim.x)
      if (ctx_lens[b] <= 0) {
        uint4* to = reinterpret_cast<uint4*>(out + static_cast<size_t>(b) * num_q_heads * D);
        for (int i = lane; i < num_q_heads * D / 8; i += 32) to[i] = make_uint4(0u, 0u, 0u, 0u);
        if (lane == 0) rows[b] = make_int2(0, 0);
      }
  };
  Kv8Walk walk;
  walk.start(ctx_lens, batch, max_pages, min_run, lane, err);
  if (walk.begin >= walk.total) {
    if (warp == HKV) zero_rows();
    return;
  }
  walk.fetch(lane);
  int L = 0, n = 0;
  int stage = 0;  // counts on over the parts

  if (warp == HKV) {
    // ------------------------------------------------------------ producer --
    const int lp = lane >> 1, lkv = lane & 1;  // lane -> (page of the stage, keys or values); one box each
    bool alive = true;
    for (int part = 0; walk.next(lane, L, n) && alive; ++part, walk.advance(n)) {
      const int* table_row = block_table + static_cast<size_t>(walk.row) * max_pages + walk.off;
      auto page_id = [&](int p) {
        int id = p < n ? table_row[p] : 0;
        if (id < 0 || id >= num_blocks) {
          set_error(err, kErrDevBadBlockId);
          id = 0;
        }
        return id;
      };
      int next_ids = page_id(lane), ids = 0;
      // (rooms that are free from the start are not waited for: 7.4 -> 7.05 us for one row of 777 tokens)
      if (part > 0) alive = mbar_wait_warp(bar_q + 8, (part & 1) ^ 1, err);
      if (!alive) break;
      const uint32_t q_bytes = heads * D * 2;
      if (lane == 0) mbar_arrive_expect_tx(bar_q, HKV * q_bytes);
      __syncwarp();
      if (lane < HKV)
        bulk_load(q_sm + lane * q_bytes, q + (static_cast<size_t>(walk.row) * num_q_heads + (kv0 + lane) * group + q0) * D, q_bytes, bar_q);
      Word ks{}, vs{};
      for (int p = 0; p < n; p += PPS, ++stage) {
        if ((p & 31) == 0) {  // ids of 32 pages at a time, one per lane, asked for a batch ahead; their scales
          ids = next_ids;
          if (p + lane < n) {
            const size_t cell = static_cast<size_t>(ids) * num_kv_heads + kv0;
            ks = *reinterpret_cast<const Word*>(k_scale + cell);
            vs = *reinterpret_cast<const Word*>(v_scale + cell);
          }
          next_ids = page_id(p + 32 + lane);
        }
        const int id = __shfl_sync(0xffffffffu, ids, (p + lp) & 31);
        const int slot = stage % STAGES, pages = min(PPS, n - p);
        if (stage >= STAGES) alive = mbar_wait_warp(bars + 8 * (STAGES + slot), (stage / STAGES & 1) ^ 1, err);
        if (!alive) break;
        // The copies may end before the stage's bytes are announced: its phase cannot, without the arrival that comes with them.
        // So they do not wait for the scales.
        if (lp < pages)
          tma_load_2d(ring + slot * Cfg::kStageBytes + lane * Cfg::kPageBytes, lkv ? &v_map : &k_map, bars + 8 * slot, 0,
                      (id * num_kv_heads + kv0) * (Cfg::kHeadBytes / 128));
        const int u = lane - (p & 31);
        if (u >= 0 && u < pages) {
          uint8_t* to = smem_raw + (scale_sm - smem_u32(smem_raw)) + (slot * PPS + u) * 16;
          *reinterpret_cast<Word*>(to) = ks;
          *reinterpret_cast<Word*>(to + 8) = vs;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(bars + 8 * slot, pages * 2 * Cfg::kPageBytes);
      }
    }
    zero_rows();
    return;
  }

  // --------------------------------------------------------------- consumers --
  const int kvh = kv0 + warp;
  const int g = lane >> 2, tq = lane & 3;
  constexpr int KS = D / 16;                       // k-steps of S^T
  constexpr int VB = D / 8;                        // bytes of a V row that a thread takes: columns g * VB ..
  constexpr int VW = VB / 4;                       // as words

  // Address of a 16-byte piece of a token's row, relative to the head's page.
  auto piece = [](int token, int c) {
    if constexpr (D == 128) return static_cast<uint32_t>(token * 128 + ((c ^ (token & 7)) << 4));
    const int row = token >> 1;
    return static_cast<uint32_t>(row * 128 + ((((token & 1) * 4 + c) ^ (row & 7)) << 4));
  };
  const int tok = g ^ ((g & 1) << 2);  // tokens tok, tok + 8: rows g, g + 8 of S^T
  const int tv = 2 * tq, tv1 = (2 * tq) ^ 5;  // tokens of rows 2 tq, 2 tq + 1
  uint32_t k_off[D / 64], v_off[2];
#pragma unroll
  for (int c = 0; c < D / 64; ++c) k_off[c] = piece(tok, c * 4 + tq);
  v_off[0] = piece(tv, g * VB / 16) + (D == 64 ? (g & 1) * 8 : 0);
  v_off[1] = piece(tv1, g * VB / 16) + (D == 64 ? (g & 1) * 8 : 0);
  // eight tokens on: the same piece, since eight rows (or four rows of two tokens, with bit 2 of the row) are one swizzle period
  constexpr uint32_t kEight = 8 * D;

  bool alive = true;  // after a wait that ran out the warp goes through its parts without waiting, so that counters come out even
#pragma unroll 1
  for (int part = 0; walk.next(lane, L, n); ++part, walk.advance(n)) {
    const size_t row0 = static_cast<size_t>(walk.row) * num_q_heads + kvh * group + q0;
    // Q^T fragments, f16.  k-step 4 c + w of thread tq: elements 64 c + 16 tq + 4 w + 0..3 of head_dim (16 tq + 4 w + .. for D = 64).
    uint32_t qb[NT][KS][2];
    // What scores of heads 8 t + 2 tq and + 1 are to be multiplied by, but for the page's scale.  One tile: two factors.  Two tiles, where four
    // registers across the loop made the compiler spill others (16 heads on one 168 against 162 us): the two powers of two of a tile in the halves
    // of a register, taken apart where they are used.  (One tile in that form: a row of 777 tokens 6.8 against 6.3 us.)
    uint32_t back[2];
    auto factor = [&](int t, int k) { return __uint_as_float(NT == 1 ? back[k] : k ? back[t] & 0xffff0000u : back[t] << 16); };
    {
      if (alive) alive = mbar_wait_warp(bar_q, part & 1, err);
      uint32_t top[NT];  // largest magnitudes of head 8 t + g so far, two side by side
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        top[t] = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          qb[t][ks][0] = qb[t][ks][1] = 0u;
          if (8 * t + g < heads)
            lds_words<8>(q_sm + ((warp * heads + 8 * t + g) * D + (ks >> 2) * 64 + tq * 16 + (ks & 3) * 4) * 2, qb[t][ks]);
          top[t] = __vmaxu2(top[t], __vmaxu2(qb[t][ks][0] & 0x7fff7fffu, qb[t][ks][1] & 0x7fff7fffu));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q + 8);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        uint32_t m2 = max(top[t] >> 16, top[t] & 0xffffu);  // the head's four lanes share it
        m2 = max(m2, __shfl_xor_sync(0xffffffffu, m2, 1));
        m2 = max(m2, __shfl_xor_sync(0xffffffffu, m2, 2));
        // bf16 and fp32 have the same exponents, -127 (zeros) to 128 (infinities); tiny queries may stay below the top.  Scores of a head that
        // is not finite are all infinite or NaN, so its softmax is NaN.
        const int shift = min(kKv8QueryTop - (static_cast<int>(m2 >> 7) - 127), 100);
        const float by = m2 < 0x7f80u ? power_of_two(shift) : NAN;
        const uint32_t mine = __float_as_uint((NT == 1 ? scale_log2 : 1.f) * power_of_two(-shift));
        const uint32_t a = __shfl_sync(0xffffffffu, mine, 8 * tq), b = __shfl_sync(0xffffffffu, mine, 8 * tq + 4);  // of lanes whose g is 2 tq (+ 1)
        if (NT == 1) back[0] = a, back[1] = b;
        else back[t] = a >> 16 | b;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            qb[t][ks][k] = pack_f16x2(__uint_as_float(qb[t][ks][k] << 16) * by, __uint_as_float(qb[t][ks][k] & 0xffff0000u) * by);
      }
    }

    float o[NT][D / 16][4];  // O^T: rows g * VB + 2 j (+ 1), columns: heads 2 tq, 2 tq + 1
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[t][j][0] = o[t][j][1] = o[t][j][2] = o[t][j][3] = 0.f;
    }

#pragma unroll 1
    for (int p0 = 0; p0 < n; p0 += PPS, ++stage) {
      const int slot = stage % STAGES;
      const int left = L - (walk.off + p0) * kKvPage;  // tokens of the row from this stage on
      if (alive) alive = mbar_wait_warp(bars + 8 * slot, stage / STAGES & 1, err);
      const uint32_t base = ring + slot * Cfg::kStageBytes + warp * Cfg::kHeadBytes;
      float s[PPS][NT][4];
      int ev[PPS];
#pragma unroll
      for (int u = 0; u < PPS; ++u) {
#pragma unroll
        for (int t = 0; t < NT; ++t) s[u][t][0] = s[u][t][1] = s[u][t][2] = s[u][t][3] = -INFINITY;
        ev[u] = 0;
        if (u > 0 && p0 + u >= n) continue;
        const uint32_t kb = base + u * 2 * Cfg::kPageBytes;
        float acc[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          uint32_t x[4], y[4];
          lds_words<16>(kb + k_off[c], x);
          lds_words<16>(kb + (D == 128 ? k_off[c] + kEight : (k_off[c] ^ 64u) + kEight), y);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a0, a1, a2, a3;
            e4m3x4_to_f16(x[w], a0, a2);
            e4m3x4_to_f16(y[w], a1, a3);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_f16_16816(acc[t], a0, a1, a2, a3, qb[t][c * 4 + w][0], qb[t][c * 4 + w][1]);
          }
        }
        int kbyte, vbyte;
        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(kbyte) : "r"(scale_sm + (slot * PPS + u) * 16 + warp));
        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(vbyte) : "r"(scale_sm + (slot * PPS + u) * 16 + 8 + warp));
        const float f = (NT == 1 ? 1.f : scale_log2) * power_of_two(scale_exponent(kbyte));
        ev[u] = scale_exponent(vbyte);
        const float lv = static_cast<float>(ev[u]);
        const int here = left - u * kKvPage;  // tokens of this page, if fewer than 16
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (NT == 2) asm volatile("" : "+r"(back[t]));  // not ahead of the loop
          const float f_t[2] = {factor(t, 0) * f, factor(t, 1) * f};
#pragma unroll
          for (int k = 0; k < 4; ++k) s[u][t][k] = tok + (k >> 1) * 8 < here ? fmaf(acc[t][k], f_t[k & 1], lv) : -INFINITY;
        }
        if (here < kKvPage) {
          // the last page: what lies behind the last token may be NaN, which a weight of zero does not undo
          const uint32_t vb = kb + Cfg::kPageBytes;
          for (int x = here; x < kKvPage; ++x)
            if (lane < D / 4) asm volatile("st.shared.b32 [%0], %1;" ::"r"(vb + piece(x, lane >> 2) + (lane & 3) * 4), "r"(0) : "memory");
          fence_proxy_async();  // a later copy overwrites the stage
          __syncwarp();
        }
      }

      // references: s is the exponent of the weight times its value scale
      bool over = false;
      float top[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float x = fmaxf(s[0][t][k], s[0][t][k + 2]);
#pragma unroll
          for (int u = 1; u < PPS; ++u) x = fmaxf(x, fmaxf(s[u][t][k], s[u][t][k + 2]));
          top[t][k] = x;
          over |= x > m[t][k] + kKv8RefSlack;
        }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float x = top[t][k];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            x = fmaxf(x, m[t][k]);
            const float a = x == -INFINITY ? 1.f : fast_ex2(m[t][k] - x);  // still nothing but scores of -inf: sums are zero
            m[t][k] = x;
            l[t][k] *= a;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              o[t][j][k] *= a;
              o[t][j][k + 2] *= a;
            }
          }
      }

#pragma unroll
      for (int u = 0; u < PPS; ++u) {
        if (u > 0 && p0 + u >= n) continue;
        uint32_t pb[NT][2];
        const float iv = power_of_two(-ev[u]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float e[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) e[k] = fast_ex2(s[u][t][k] - (m[t][k & 1] == -INFINITY ? 0.f : m[t][k & 1] - kKv8Lift));
          l[t][0] = fmaf(e[0] + e[2], iv, l[t][0]);
          l[t][1] = fmaf(e[1] + e[3], iv, l[t][1]);
          pb[t][0] = transpose_8x8(pack_f16x2(e[0], e[1]));
          pb[t][1] = transpose_8x8(pack_f16x2(e[2], e[3]));
        }
        const uint32_t vb = base + u * 2 * Cfg::kPageBytes + Cfg::kPageBytes;
        uint32_t w00[VW], w01[VW], w10[VW], w11[VW];  // tokens tv, tv1, tv + 8, tv1 + 8
        lds_words<VB>(vb + v_off[0], w00);
        lds_words<VB>(vb + v_off[1], w01);
        lds_words<VB>(vb + (D == 128 ? v_off[0] + kEight : (v_off[0] ^ 64u) + kEight), w10);
        lds_words<VB>(vb + (D == 128 ? v_off[1] + kEight : (v_off[1] ^ 64u) + kEight), w11);
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t a[4][2];  // columns 0..3 of the word x token pairs
          e4m3x4_to_f16(__byte_perm(w00[w], w01[w], 0x5140), a[0][0], a[1][0]);
          e4m3x4_to_f16(__byte_perm(w00[w], w01[w], 0x7362), a[2][0], a[3][0]);
          e4m3x4_to_f16(__byte_perm(w10[w], w11[w], 0x5140), a[0][1], a[1][1]);
          e4m3x4_to_f16(__byte_perm(w10[w], w11[w], 0x7362), a[2][1], a[3][1]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_f16_16816(o[t][2 * w], a[0][0], a[1][0], a[0][1], a[1][1], pb[t][0], pb[t][1]);
            mma_f16_16816(o[t][2 * w + 1], a[2][0], a[3][0], a[2][1], a[3][1], pb[t][0], pb[t][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + 8 * (STAGES + slot));
    }

    const int row_at = walk.at - walk.off;  // first page of the row among all pages
    const int first_run = row_at / walk.per, parts = (row_at + (L + kKvPage - 1) / kKvPage - 1) / walk.per - first_run + 1;
    // a part that begins with the run is the first of its two, one that does not is the second and the row's first part
    const bool second = walk.at != walk.begin;
    const size_t here = static_cast<size_t>(blockIdx.x) * 2 + second;
    if (first_run == static_cast<int>(blockIdx.x) && blockIdx.y == 0 && warp == 0 && lane == 0)
      rows[walk.row] = make_int2(first_run * 2 + second, parts);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float sum = l[t][k];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const int head = 8 * t + 2 * tq + k;
        if (head >= heads) continue;
        if (parts == 1) {
          const float inv = 1.f / sum;
          uint32_t r[VB / 2];
#pragma unroll
          for (int j = 0; j < D / 16; ++j) r[j] = pack_bf16x2(o[t][j][k] * inv, o[t][j][k + 2] * inv);
          uint32_t* to = reinterpret_cast<uint32_t*>(out + (row0 + head) * D + g * VB);
#pragma unroll
          for (int j = 0; j < D / 16; j += 4) *reinterpret_cast<uint4*>(to + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
        } else {
          const size_t prow = here * num_q_heads + kvh * group + q0 + head;
          float* to = part_o + prow * D + g * VB;
#pragma unroll
          for (int j = 0; j < D / 16; j += 2)
            *reinterpret_cast<float4*>(to + 2 * j) = make_float4(o[t][j][k], o[t][j][k + 2], o[t][j + 1][k], o[t][j + 1][k + 2]);
          if (g == 0) part_ml[prow] = make_float2(m[t][k], sum);
        }
      }
  }
#endif
}

// Where the parts of a (row, query head) are: part 0, then `next`, `next` + `step`, ...  With `rows` they are those of kv8_attn_decode_kernel;
// without, every row has `parts` of them, side by side, some perhaps empty (their reference is -inf and their sums are not written).
struct Kv8Parts {
  int n;
  long long first, next;
  int step;
  __device__ __forceinline__ Kv8Parts(const int2* rows, int row, int num_q_heads, int parts) {
    if (rows == nullptr) {
      n = parts;
      first = static_cast<long long>(row) * parts;
      next = first + 1;
      step = 1;
    } else {
      const int2 at = rows[row / num_q_heads];
      const int head = row % num_q_heads;
      n = at.y;
      first = static_cast<long long>(at.x) * num_q_heads + head;
      next = static_cast<long long>((at.x | 1) + 1) * num_q_heads + head;  // the first part of the run after
      step = 2 * num_q_heads;
    }
  }
  __device__ __forceinline__ size_t at(int k) const { return static_cast<size_t>(k == 0 ? first : next + static_cast<long long>(k - 1) * step); }
};

// Joins the parts of one (row, query head) per warp, eight at a time, each lane D / 32 columns: for batches, whose rows have a handful.
template <int D>
__global__ void __launch_bounds__(128)
kv8_attn_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, const int2* __restrict__ rows,
                     __nv_bfloat16* __restrict__ out, int num_q_heads, int num_rows, int parts) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31, row = static_cast<int>(blockIdx.x * 4 + (threadIdx.x >> 5));
  if (row >= num_rows) return;
  const Kv8Parts where(rows, row, num_q_heads, parts);
  if (rows != nullptr && where.n <= 1) return;  // written by its one CTA
  float top = -INFINITY, den = 0.f, acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
#pragma unroll 1
  for (int k0 = 0; k0 < where.n; k0 += 8) {
    float v[8][V];
    float2 ml[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int j = 0; j < V; ++j) v[u][j] = 0.f;
      if (k0 + u < where.n) {
        const size_t from = where.at(k0 + u);
        ml[u] = part_ml[from];
#pragma unroll
        for (int j = 0; j < V; ++j) v[u][j] = part_o[from * D + lane * V + j];
      }
    }
    float t = top;
#pragma unroll
    for (int u = 0; u < 8; ++u) t = fmaxf(t, ml[u].x);
    const float ref = t == -INFINITY ? 0.f : t;
    const float a = fast_ex2(top - ref);
    top = t;
    den *= a;
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] *= a;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float w = fast_ex2(ml[u].x - ref);
      den = fmaf(w, ml[u].y, den);
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] = fmaf(w, ml[u].x == -INFINITY ? 0.f : v[u][j], acc[j]);
    }
  }
  const float inv = 1.f / den;
  uint32_t* to = reinterpret_cast<uint32_t*>(out + static_cast<size_t>(row) * D + lane * V);
#pragma unroll
  for (int j = 0; j < V; j += 2) to[j / 2] = pack_bf16x2(acc[j] * inv, acc[j + 1] * inv);
}

// The same for few rows of many parts: a CTA of WARPS warps per (row, query head) and 32 columns, eight lanes per part, so that all parts are
// asked for at once: 32 parts a round with four warps, or 320 with sixteen.  (16 warps over all columns with three rounds: 8 us for 296 parts.)
template <int D, int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
kv8_attn_join_wide_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, const int2* __restrict__ rows,
                          __nv_bfloat16* __restrict__ out, int num_q_heads, int parts) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int kRound = WARPS == 4 ? 2 : 5;  // parts of a thread and round
  __shared__ float4 o_sm[WARPS][8];
  __shared__ float2 ml_sm[WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.y * 32 + (lane & 7) * 4;
  const int row = blockIdx.x;
  const Kv8Parts where(rows, row, num_q_heads, parts);
  if (rows != nullptr && where.n <= 1) return;
  float top = -INFINITY, den = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int k0 = warp * 4 + (lane >> 3); k0 < where.n; k0 += kRound * WARPS * 4) {
    float4 v[kRound];
    float2 ml[kRound];
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      const int k = k0 + u * WARPS * 4;
      ml[u] = make_float2(-INFINITY, 0.f);
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k < where.n) {
        const size_t from = where.at(k);
        ml[u] = part_ml[from];
        v[u] = *reinterpret_cast<const float4*>(part_o + from * D + col);
      }
    }
    float t = top;
#pragma unroll
    for (int u = 0; u < kRound; ++u) t = fmaxf(t, ml[u].x);
    const float ref = t == -INFINITY ? 0.f : t, a = fast_ex2(top - ref);
    top = t;
    den *= a;
    acc.x *= a, acc.y *= a, acc.z *= a, acc.w *= a;
#pragma unroll
    for (int u = 0; u < kRound; ++u) {
      const float w = fast_ex2(ml[u].x - ref);
      den = fmaf(w, ml[u].y, den);
      if (ml[u].x != -INFINITY) {
        acc.x = fmaf(w, v[u].x, acc.x);
        acc.y = fmaf(w, v[u].y, acc.y);
        acc.z = fmaf(w, v[u].z, acc.z);
        acc.w = fmaf(w, v[u].w, acc.w);
      }
    }
  }
  // the four parts that a warp takes side by side, then the warps, each time against the common reference
  auto into = [](float mine, float common) { return fast_ex2(mine - (common == -INFINITY ? 0.f : common)); };
  const float warp_top = warp_max(top), a = into(top, warp_top);
  den *= a;
  acc.x *= a, acc.y *= a, acc.z *= a, acc.w *= a;
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) {
    den += __shfl_xor_sync(0xffffffffu, den, o);
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, o);
    acc.y += __shfl_xor_sync(0xffffffffu, acc.y, o);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, o);
    acc.w += __shfl_xor_sync(0xffffffffu, acc.w, o);
  }
  if (lane < 8) o_sm[warp][lane] = acc;
  if (lane == 0) ml_sm[warp] = make_float2(warp_top, den);
  __syncthreads();
  if (threadIdx.x >= 32) return;
  float t = ml_sm[0].x;
#pragma unroll
  for (int w = 1; w < WARPS; ++w) t = fmaxf(t, ml_sm[w].x);
  float num = 0.f, sum = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const float x = into(ml_sm[w].x, t);
    num += x * reinterpret_cast<const float*>(o_sm[w])[lane];
    sum += x * ml_sm[w].y;
  }
  out[static_cast<size_t>(row) * D + blockIdx.y * 32 + lane] = __float2bfloat16(num / sum);
}

// `expected`: parts that a row is likely to have.  The wide form where they are many and the rows few: us for a whole call, narrow and
// wide, 528 rows of 18 parts 12.3, 10.3; 1088 rows of 11 parts 27.7, 29.7.
template <int D>
static int launch_join(const float* o, const float2* ml, const int2* rows, void* out, int hq, int num_rows, int parts, int expected,
                       cudaStream_t st) {
  __nv_bfloat16* to = static_cast<__nv_bfloat16*>(out);
  if (expected <= 8 || num_rows >= 1024)
    B200_CUDA(launch_overlapped(kv8_attn_join_kernel<D>, dim3((num_rows + 3) / 4), dim3(128), 0, st, o, ml, rows, to, hq, num_rows, parts));
  else if (expected <= 64)
    B200_CUDA(launch_overlapped(kv8_attn_join_wide_kernel<D, 4>, dim3(num_rows, D / 32), dim3(128), 0, st, o, ml, rows, to, hq, parts));
  else
    B200_CUDA(launch_overlapped(kv8_attn_join_wide_kernel<D, 16>, dim3(num_rows, D / 32), dim3(512), 0, st, o, ml, rows, to, hq, parts));
  return 0;
}
int launch_kv8_join(int head_dim, const AttnWorkspace& w, void* out, int rows, int hq, int parts, cudaStream_t st) {
  return head_dim == 128 ? launch_join<128>(w.o, w.ml, nullptr, out, hq, rows * hq, parts, parts, st)
                         : launch_join<64>(w.o, w.ml, nullptr, out, hq, rows * hq, parts, parts, st);
}

// How a call is laid out.  `min_run`: pages of a run at least.
struct Kv8Plan {
  int hkv, nt, slices, runs, min_run;
};
static int kv8_plan(int batch, int hq, int hkv, int head_dim, int max_pages, int split_tokens, Kv8Plan* p) {
  const int group = hq / hkv;
  p->hkv = kv8_heads_per_cta(head_dim, hkv);
  p->nt = group > 8 ? 2 : 1;
  p->slices = (group + 15) / 16;
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc) return rc;
  const int y = hkv / p->hkv * p->slices, held = kv8_ctas_per_sm(head_dim, p->hkv, p->nt) * sms;
  p->runs = y >= held ? 1 : held / y;
  // Short rows: a run's start costs about as much as four pages, a join as much as a run.  us with runs of at least 1, 2, 4, 8 pages, 32 /
  // 4 heads of 128: one row of 300 tokens 6.6, 6.9, 7.2, 8.7, of 1500 8.2, 7.4, 7.6, 9.0, of 6000 9.4 each; 4 rows of 300 7.6, 8.8, 9.4,
  // 10.6, of 1000 10.5, 9.4, 9.9, 10.8.
  p->min_run = split_tokens > 0 ? split_tokens / kKvPage : 2;
  return 0;
}

struct Kv8Args {
  const void *q, *k_pool, *v_pool, *k_scale, *v_scale;
  const int *table, *ctx;
  void* out;
  Kv8Workspace w;
  int batch, hq, hkv, num_blocks, max_pages;
  float scale;
  Kv8Plan plan;
  cudaStream_t st;
};

template <int D, int HKV, int NT, int PPS, int STAGES, int CTAS>
static int launch_kv8_decode(const Kv8Args& a) {
  using Cfg = Kv8Cfg<D, HKV, NT, PPS, STAGES>;
  static_assert(CTAS * (Cfg::kSmemBytes + 1024 + 128) <= 228 * 1024, "runs are cut for CTAS per SM");
  CUtensorMap kmap, vmap;
  const uint64_t rows = static_cast<uint64_t>(a.num_blocks) * a.hkv * (Cfg::kHeadBytes / 128);
  int rc = get_tensor_map_2d(a.k_pool, rows, 128, 1, Cfg::kPageBytes / 128, 128, &kmap);
  if (rc) return rc;
  rc = get_tensor_map_2d(a.v_pool, rows, 128, 1, Cfg::kPageBytes / 128, 128, &vmap);
  if (rc) return rc;
  auto kernel = kv8_attn_decode_kernel<D, HKV, NT, PPS, STAGES, CTAS>;
  rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), Cfg::kSmemBytes);
  if (rc) return rc;
  B200_CUDA(launch_overlapped(kernel, dim3(a.plan.runs, a.hkv / HKV * a.plan.slices), dim3(Cfg::kThreads), Cfg::kSmemBytes, a.st, kmap, vmap,
                              static_cast<const __nv_bfloat16*>(a.q), static_cast<const uint8_t*>(a.k_scale),
                              static_cast<const uint8_t*>(a.v_scale), a.table, a.ctx, a.w.o, a.w.ml, a.w.rows,
                              static_cast<__nv_bfloat16*>(a.out), a.w.err, a.batch, a.hq, a.hkv, a.num_blocks, a.max_pages, a.plan.min_run,
                              a.scale * 1.4426950408889634f));
  if (a.batch == 1 && a.max_pages <= a.plan.min_run) return 0;  // one run
  // Rows share the runs: a row has about runs / batch parts, and no more than its pages give.
  const int expected = static_cast<int>(std::min<long long>(a.plan.runs / a.batch, static_cast<long long>(a.max_pages - 1) / a.plan.min_run) + 1);
  return launch_join<D>(a.w.o, a.w.ml, a.w.rows, a.out, a.hq, a.batch * a.hq, 0, expected, a.st);
}

template <int D, int NT>
static int launch_kv8_heads(const Kv8Args& a) {
  if constexpr (D == 128) {  // the only head_dim with 8 (kv8_heads_per_cta)
    if (a.plan.hkv == 8) return launch_kv8_decode<D, 8, NT, 1, 5, kv8_ctas_per_sm(D, 8, NT)>(a);
  }
  switch (a.plan.hkv) {
    case 1: return launch_kv8_decode<D, 1, NT, 2, 4, kv8_ctas_per_sm(D, 1, NT)>(a);
    case 2: return launch_kv8_decode<D, 2, NT, 2, D == 128 ? 3 : 4, kv8_ctas_per_sm(D, 2, NT)>(a);
    default: return launch_kv8_decode<D, 4, NT, D == 128 && NT == 2 ? 1 : 2, D == 128 ? (NT == 2 ? 5 : 3) : 4, kv8_ctas_per_sm(D, 4, NT)>(a);
  }
}

}  // namespace b200

using namespace b200;

int b200::check_kv8(const char* name, int batch, int hq, int hkv, int head_dim, int num_blocks, int max_pages, const void* q,
                    const void* k_pool, const void* v_pool, const void* out, float scale) {
  B200_REQUIRE(batch > 0 && hq > 0 && hkv > 0 && num_blocks > 0 && max_pages > 0, "%s: non-positive dimension", name);
  B200_REQUIRE(hq % hkv == 0, "%s: q heads %d not a multiple of kv heads %d", name, hq, hkv);
  B200_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim %d is neither 64 nor 128", name, head_dim);
  B200_REQUIRE(static_cast<long long>(max_pages) * kKvPage < (1ll << 31) && static_cast<long long>(num_blocks) * hkv * kKvPage < (1ll << 31),
               "%s: positions or pool rows past 2^31", name);
  B200_REQUIRE(((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool) | reinterpret_cast<uintptr_t>(q) |
                 reinterpret_cast<uintptr_t>(out)) & 15) == 0,
               "%s: pools, q and out must be 16-byte aligned", name);
  B200_REQUIRE(scale > 0.f && scale < 3e38f, "%s: scale must be positive and finite", name);
  return 0;
}

extern "C" size_t b200_kv8_attn_workspace_bytes(int batch, int num_q_heads, int num_kv_heads, int head_dim, int max_pages_per_seq,
                                                int split_tokens) {
  if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || max_pages_per_seq <= 0 || split_tokens < 0 ||
      num_q_heads % num_kv_heads != 0)
    return 256;
  Kv8Plan p;
  if (kv8_plan(batch, num_q_heads, num_kv_heads, head_dim, max_pages_per_seq, split_tokens, &p)) return 256;
  return carve_kv8(nullptr, batch, p.runs, num_q_heads, head_dim).bytes;
}

extern "C" int b200_kv8_attn_decode(const void* q, const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale,
                                    const int32_t* block_table, const int32_t* ctx_lens, void* out, void* workspace,
                                    size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads, int head_dim, int num_blocks,
                                    int max_pages_per_seq, float scale, int split_tokens, void* stream) {
  B200_REQUIRE(q && k_pool && v_pool && k_scale && v_scale && block_table && ctx_lens && out && workspace, "kv8_attn_decode: null pointer");
  int rc = check_kv8("kv8_attn_decode", batch, num_q_heads, num_kv_heads, head_dim, num_blocks, max_pages_per_seq, q, k_pool, v_pool, out, scale);
  if (rc) return rc;
  B200_REQUIRE(on_words(block_table, ctx_lens), "kv8_attn_decode: block table and lengths must be 4-byte aligned");
  B200_REQUIRE(split_tokens >= 0 && split_tokens % kKvPage == 0, "kv8_attn_decode: split_tokens %d not a multiple of %d", split_tokens, kKvPage);
  B200_REQUIRE(static_cast<long long>(batch) * max_pages_per_seq < (1ll << 31), "kv8_attn_decode: the table has more than 2^31 entries");
  rc = check_device(nullptr);
  if (rc) return rc;
  Kv8Args a{q, k_pool, v_pool, k_scale, v_scale, block_table, ctx_lens, out, {}, batch, num_q_heads, num_kv_heads, num_blocks,
            max_pages_per_seq, scale, {}, as_stream(stream)};
  rc = kv8_plan(batch, num_q_heads, num_kv_heads, head_dim, max_pages_per_seq, split_tokens, &a.plan);
  if (rc) return rc;
  B200_REQUIRE(num_kv_heads / a.plan.hkv * a.plan.slices <= 65535 && static_cast<long long>(batch) * num_q_heads < (1ll << 31),
               "kv8_attn_decode: grid too large");
  B200_REQUIRE(reinterpret_cast<uintptr_t>(k_scale) % a.plan.hkv == 0 && reinterpret_cast<uintptr_t>(v_scale) % a.plan.hkv == 0,
               "kv8_attn_decode: scales must be %d-byte aligned", a.plan.hkv);
  a.w = carve_kv8(workspace, batch, a.plan.runs, num_q_heads, head_dim);
  if (workspace_bytes < a.w.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) {
    set_detail("kv8_attn_decode: workspace of %zu bytes at %p, %zu on a 16-byte boundary are needed", workspace_bytes, workspace, a.w.bytes);
    return -kErrWorkspace;
  }
  if (head_dim == 128) return a.plan.nt == 1 ? launch_kv8_heads<128, 1>(a) : launch_kv8_heads<128, 2>(a);
  return a.plan.nt == 1 ? launch_kv8_heads<64, 1>(a) : launch_kv8_heads<64, 2>(a);
}
