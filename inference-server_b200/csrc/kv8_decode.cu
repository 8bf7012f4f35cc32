// Paged decode attention over the 8-bit page cache (kv8.cuh) for sm_100a: the counterpart of paged_attn.cu, which reads 16-bit pools,
// and so of the same steps of the reference (src/inference_server/kv_cache/hf_format.py:21-45 and
// src/inference_server/backends/torch_backend.py:305-322).
//
// Mathematics.  A page and kv head has scales 2^ek (keys) and 2^ev (values).  With scores s_t = scale * log2(e) * 2^ek (q . k_t) of the
// e4m3 numbers k_t, the output is  sum_t 2^(s_t + ev) v_t / sum_t 2^s_t.  A value's scale is taken into its weight's exponent:
// p_t = 2^(s_t + ev - m), where m follows the maximum of s_t + ev, so the largest weight sees the largest product and not the largest
// score.  The denominator is sum_t p_t 2^-ev.  Everything that has a scale in it is an fp32 exponent; e4m3 numbers become f16 exactly, and
// weights are f16, whose 11 bits leave them a 16th of the error of bf16.  Weights are taken so that
// the largest is between 2^6 and 2^14; those below 2^-14 lose bits.  Queries are multiplied by a power of two that brings the largest of a kv group to 2^14 and become f16: what loses bits
// is 2^-28 of the largest.  Sums are fp32.  With |ev| <= 32 the sums p_t 2^-ev stay below 2^14 * 2^32 * tokens.
//
//   grid   (batch, splits, groups of kv heads x slices of 16 query heads); block = one consumer warp per kv head + a producer warp.  A
//          CTA owns `split_tokens` tokens of a sequence; the kv heads of a page are adjacent, so a page is one contiguous read of
//          16 * HKV * D bytes for the keys and one for the values.
//   load   TMA boxes of 128-byte rows with 128-byte swizzle into a ring of stages of PPS pages.
//   math   transposed: S^T = K Q^T and O^T = V^T P^T with mma.sync m16n8k16, so that the 16 rows of the tile are tokens, or columns of V,
//          and not the few heads of a group: 16 MMAs per page, half of what the other orientation needs, and 32 accumulators a thread.
//          The order of head_dim in the products is free, so a thread's A operands come from its own 16-byte pieces of K rows without a
//          transposition; those of V^T take bytes of two tokens and one column together with one byte permutation per four bytes of
//          each.  P^T comes from S^T by one movmatrix per 8 x 8 tile.
//   max    lazy, against 2^8: whether any score of the page outgrew its row's reference is one vote; only then are there shuffles.
//   out    a sequence that fits one split is written by its CTA.  Otherwise fp32 partials (o, m, l), joined by a second kernel.
//
// Bank conflicts: a token's row is 128 bytes, its 16-byte pieces XORed with the row number.  A quarter warp reads K pieces of two
// neighbouring g = lane / 4, so their rows must differ in bit 2; it reads V pieces of four tq = lane % 4, whose rows must differ in
// bits 1 and 2.  Row g of a tile is therefore token g ^ 4 (g & 1) of its eight.

#include "host.h"
#include "kv8.cuh"

namespace b200 {

constexpr float kKv8RefSlack = 8.f;    // a score may pass its reference by 2^8 before the reference moves
constexpr float kKv8Lift = 6.f;        // weights are taken times 2^6: at most 2^14 in f16
constexpr int kKv8QueryTop = 14;       // exponent that the largest query of a kv group is brought to

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

// D: head_dim.  HKV: kv heads = consumer warps.  NT: tiles of 8 query heads per kv head.  PPS: pages per stage.
template <int D, int HKV, int NT, int PPS, int STAGES>
struct Kv8Cfg {
  static constexpr int kThreads = (HKV + 1) * 32;
  static constexpr int kHeadBytes = kKvPage * D;
  static constexpr int kPageBytes = HKV * kHeadBytes;      // keys, or values, of a page's kv heads
  static constexpr int kStageBytes = PPS * 2 * kPageBytes;  // page by page: keys, values
  static constexpr int kRingBytes = STAGES * kStageBytes;
  static constexpr int kSmemBytes = kRingBytes + 1024 /* alignment slack */ + 16 * STAGES /* barriers */;
};

template <int D, int HKV, int NT, int PPS, int STAGES, int CTAS>
__global__ void __launch_bounds__((HKV + 1) * 32, CTAS)
kv8_attn_decode_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                       const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale,
                       const int* __restrict__ block_table, const int* __restrict__ ctx_lens, float* __restrict__ part_o,
                       float2* __restrict__ part_ml, __nv_bfloat16* __restrict__ out, int* __restrict__ err, int num_q_heads,
                       int num_kv_heads, int num_blocks, int max_pages, int split_tokens, int max_splits, float scale_log2) {
#ifdef B200_DEVICE_OK
  grid_dep_wait();  // lengths, queries and the new tokens' pages come from the kernels before
  grid_dep_launch();
  using Cfg = Kv8Cfg<D, HKV, NT, PPS, STAGES>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = ring + Cfg::kRingBytes;  // full[STAGES], empty[STAGES]

  const int b = blockIdx.x, split = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head_groups = num_kv_heads / HKV;
  const int kv0 = static_cast<int>(blockIdx.z) % head_groups * HKV;   // first kv head of this CTA
  const int q0 = static_cast<int>(blockIdx.z) / head_groups * (8 * NT);  // first query head of the group
  const int group = num_q_heads / num_kv_heads;
  const int heads = min(group - q0, 8 * NT);  // query heads of a kv head here

  int L = ctx_lens[b];
  if (L < 0 || L > max_pages * kKvPage) {
    if (threadIdx.x == 0) set_error(err, kErrDevBadCtxLen);
    L = L < 0 ? 0 : max_pages * kKvPage;
  }
  const int start = split * split_tokens;
  if (start >= L) {  // uniform for the whole CTA
    if (L == 0 && split == 0 && blockIdx.z == 0)  // a row with no context attends to nothing: zeros
      for (int i = threadIdx.x; i < num_q_heads * D; i += blockDim.x)
        out[static_cast<size_t>(b) * num_q_heads * D + i] = __float2bfloat16(0.f);
    return;
  }
  const int end = min(L, start + split_tokens);
  const int npages = (end - start + kKvPage - 1) / kKvPage;
  const int nstages = (npages + PPS - 1) / PPS;
  const int* table_row = block_table + static_cast<size_t>(b) * max_pages + start / kKvPage;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bars + 8 * s, 1);
      mbar_init(bars + 8 * (STAGES + s), HKV);
    }
    fence_mbar_init();
    fence_proxy_async();
  }
  __syncthreads();

  if (warp == HKV) {
    // ------------------------------------------------------------ producer --
    if (lane == 0) {
      tma_prefetch_desc(&k_map);
      tma_prefetch_desc(&v_map);
    }
    const int lp = lane >> 1, lkv = lane & 1;  // lane -> (page of the stage, keys or values); one box each
    int ids = 0;                               // page ids, 32 at a time, one per lane
    for (int i = 0; i < nstages; ++i) {
      const int p0 = i * PPS;
      if ((p0 & 31) == 0) {
        ids = p0 + lane < npages ? table_row[p0 + lane] : 0;
        if (ids < 0 || ids >= num_blocks) {
          set_error(err, kErrDevBadBlockId);
          ids = 0;
        }
      }
      const int id = __shfl_sync(0xffffffffu, ids, (p0 + lp) & 31);
      const int slot = i % STAGES;
      const uint32_t phase = (i / STAGES) & 1;
      if (!mbar_wait(bars + 8 * (STAGES + slot), phase ^ 1, err)) break;
      const int pages = min(PPS, npages - p0);
      if (lane == 0) mbar_arrive_expect_tx(bars + 8 * slot, pages * 2 * Cfg::kPageBytes);
      __syncwarp();
      if (lp < pages)
        tma_load_2d(ring + slot * Cfg::kStageBytes + lane * Cfg::kPageBytes, lkv ? &v_map : &k_map, bars + 8 * slot, 0,
                    (id * num_kv_heads + kv0) * (Cfg::kHeadBytes / 128));
    }
    return;
  }

  // --------------------------------------------------------------- consumers --
  const int kvh = kv0 + warp;
  const int g = lane >> 2, tq = lane & 3;
  constexpr int KS = D / 16;                       // k-steps of S^T
  constexpr int VB = D / 8;                        // bytes of a V row that a thread takes: columns g * VB ..
  constexpr int VW = VB / 4;                       // as words
  const size_t row0 = static_cast<size_t>(b) * num_q_heads + kvh * group + q0;

  // Scales of 32 pages at a time, one per lane, asked for a batch ahead.
  auto page_id = [&](int p) {
    const int id = p < npages ? table_row[p] : 0;
    return id < 0 || id >= num_blocks ? 0 : id;  // the producer reports it
  };
  int ids = page_id(lane);
  int ek = k_scale[static_cast<size_t>(ids) * num_kv_heads + kvh], ev = v_scale[static_cast<size_t>(ids) * num_kv_heads + kvh];
  int ek_next = 0, ev_next = 0;
  ids = page_id(32 + lane);

  // Q^T fragments, f16.  k-step 4 c + w of thread tq: elements 64 c + 16 tq + 4 w + 0..3 of head_dim (16 tq + 4 w + .. for D = 64).
  uint32_t qb[NT][KS][2];
  float f_q;  // what a score is to be multiplied by, but for the page's scale
  {
    uint2 raw[NT][KS];
    uint32_t top = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        raw[n][ks] = make_uint2(0u, 0u);
        if (8 * n + g < heads)
          raw[n][ks] = __ldg(reinterpret_cast<const uint2*>(q + (row0 + 8 * n + g) * D + (ks >> 2) * 64 + tq * 16 + (ks & 3) * 4));
        const uint32_t a = raw[n][ks].x & 0x7fff7fffu, c = raw[n][ks].y & 0x7fff7fffu;
        top = max(top, max(max(a >> 16, a & 0xffffu), max(c >> 16, c & 0xffffu)));
      }
    top = __reduce_max_sync(0xffffffffu, top);
    // bf16 and fp32 have the same exponents, -127 (zeros) to 128 (infinities); tiny queries may stay below the top
    const int shift = min(kKv8QueryTop - (static_cast<int>(top >> 7) - 127), 100);
    const float by = power_of_two(shift);
    f_q = scale_log2 * power_of_two(-shift);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint32_t x = raw[n][ks].x, y = raw[n][ks].y;
        qb[n][ks][0] = pack_f16x2(__uint_as_float(x << 16) * by, __uint_as_float(x & 0xffff0000u) * by);
        qb[n][ks][1] = pack_f16x2(__uint_as_float(y << 16) * by, __uint_as_float(y & 0xffff0000u) * by);
      }
  }

  float o[NT][D / 16][4];  // O^T: rows g * VB + 2 j (+ 1), columns: heads 2 tq, 2 tq + 1
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
  }

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

  bool alive = true;
  for (int i = 0; i < nstages && alive; ++i) {
    const int slot = i % STAGES;
    const uint32_t phase = (i / STAGES) & 1;
    const int p0 = i * PPS;
    if ((p0 & 31) == 0) {
      if (p0 > 0) {
        ek = ek_next;
        ev = ev_next;
      }
      if (p0 + 32 < npages) {
        ek_next = k_scale[static_cast<size_t>(ids) * num_kv_heads + kvh];
        ev_next = v_scale[static_cast<size_t>(ids) * num_kv_heads + kvh];
        ids = page_id(p0 + 64 + lane);
      }
    }
    alive = mbar_wait(bars + 8 * slot, phase, err);
    if (alive) {
      const uint32_t base = ring + slot * Cfg::kStageBytes + warp * Cfg::kHeadBytes;
      float s[PPS][NT][4], lv[PPS];
#pragma unroll
      for (int u = 0; u < PPS; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = -INFINITY;
        lv[u] = 0.f;
        if (u > 0 && p0 + u >= npages) continue;
        const uint32_t kb = base + u * 2 * Cfg::kPageBytes;
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
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
            for (int n = 0; n < NT; ++n) mma_f16_16816(acc[n], a0, a1, a2, a3, qb[n][c * 4 + w][0], qb[n][c * 4 + w][1]);
          }
        }
        const float f = f_q * power_of_two(scale_exponent(__shfl_sync(0xffffffffu, ek, (p0 + u) & 31)));
        lv[u] = static_cast<float>(scale_exponent(__shfl_sync(0xffffffffu, ev, (p0 + u) & 31)));
        const int t0 = start + (p0 + u) * kKvPage + tok;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[u][n][k] = t0 + (k >> 1) * 8 < L ? fmaf(acc[n][k], f, lv[u]) : -INFINITY;
        if (start + (p0 + u) * kKvPage + kKvPage > L) {
          // the last page: what lies behind the last token may be NaN, which a weight of zero does not undo.  Nothing loads into
          // this stage again.
          const uint32_t vb = kb + Cfg::kPageBytes;
          for (int t = L - (start + (p0 + u) * kKvPage); t < kKvPage; ++t)
            if (lane < D / 4) asm volatile("st.shared.b32 [%0], %1;" ::"r"(vb + piece(t, lane >> 2) + (lane & 3) * 4), "r"(0) : "memory");
          __syncwarp();
        }
      }

      // references: s is the exponent of the weight times its value scale
      bool over = false;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float t = fmaxf(s[0][n][k], s[0][n][k + 2]);
#pragma unroll
          for (int u = 1; u < PPS; ++u) t = fmaxf(t, fmaxf(s[u][n][k], s[u][n][k + 2]));
          top[n][k] = t;
          over |= t > m[n][k] + kKv8RefSlack;
        }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float t = top[n][k];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
            t = fmaxf(t, m[n][k]);
            const float a = t == -INFINITY ? 1.f : fast_ex2(m[n][k] - t);  // still nothing but scores of -inf: sums are zero
            m[n][k] = t;
            l[n][k] *= a;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              o[n][j][k] *= a;
              o[n][j][k + 2] *= a;
            }
          }
      }

#pragma unroll
      for (int u = 0; u < PPS; ++u) {
        if (u > 0 && p0 + u >= npages) continue;
        uint32_t pb[NT][2];
        const float iv = power_of_two(-static_cast<int>(lv[u]));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) p[k] = fast_ex2(s[u][n][k] - (m[n][k & 1] == -INFINITY ? 0.f : m[n][k & 1] - kKv8Lift));
          l[n][0] = fmaf(p[0] + p[2], iv, l[n][0]);
          l[n][1] = fmaf(p[1] + p[3], iv, l[n][1]);
          pb[n][0] = transpose_8x8(pack_f16x2(p[0], p[1]));
          pb[n][1] = transpose_8x8(pack_f16x2(p[2], p[3]));
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
          for (int n = 0; n < NT; ++n) {
            mma_f16_16816(o[n][2 * w], a[0][0], a[1][0], a[0][1], a[1][1], pb[n][0], pb[n][1]);
            mma_f16_16816(o[n][2 * w + 1], a[2][0], a[3][0], a[2][1], a[3][1], pb[n][0], pb[n][1]);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(bars + 8 * (STAGES + slot));
  }

  const int nsplits = (L + split_tokens - 1) / split_tokens;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float sum = l[n][k];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      const int head = 8 * n + 2 * tq + k;
      if (head >= heads) continue;
      if (nsplits == 1) {
        const float inv = 1.f / sum;
        uint32_t r[VB / 2];
#pragma unroll
        for (int j = 0; j < D / 16; ++j) r[j] = pack_bf16x2(o[n][j][k] * inv, o[n][j][k + 2] * inv);
        uint32_t* to = reinterpret_cast<uint32_t*>(out + (row0 + head) * D + g * VB);
#pragma unroll
        for (int j = 0; j < D / 16; j += 4) *reinterpret_cast<uint4*>(to + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
      } else {
        const size_t prow = (row0 + head) * max_splits + split;
        float* to = part_o + prow * D + g * VB;
#pragma unroll
        for (int j = 0; j < D / 16; j += 2)
          *reinterpret_cast<float4*>(to + 2 * j) = make_float4(o[n][j][k], o[n][j][k + 2], o[n][j + 1][k], o[n][j + 1][k + 2]);
        if (g == 0) part_ml[prow] = make_float2(m[n][k], sum);
      }
    }
#endif
}

// Joins the partials of one (row, query head): a CTA of four warps, warp w taking splits w, w + 4, ..., each lane D / 32
// columns.  The sums over splits are taken in a fixed order.  Without lengths every row has max_splits of them, some perhaps empty (their
// reference is -inf and their sums are not written).
template <int D>
__global__ void __launch_bounds__(128)
kv8_attn_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, const int* __restrict__ ctx_lens,
                     __nv_bfloat16* __restrict__ out, int num_q_heads, int max_splits, int split_tokens, int max_ctx) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int V = D / 32;
  __shared__ float o_sm[4][D];
  __shared__ float ml_sm[4][2];
  const size_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int n = max_splits;
  if (ctx_lens != nullptr) {
    const int L = min(max(ctx_lens[row / num_q_heads], 0), max_ctx);
    n = (L + split_tokens - 1) / split_tokens;
    if (n <= 1) return;  // written by its one CTA
  }
  const size_t base = row * max_splits;
  float top = -INFINITY, den = 0.f, acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  for (int s0 = warp; s0 < n; s0 += 16) {  // four splits of this warp at a time
    float v[4][V];
    float2 ml[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      ml[u] = make_float2(-INFINITY, 0.f);
      const int s = s0 + 4 * u;
      if (s < n) {
        ml[u] = part_ml[base + s];
        const float* from = part_o + (base + s) * D + lane * V;
#pragma unroll
        for (int j = 0; j < V; ++j) v[u][j] = from[j];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (ml[u].x == -INFINITY) v[u][j] = 0.f;
    const float t = fmaxf(fmaxf(top, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x));
    const float ref = t == -INFINITY ? 0.f : t;
    const float a = exp2f(top - ref);
    top = t;
    den *= a;
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] *= a;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float w = exp2f(ml[u].x - ref);
      den += w * ml[u].y;
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += w * v[u][j];
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) o_sm[warp][lane * V + j] = acc[j];
  if (lane == 0) {
    ml_sm[warp][0] = top;
    ml_sm[warp][1] = den;
  }
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= D) return;
  const float t = fmaxf(fmaxf(ml_sm[0][0], ml_sm[1][0]), fmaxf(ml_sm[2][0], ml_sm[3][0]));
  const float ref = t == -INFINITY ? 0.f : t;
  float num = 0.f, sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float x = exp2f(ml_sm[w][0] - ref);
    num += x * o_sm[w][d];
    sum += x * ml_sm[w][1];
  }
  out[row * D + d] = __float2bfloat16(num / sum);
}

int launch_kv8_join(int head_dim, const AttnWorkspace& w, const int* ctx_lens, void* out, int rows, int hq, int max_splits, int split_tokens,
                    int max_ctx, cudaStream_t st) {
  B200_CUDA(launch_overlapped(head_dim == 128 ? kv8_attn_join_kernel<128> : kv8_attn_join_kernel<64>, dim3(rows * hq), dim3(128), 0, st, w.o,
                              w.ml, ctx_lens, static_cast<__nv_bfloat16*>(out), hq, max_splits, split_tokens, max_ctx));
  return 0;
}

// Tokens per split where the caller names none.  Few rows: so that all CTAs are there at once and the GPU is full, but no fewer than 64
// tokens; a full batch: 512, long enough that partials cost little and short enough that rows of different lengths even out.
static int kv8_split_tokens(int batch, int head_ctas, int max_pages, int sms) {
  const long long tokens = static_cast<long long>(max_pages) * kKvPage;
  const long long ctas = 2ll * sms / (static_cast<long long>(batch) * head_ctas);
  if (ctas < 2) return 512;
  const long long split = ((tokens + ctas - 1) / ctas + kKvPage - 1) / kKvPage * kKvPage;
  return static_cast<int>(split < 64 ? 64 : split > 512 && batch > 8 ? 512 : split);
}

struct Kv8Plan {
  int hkv, nt, slices, split, max_splits;
};
static int kv8_plan(int batch, int hq, int hkv, int max_pages, int split_tokens, Kv8Plan* p) {
  const int group = hq / hkv;
  p->hkv = hkv % 8 == 0 ? 8 : hkv % 4 == 0 ? 4 : hkv % 2 == 0 ? 2 : 1;
  p->nt = group > 8 ? 2 : 1;
  p->slices = (group + 15) / 16;
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc) return rc;
  p->split = split_tokens > 0 ? split_tokens : kv8_split_tokens(batch, hkv / p->hkv * p->slices, max_pages, sms);
  p->max_splits = static_cast<int>((static_cast<long long>(max_pages) * kKvPage + p->split - 1) / p->split);
  return 0;
}

struct Kv8Args {
  const void *q, *k_pool, *v_pool, *k_scale, *v_scale;
  const int *table, *ctx;
  void* out;
  AttnWorkspace w;
  int batch, hq, hkv, num_blocks, max_pages;
  float scale;
  Kv8Plan plan;
  cudaStream_t st;
};

template <int D, int HKV, int NT, int PPS, int STAGES, int CTAS>
static int launch_kv8_decode(const Kv8Args& a) {
  using Cfg = Kv8Cfg<D, HKV, NT, PPS, STAGES>;
  CUtensorMap kmap, vmap;
  const uint64_t rows = static_cast<uint64_t>(a.num_blocks) * a.hkv * (Cfg::kHeadBytes / 128);
  int rc = get_tensor_map_2d(a.k_pool, rows, 128, 1, Cfg::kPageBytes / 128, 128, &kmap);
  if (rc) return rc;
  rc = get_tensor_map_2d(a.v_pool, rows, 128, 1, Cfg::kPageBytes / 128, 128, &vmap);
  if (rc) return rc;
  auto kernel = kv8_attn_decode_kernel<D, HKV, NT, PPS, STAGES, CTAS>;
  rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), Cfg::kSmemBytes);
  if (rc) return rc;
  B200_CUDA(launch_overlapped(kernel, dim3(a.batch, a.plan.max_splits, a.hkv / HKV * a.plan.slices), dim3(Cfg::kThreads), Cfg::kSmemBytes,
                              a.st, kmap, vmap, static_cast<const __nv_bfloat16*>(a.q), static_cast<const uint8_t*>(a.k_scale),
                              static_cast<const uint8_t*>(a.v_scale), a.table, a.ctx, a.w.o, a.w.ml, static_cast<__nv_bfloat16*>(a.out),
                              a.w.err, a.hq, a.hkv, a.num_blocks, a.max_pages, a.plan.split, a.plan.max_splits,
                              a.scale * 1.4426950408889634f));
  if (a.plan.max_splits > 1)
    return launch_kv8_join(D, a.w, a.ctx, a.out, a.batch, a.hq, a.plan.max_splits, a.plan.split, a.max_pages * kKvPage, a.st);
  return 0;
}

template <int D, int NT>
static int launch_kv8_heads(const Kv8Args& a) {
  switch (a.plan.hkv) {
    case 1: return launch_kv8_decode<D, 1, NT, 2, 4, 6>(a);
    case 2: return launch_kv8_decode<D, 2, NT, 2, 4, NT == 1 ? 4 : 3>(a);
    case 4: return launch_kv8_decode<D, 4, NT, 2, 3, 2>(a);
    default: return launch_kv8_decode<D, 8, NT, 1, D == 128 ? 6 : 8, 1>(a);
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
  if (kv8_plan(batch, num_q_heads, num_kv_heads, max_pages_per_seq, split_tokens, &p)) return 256;
  return carve(nullptr, batch, num_q_heads, head_dim, p.max_splits).bytes;
}

extern "C" int b200_kv8_attn_decode(const void* q, const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale,
                                    const int32_t* block_table, const int32_t* ctx_lens, void* out, void* workspace,
                                    size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads, int head_dim, int num_blocks,
                                    int max_pages_per_seq, float scale, int split_tokens, void* stream) {
  B200_REQUIRE(q && k_pool && v_pool && k_scale && v_scale && block_table && ctx_lens && out && workspace, "kv8_attn_decode: null pointer");
  int rc = check_kv8("kv8_attn_decode", batch, num_q_heads, num_kv_heads, head_dim, num_blocks, max_pages_per_seq, q, k_pool, v_pool, out, scale);
  if (rc) return rc;
  B200_REQUIRE(split_tokens >= 0 && split_tokens % kKvPage == 0, "kv8_attn_decode: split_tokens %d not a multiple of %d", split_tokens, kKvPage);
  rc = check_device(nullptr);
  if (rc) return rc;
  Kv8Args a{q, k_pool, v_pool, k_scale, v_scale, block_table, ctx_lens, out, {}, batch, num_q_heads, num_kv_heads, num_blocks,
            max_pages_per_seq, scale, {}, as_stream(stream)};
  rc = kv8_plan(batch, num_q_heads, num_kv_heads, max_pages_per_seq, split_tokens, &a.plan);
  if (rc) return rc;
  B200_REQUIRE(a.plan.max_splits <= 65535 && num_kv_heads / a.plan.hkv * a.plan.slices <= 65535 &&
                   static_cast<long long>(batch) * num_q_heads < (1ll << 31),
               "kv8_attn_decode: grid too large");
  a.w = carve(workspace, batch, num_q_heads, head_dim, a.plan.max_splits);
  if (workspace_bytes < a.w.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) {
    set_detail("kv8_attn_decode: workspace of %zu bytes at %p, %zu on a 16-byte boundary are needed", workspace_bytes, workspace, a.w.bytes);
    return -kErrWorkspace;
  }
  if (head_dim == 128) return a.plan.nt == 1 ? launch_kv8_heads<128, 1>(a) : launch_kv8_heads<128, 2>(a);
  return a.plan.nt == 1 ? launch_kv8_heads<64, 1>(a) : launch_kv8_heads<64, 2>(a);
}
