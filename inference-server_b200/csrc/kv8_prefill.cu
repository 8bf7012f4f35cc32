// Causal attention of a chunk of prompt tokens over the 8-bit page cache (kv8.cuh) on the tcgen05 tensor cores (sm_100a), head_dim 64 or 128,
// up to 128 query heads per kv head: the counterpart of paged_prefill_pairs.cu, which reads 16-bit pools and has the same shape of
// work (rows of the score matrix, tiles of 128 keys, two tiles of rows in flight per CTA), and replaces the same steps of the
// reference (src/inference_server/kv_cache/hf_format.py:21-45 + src/inference_server/backends/torch_backend.py:107-147).
//
// Mathematics as in kv8_decode.cu: a value's scale is taken into its weight's exponent, keys' scales multiply the scores.
//
//   S = Q K^T   from the 8-bit keys as they are, kind::f8f6f4 with both operands K-major in shared memory.  A query is the sum of two
//               e4m3 numbers, hi = the nearest and lo = what is left: bf16 has 8 bits, hi takes 4, and lo needs 4 more, so the sum is exact
//               but for the ends of the range (rows are brought to a top in (224, 448]; a query 2^-7 of the row's largest
//               or smaller loses bits below 2^-19 of it).  Two products of twice the rate cost what one in 16 bits does, and keys need
//               neither conversion nor room in 16 bits.
//   P V         kind::f16: weights are f16 in TMEM (11 bits), values are converted to f16 (exactly) by four warps and
//               stored as MN-major swizzled tiles.  A conversion serves both tiles of rows.
//
//   grid     (CTAs of tiles, late ones first) x splits of the keys x kv heads.  The keys are split where the tiles alone leave SMs idle; fp32
//            partials are then joined by kv8_attn_join_kernel.
//   warp 0   producer: per key tile, 8 pages of keys by TMA into three stages and 8 of values as plain bulk copies into two.  It does nothing
//            else: when it converted values too, it asked for keys so late that S waited for memory.
//   warp 1   S issuer (one thread), warp 2 P V issuer (one thread).
//   warps 4-7    a quarter of a tile's values each: 16 bytes of a row to 16 f16 numbers; zero for what lies behind the last token, where a page
//            may hold NaN, and for NaN in a tile that some row sees in part; what they took out there they put into the rows that see it, at the
//            end.  One such warp per scheduler: with two of them on two, the softmax warps beside them held up the others.
//   warps 8-11, 12-15   first the queries of both tiles (bf16 to hi and lo, a row's top by shuffles), then the softmax of tile 0 and of tile 1,
//            a thread per score row; the scales of a key tile's 8 pages come to each warp by its own lanes, two key tiles
//            ahead (ids) and one (scales), and from a corner of shared memory to all lanes, put there once the tile before is done, so that
//            nothing lies between a tile's scores and their room being free again.  (Two threads per row, 16 softmax warps, and one
//            predicate per key tile between them: 296 us where a thread per row took 276.)
//   A CTA with one tile of rows takes every second key tile of it on the other tile's warps, with an accumulator and reference of their own,
//   and adds the two up at the end.
//
// Bound by the softmax: a key tile of a CTA with two tiles of rows takes about 3650 cycles, in which each scheduler issues 2000 instructions of its
// three busy warps, the special-function units need 2048 for the exponentials and the tensor core is busy for 1024.  Dependent steps
// (scores, maximum, exponentials, weights) leave the rest; halves of 64 keys by turns, the next one fetched meanwhile, made the steps more
// and not shorter (359 us), and so did a quarter of the exponentials by a polynomial (271).  32 / 4 heads of 128, in graphs of calls: 2048 tokens 50
// to 53 us, 1024 behind 14336 233 to 249 us by the clock (1.07 to 1.00 PFLOP/s; 202 over 16-bit pools, whose values need no conversion), 17 behind
// 14001 (64 / 4 heads) 27 us.  Heads of 64 have half the products for the same exponentials: 2048 tokens 26 us with 16 / 2 heads, 1024 behind
// 14336 127 us with 16 / 2 and 221 with 32 / 4, where exponentials alone are 54 and 108.
//
// Every mbarrier wait is bounded; a wait that runs out records kErrDevWaitTimeout and the thread stops waiting but keeps the loop
// structure, so the kernel ends.
// TMEM: O0, O1, S 128 columns each, P0, P1 64 (two f16 per column).

#include <algorithm>

#include "host.h"
#include "kv8.cuh"
#include "prefill_tc.cuh"

namespace b200 {

constexpr int kKv8SoftmaxWarps = 8;
constexpr int kKv8PrefillThreads = (8 + kKv8SoftmaxWarps) * 32;
constexpr int kKv8KStages = 3;
constexpr float kKv8PLift = 6.f;  // weights are taken times 2^6, at most 2^14 with the slack of kTcRescaleLog2

template <int D>
struct Kv8PrefillCfg {
  static constexpr int kTile8 = kTcKeys * D;                 // bytes of 128 rows in 8 bits
  static constexpr int kTile16 = 2 * kTile8;
  static constexpr int kQ = 0;                                // [2 tiles][hi, lo]
  static constexpr int kK = kQ + 4 * kTile8;                   // [kKv8KStages]
  static constexpr int kRaw = kK + kKv8KStages * kTile8;       // [2 stages] values as they are
  static constexpr int kV = kRaw + 2 * kTile8;                 // [2 stages] values in f16
  static constexpr int kScales = kV + 2 * kTile16;             // [8 warps][2][8 pages] float4
  static constexpr int kRowScale = kScales + 8 * 2 * 8 * 16;   // [2 tiles][128] float
  static constexpr int kSums = kRowScale + 2 * 128 * 4;        // the same
  static constexpr int kRefs = kSums + 2 * 128 * 4;            // the same
  static constexpr int kBars = kRefs + 2 * 128 * 4;
  static constexpr int kSmemBytes = kBars + 256 + 1024 /* alignment slack */;
};

// Descriptor of a K-major operand tile in 8 bits: rows of 128 bytes with 128-byte swizzle, or of 64 bytes with 64-byte swizzle.
template <int D>
__device__ __forceinline__ uint64_t desc_k8(uint32_t smem_addr) {
  if constexpr (D == 128) return umma_desc_k128(smem_addr);
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1) << 16;           // leading byte offset (unused)
  d |= static_cast<uint64_t>(512 >> 4) << 32;    // groups of 8 rows
  d |= static_cast<uint64_t>(1) << 46;           // descriptor version (sm_100)
  d |= static_cast<uint64_t>(4) << 61;           // 64-byte swizzle
  return d;
}
// f16 x f16 -> f32, A K-major, B MN-major.
__host__ __device__ constexpr uint32_t idesc_f16_mn(uint32_t m, uint32_t n) {
  return (1u << 4) | (1u << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// D[tmem] (+)= A[tmem] * B[smem], f16: a lane of A is a row, a 32-bit column two neighbouring K elements.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float max_of_3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// One warp's quarter of a tile of values, rows row0 .. row0 + 31, to f16; those from `rows` on hold no tokens and become zero (a page may hold
// NaN there).  A lane takes 16 bytes of a row at a time, which become two pieces of a swizzled row.  For head_dim 128 a quarter warp
// takes the first half of one row and the second half of the next: its loads are in different banks, and so are its stores,
// whose pieces are XORed with numbers that differ in bit 0.  Addresses are a register and a constant: with address arithmetic in a loop
// 1024 tokens behind 14336 took 234 us instead of 231, for these warps share their schedulers' issue slots with the softmax warps.  (By the
// same token, integer arithmetic instead of conversions, 10 instructions for 2 per four numbers, took 250 us.)
template <int D>
__device__ __forceinline__ void values_to_f16(uint32_t from, uint32_t to, int row0, int rows, int lane) {
  constexpr int kPieces = D / 16, kRowsAt = 32 / kPieces;  // pieces of a row; rows that the warp takes at a time
  constexpr uint32_t kAtomGroup = D / 64 * 1024;           // 8 rows of f16
  if (rows < row0 + kTcKeys / 4) {
    for (int i = max(rows, row0) * kPieces + lane; i < (row0 + kTcKeys / 4) * kPieces; i += 32)
      asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(from + i * 16), "r"(0) : "memory");
    __syncwarp();
  }
  const int odd = (lane >> 2) & 1;
  const int c = D == 128 ? (lane & 3) + 4 * (((lane >> 3) & 1) ^ odd) : lane & 3;
  const int lr = D == 128 ? 2 * (lane >> 4) + odd : lane >> 2;
  const uint32_t src = from + (row0 + lr) * D + c * 16;
  const uint32_t row = to + (row0 >> 3) * kAtomGroup + (c >> 2) * 1024;
  constexpr int kOdd = kRowsAt == 4 ? 2 : 1;  // rows of a lane within a group of 8
  uint32_t put[kOdd][2];
#pragma unroll
  for (int u = 0; u < kOdd; ++u)
#pragma unroll
    for (int k = 0; k < 2; ++k) put[u][k] = row + swz128(lr + u * kRowsAt, ((2 * c) & 7) + k);
  constexpr int kSteps = kTcKeys / 4 / kRowsAt;
  uint32_t w[4];
  lds_words<16>(src, w);
#pragma unroll
  for (int r = 0; r < kSteps; ++r) {
    uint32_t a[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) e4m3x4_to_f16(w[k], a[2 * k], a[2 * k + 1]);
    if (r + 1 < kSteps) lds_words<16>(src + (r + 1) * kRowsAt * D, w);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(put[r % kOdd][k] + r / kOdd * kAtomGroup), "r"(a[4 * k]), "r"(a[4 * k + 1]), "r"(a[4 * k + 2]),
                   "r"(a[4 * k + 3])
                   : "memory");
  }
  fence_proxy_async();  // the tensor core reads the tile, and the next copy writes the stage, through the async proxy
  __syncwarp();
}

// The NaN codes of four e4m3 numbers: the top bit of each such byte.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Makes NaN zero in the first `rows` rows of a warp's quarter of a raw tile; whether there was any.
template <int D>
__device__ __forceinline__ bool nan_to_zero(uint32_t from, int rows, int lane) {
  bool any = false;
#pragma unroll
  for (int i0 = 0; i0 < kTcKeys / 4 * (D / 16); i0 += 32) {
    const int i = i0 + lane;
    if (i >= rows * (D / 16)) continue;
    uint32_t w[4], nan[4];
    lds_words<16>(from + i * 16, w);
#pragma unroll
    for (int k = 0; k < 4; ++k) nan[k] = nan_codes(w[k]);
    if (nan[0] | nan[1] | nan[2] | nan[3]) {
      any = true;
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] &= ~((nan[k] >> 7) * 0xffu);
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(from + i * 16), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
  }
  __syncwarp();  // other lanes read what this one wrote
  return __any_sync(0xffffffffu, any);
}

template <int D>
__global__ void __launch_bounds__(kKv8PrefillThreads, 1)
kv8_attn_prefill_kernel(const __grid_constant__ CUtensorMap k_map, const uint8_t* __restrict__ v_pool, const uint8_t* __restrict__ k_scale,
                        const uint8_t* __restrict__ v_scale, const int* __restrict__ table_row, const __nv_bfloat16* __restrict__ q,
                        __nv_bfloat16* __restrict__ out, float* __restrict__ part_o, float2* __restrict__ part_ml, int* __restrict__ err,
                        int num_tokens, int first_pos, int num_q_heads, int num_kv_heads, int num_blocks, float scale_log2, int pairs,
                        int splits, int split_tiles) {
#ifdef B200_DEVICE_OK
  using Cfg = Kv8PrefillCfg<D>;
  constexpr int kPageBytes8 = kKvPage * D, kPageBytes16 = 2 * kPageBytes8;
  constexpr uint32_t kAtomGroup = D / 64 * 1024;  // 8 rows of f16
  const int gr = num_q_heads / num_kv_heads;
  const int QT = kTcRows / gr;  // prompt positions per tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + Cfg::kBars;
  const uint32_t bar_kfull = bars, bar_kempty = bars + 32;        // [3 stages] each
  const uint32_t bar_rawfull = bars + 64, bar_rawempty = bars + 80;  // [2 stages] each
  const uint32_t bar_vfull = bars + 96, bar_vempty = bars + 112;
  const uint32_t bar_q = bars + 128;                              // Q written
  const uint32_t bar_sempty = bars + 136;                         // S read
  const uint32_t bar_sfull = bars + 144;                          // [2 tiles] S written, for this tile
  const uint32_t bar_odone = bars + 160;                          // [2 tiles] O += P V finished
  const uint32_t bar_pfull = bars + 176;                          // [2 tiles][2 halves of 64 keys] P written, O rescaled
  uint32_t* tmem_base_sm = reinterpret_cast<uint32_t*>(base_ptr + Cfg::kBars + 240);
  volatile int* nan_sm = reinterpret_cast<int*>(base_ptr + Cfg::kBars + 244);  // a NaN value was taken out of a tile that some row sees in part
  float* row_scale = reinterpret_cast<float*>(base_ptr + Cfg::kRowScale);
  float* sums = reinterpret_cast<float*>(base_ptr + Cfg::kSums);
  float* refs = reinterpret_cast<float*>(base_ptr + Cfg::kRefs);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 32) tma_prefetch_desc(&k_map);
  if (threadIdx.x == 0) {
    *nan_sm = 0;
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar_rawfull + 8 * s, 1);
      mbar_init(bar_rawempty + 8 * s, 4);
      mbar_init(bar_vfull + 8 * s, 4);
      mbar_init(bar_vempty + 8 * s, 1);
      mbar_init(bar_sfull + 8 * s, 1);
      mbar_init(bar_odone + 8 * s, 1);
      mbar_init(bar_pfull + 16 * s, 4);
      mbar_init(bar_pfull + 16 * s + 8, 4);
    }
    for (int s = 0; s < kKv8KStages; ++s) {
      mbar_init(bar_kfull + 8 * s, 1);
      mbar_init(bar_kempty + 8 * s, 1);
    }
    mbar_init(bar_q, kKv8SoftmaxWarps);
    mbar_init(bar_sempty, 4);
    fence_mbar_init();
    fence_proxy_async();
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_base_sm), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_sm;
  const uint32_t tmem_o = tmem_base, tmem_s = tmem_base + 2 * kTcKeys, tmem_p = tmem_s + kTcKeys;  // O0, O1, S, P0, P1
  // late positions first, all splits and kv heads of them side by side; the first `pairs` CTAs of a head take two tiles of rows each
  const int h = static_cast<int>(blockIdx.x) % num_kv_heads, rest = static_cast<int>(blockIdx.x) / num_kv_heads;
  const int split = rest % splits, cta = rest / splits;
  const int own = cta < pairs ? 2 : 1;
  const int t0 = ((num_tokens + QT - 1) / QT - own - cta - min(cta, pairs)) * QT;
  const int t_end = min(t0 + own * QT, num_tokens);
  const int last_pos = first_pos + t_end - 1;
  // key tiles of this CTA: kt0 ..; a tile of rows takes the first n_of[] of them, or, alone, accumulator 0 the even and 1 the odd ones
  const int kt0 = split * split_tiles;
  const int n_tiles = max(0, min(last_pos / kTcKeys + 1, kt0 + split_tiles) - kt0);
  int n_of[2] = {(n_tiles + 1) / 2, n_tiles / 2};
  if (own == 2) {
    n_of[0] = max(0, min(n_tiles, (first_pos + t0 + QT - 1) / kTcKeys + 1 - kt0));
    n_of[1] = n_tiles;
  }
  const int stride = own == 2 ? 1 : 2;  // key tiles from one of an accumulator to its next
  const int last_page = last_pos / kKvPage;

  grid_dep_wait();  // set-up done; Q and this chunk's pages come from the kernels before
  grid_dep_launch();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      // ------------------------------------------------- pages ------
      // Lane i of the first 8 owns page i of a tile's keys, of the second 8 that of its values.
      const int pg = lane & 7;
      bool alive = true;
      int next = __ldg(table_row + min(kt0 * kTcPages + pg, last_page)), ks = 0, kphase = 1;
#pragma unroll 1
      for (int j = 0; j < n_tiles && alive; ++j) {
        // the last page stands in for those behind it, so that every stage is the same number of bytes
        int page = next;
        next = __ldg(table_row + min((kt0 + j + 1) * kTcPages + pg, last_page));
        if (page < 0 || page >= num_blocks) {
          set_error(err, kErrDevBadBlockId);
          page = 0;
        }
        const size_t cell = static_cast<size_t>(page) * num_kv_heads + h;
        alive = mbar_wait_warp(bar_kempty + 8 * ks, kphase, err);
        if (!alive) break;
        if (lane == 0) mbar_arrive_expect_tx(bar_kfull + 8 * ks, Cfg::kTile8);
        __syncwarp();
        if (lane < kTcPages)
          tma_load_2d(base + Cfg::kK + ks * Cfg::kTile8 + pg * kPageBytes8, &k_map, bar_kfull + 8 * ks, 0, static_cast<int>(cell) * kKvPage);
        if (++ks == kKv8KStages) {
          ks = 0;
          kphase ^= 1;
        }
        const int st = j & 1;
        alive = mbar_wait_warp(bar_rawempty + 8 * st, ((j >> 1) & 1) ^ 1, err);
        if (!alive) break;
        if (lane == 0) mbar_arrive_expect_tx(bar_rawfull + 8 * st, Cfg::kTile8);
        __syncwarp();
        if (lane >= 8 && lane < 16)
          bulk_load(base + Cfg::kRaw + st * Cfg::kTile8 + pg * kPageBytes8, v_pool + cell * kPageBytes8, kPageBytes8, bar_rawfull + 8 * st);
      }
    } else if (warp == 1) {
      // ------------------------------------------------- S = Q K^T ------
      if (elect_one()) {
        constexpr uint32_t idesc_s = umma_idesc_f8(kTcRows, kTcKeys);
        bool alive = true;
        uint32_t n = 0, st = 0, phase = 0;
#pragma unroll 1
        for (int j = 0; j < n_tiles && alive; ++j) {
          alive = mbar_wait(bar_kfull + 8 * st, phase, err);
          if (j == 0 && alive) alive = mbar_wait(bar_q, 0, err);
          const uint64_t b0 = desc_k8<D>(base + Cfg::kK + st * Cfg::kTile8);
#pragma unroll 1
          for (int t = 0; t < 2; ++t) {
            // none of this tile's rows sees these keys, or they are the other accumulator's
            if (own == 2 ? j >= (t ? n_of[1] : n_of[0]) : (j & 1) != t) continue;
            if (n > 0 && alive) alive = mbar_wait(bar_sempty, (n & 1) ^ 1, err);  // nothing has been written yet at first
            if (!alive) break;
            ++n;
            tc_fence_after();
            const uint64_t a0 = desc_k8<D>(base + Cfg::kQ + 2 * (own == 2 ? t : 0) * Cfg::kTile8);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {  // hi, then lo
              constexpr int kSteps = D / 32;
              tc_mma_f8(tmem_s, a0 + (k / kSteps * (Cfg::kTile8 >> 4) + k % kSteps * 2), b0 + k % kSteps * 2, idesc_s, k > 0 ? 1u : 0u);
            }
            tc_commit(bar_sfull + 8 * t);
          }
          tc_commit(bar_kempty + 8 * st);
          if (++st == kKv8KStages) {
            st = 0;
            phase ^= 1;
          }
        }
      }
    } else if (warp == 2 && elect_one()) {
      // ------------------------------------------------- O += P V ------
      constexpr uint32_t idesc_o = idesc_f16_mn(kTcRows, D);
      bool alive = true;
#pragma unroll 1
      for (int j = 0; j < n_tiles && alive; ++j) {
        const int st = j & 1;
        alive = mbar_wait(bar_vfull + 8 * st, (j >> 1) & 1, err);
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
          if (own == 2 ? j >= (t ? n_of[1] : n_of[0]) : (j & 1) != t) continue;
          const int i = own == 2 ? j : j >> 1;
          const uint64_t b0 = umma_desc_mn128(base + Cfg::kV + st * Cfg::kTile16, 1024, kAtomGroup);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (alive) alive = mbar_wait(bar_pfull + 16 * t + 8 * half, i & 1, err);
            if (!alive) break;
            tc_fence_after();
#pragma unroll
            for (int kk = half * 4; kk < half * 4 + 4; ++kk)  // 16 keys each
              mma_f16_ts(tmem_o + t * kTcKeys, tmem_p + t * 64 + kk * 8, b0 + kk * (kPageBytes16 >> 4), idesc_o, (i > 0 || kk > 0) ? 1u : 0u);
          }
          tc_commit(bar_odone + 8 * t);
        }
        tc_commit(bar_vempty + 8 * st);
      }
    }
  } else if (warp < 8) {
    // ------------------------------------------------- V in f16 ------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    // Key tiles from this one on hold keys that some row of the CTA does not see.  A product takes a weight of zero times such a key's value, and a
    // NaN among the values would spoil rows ahead of it: they are taken out of these tiles, and put back by the rows that see them.
    const int edge_tile = (first_pos + t0 + 1) / kTcKeys;
    bool alive = true;
#pragma unroll 1
    for (int j = 0; j < n_tiles && alive; ++j) {
      const int st = j & 1;
      alive = mbar_wait_warp(bar_rawfull + 8 * st, (j >> 1) & 1, err) && mbar_wait_warp(bar_vempty + 8 * st, ((j >> 1) & 1) ^ 1, err);
      if (!alive) break;
      if (kt0 + j >= edge_tile) {
        const int row0 = (warp - 4) * (kTcKeys / 4), rows = min(max(last_pos - (kt0 + j) * kTcKeys + 1 - row0, 0), kTcKeys / 4);
        if (nan_to_zero<D>(base + Cfg::kRaw + st * Cfg::kTile8 + row0 * D, rows, lane)) *nan_sm = 1;
      }
      values_to_f16<D>(base + Cfg::kRaw + st * Cfg::kTile8, base + Cfg::kV + st * Cfg::kTile16, (warp - 4) * (kTcKeys / 4),
                       last_pos - (kt0 + j) * kTcKeys + 1, lane);
      if (lane == 0) {
        mbar_arrive(bar_vfull + 8 * st);
        mbar_arrive(bar_rawempty + 8 * st);
      }
    }
    // Once the rows are written, those that see such a NaN get it: a thread finds a column's first and goes through the rows from there on.  (Two
    // plain loops: loops within loops, a row a thread, took the compiler's care from the softmax warps' loop although they hardly ever run, 229 ->
    // 245 us for 1024 tokens behind 14336, here, in an idle warp or behind the rows' own stores alike.)
    __syncwarp();
    asm volatile("bar.sync 2, 384;" ::: "memory");
    const int c = threadIdx.x - 128;
    if (*nan_sm && c < D) {
      int x = max(edge_tile, kt0) * kTcKeys;
      const int end = min(last_pos + 1, (kt0 + n_tiles) * kTcKeys);
#pragma unroll 1
      for (; x < end; ++x) {
        const int page = __ldg(table_row + x / kKvPage);
        const size_t cell = static_cast<size_t>(page < 0 || page >= num_blocks ? 0 : page) * num_kv_heads + h;
        if ((__ldg(v_pool + cell * kPageBytes8 + x % kKvPage * D + c) & 0x7f) == 0x7f) break;
      }
      const int rows = x < end ? (t_end - t0) * gr : 0;
#pragma unroll 1
      for (int i = max(x - first_pos - t0, 0) * gr; i < rows; ++i) {
        const size_t oidx = static_cast<size_t>(t0 + i / gr) * num_q_heads + h * gr + i % gr;
        if (splits > 1) part_o[(oidx * splits + split) * D + c] = NAN;
        else out[oidx * D + c] = __ushort_as_bfloat16(0x7fffu);
      }
    }
  } else {
    // -------------------------------------------------------- softmax ------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int t = (warp - 8) >> 2;           // tile of rows, or accumulator
    const int quarter = warp & 3;            // TMEM lanes this warp may touch
    const int r = quarter * 32 + lane;       // score row
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_acc = tmem_s + lane_off, o_acc = tmem_o + t * kTcKeys + lane_off, p_tm = tmem_p + t * 64 + lane_off;
    const uint32_t sfull = bar_sfull + 8 * t, odone = bar_odone + 8 * t, pfull = bar_pfull + 16 * t;
    const int tile = own == 2 ? t : 0, tt0 = t0 + tile * QT, rt = r / gr, n_own = t ? n_of[1] : n_of[0];
    const int pos = first_pos + min(tt0 + rt, min(tt0 + QT, num_tokens) - 1);  // the last key this row may see
    const int first_tile = kt0 + (own == 2 ? 0 : t);

    // Scales of the pages of a key tile: lane i of 8 asks for those of page i.
    const int pg = lane & 7;
    // (Loads that stay where they are written: left to itself the compiler moves them down to where they are needed.)
    auto page_id = [&](int i) {
      int id;
      asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(id) : "l"(table_row + min((first_tile + i * stride) * kTcPages + pg, last_page)));
      return id;
    };
    int id = page_id(0), kb, vb;
    auto ask_scales = [&]() {
      const size_t cell = static_cast<size_t>(id < 0 || id >= num_blocks ? 0 : id) * num_kv_heads + h;  // the producer reports it
      asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(kb) : "l"(k_scale + cell));
      asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(vb) : "l"(v_scale + cell));
    };
    ask_scales();
    id = page_id(1);

    // Q tiles: 32 numbers of a row per thread and step, the next step's on their way.  (8 numbers, with three times the shuffles and a
    // quarter of the work side by side, took 5200 cycles a tile.)  One loop over the steps of both tiles: code that runs once has to be
    // fetched first.
    {
      constexpr int kOfRow = D / 32, kRows = 256 / kOfRow, kSteps = kTcRows / kRows;  // threads of a row; rows of a step; steps of a tile
      const int ch = threadIdx.x % kOfRow, qr0 = (threadIdx.x - 256) / kOfRow;
      uint4 v[4];
      auto load = [&](int step) {
        const int qr = step % kSteps * kRows + qr0, qt_l = qr / gr, tok = t0 + step / kSteps * QT + qt_l;
        const bool there = step < own * kSteps && qt_l < QT && tok < num_tokens;
        const uint4* from = reinterpret_cast<const uint4*>(q + (static_cast<size_t>(tok) * num_q_heads + h * gr + (qr - qt_l * gr)) * D + ch * 32);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[k] = make_uint4(0u, 0u, 0u, 0u);
          if (there) v[k] = from[k];
        }
      };
      load(0);
#pragma unroll 1
      for (int step = 0; step < own * kSteps; ++step) {
        const int u = step / kSteps, qr = step % kSteps * kRows + qr0;
        uint32_t x[16];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[4 * k] = v[k].x, x[4 * k + 1] = v[k].y, x[4 * k + 2] = v[k].z, x[4 * k + 3] = v[k].w;
        load(step + 1);
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) top = __vmaxu2(top, x[k] & 0x7fff7fffu);
        top = max(top >> 16, top & 0xffffu) << 16;
#pragma unroll
        for (int o = 1; o < kOfRow; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        // the exponent that brings the row's top to (224, 448]; tiny rows may stay below, a row with an infinity is all NaN
        const int e = max(static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), -100);
        const float by = top < 0x7f800000u ? power_of_two(-e) : NAN;
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          uint32_t pair[2], rest_of[2];
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const float a = __uint_as_float(x[2 * k + p] << 16) * by, b = __uint_as_float(x[2 * k + p] & 0xffff0000u) * by;
            pair[p] = to_e4m3x2(a, b);
            uint32_t near, unused;
            e4m3x4_to_f16(pair[p], near, unused);
            const float2 n2 = __half22float2(*reinterpret_cast<const __half2*>(&near));
            rest_of[p] = to_e4m3x2(a - n2.x, b - n2.y);
          }
          hi[k] = pair[0] | pair[1] << 16;
          lo[k] = rest_of[0] | rest_of[1] << 16;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t at = D == 128 ? (qr >> 3) * 1024 + swz128(qr & 7, 2 * ch + k) : qr * 64 + (((2 * ch + k) ^ ((qr >> 1) & 3)) << 4);
          uint8_t* to = base_ptr + Cfg::kQ + 2 * u * Cfg::kTile8 + at;
          *reinterpret_cast<uint4*>(to) = make_uint4(hi[4 * k], hi[4 * k + 1], hi[4 * k + 2], hi[4 * k + 3]);
          *reinterpret_cast<uint4*>(to + Cfg::kTile8) = make_uint4(lo[4 * k], lo[4 * k + 1], lo[4 * k + 2], lo[4 * k + 3]);
        }
        if (ch == 0) row_scale[u * kTcRows + qr] = fmaxf(scale_log2 * power_of_two(min(e, 120)), 0x1p-90f);
      }
    }
    fence_proxy_async();  // the tensor core reads Q through the async proxy
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (lane == 0) mbar_arrive(bar_q);
    const float f_q = row_scale[tile * kTcRows + r];
    float4* scales = reinterpret_cast<float4*>(base_ptr + Cfg::kScales) + (warp - 8) * 16;

    float m_run = -INFINITY, l_run = 0.f;
    bool alive = true, s_ready = false;
    int kbase = first_tile * kTcKeys;
    auto put_scales = [&](int i) {
      const int ev = scale_exponent(vb);
      if (lane < 8) scales[(i & 1) * 8 + pg] = make_float4(power_of_two(scale_exponent(kb)), static_cast<float>(ev), power_of_two(-ev), 0.f);
      __syncwarp();
      ask_scales();  // of the next key tile; past the last one those of the last page
      id = page_id(i + 2);
    };
    put_scales(0);
#pragma unroll 1
    for (int i = 0; i < n_own; ++i, kbase += stride * kTcKeys) {
      if (!__all_sync(0xffffffffu, s_ready) && alive) alive = mbar_wait(sfull, i & 1, err);
      tc_fence_after();
      float s[128];
      {
        uint32_t (&raw)[4][32] = *reinterpret_cast<uint32_t(*)[4][32]>(s);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_acc + c * 32, raw[c]);
      }
      // while S is on its way: the pages' scales, and the next key tile's are asked for
      const float4* sc = scales + (i & 1) * 8;
      float f[8], lv[8];
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float2 w = *reinterpret_cast<const float2*>(sc + p);
        f[p] = f_q * w.x;
        lv[p] = w.y;
      }
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_sempty);  // S is the other tile's now
      if (kbase + kTcKeys - 1 > pos) {  // the causal edge runs through this row
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (kbase + c > pos) s[c] = -INFINITY;
      }
      // a scale is positive: the largest product of a page is that of its largest score
      float m_new = m_run;
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float* x = s + 16 * p;
        const float a = max_of_3(max_of_3(x[0], x[1], x[2]), x[3], x[4]), b = max_of_3(max_of_3(x[5], x[6], x[7]), x[8], x[9]);
        const float c = max_of_3(max_of_3(x[10], x[11], x[12]), x[13], x[14]);
        m_new = fmaxf(m_new, fmaf(max_of_3(max_of_3(a, b, c), x[15], x[15]), f[p], lv[p]));
      }
      const bool need = m_new - m_run > kTcRescaleLog2;  // true on the first tile (m_run = -inf)
      if (__any_sync(0xffffffffu, need)) {
        if (i > 0) {
          // O may be touched once the product of the tile before has finished
          if (alive) alive = mbar_wait(odone, (i - 1) & 1, err);
          tc_fence_after();
          // a row that has seen no key yet holds exact zeros
          const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
          l_run *= alpha;
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t o[32];
            tmem_ld32(o_acc + c0, o);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
            tmem_st32(o_acc + c0, o);
          }
        }
        m_run = m_new;
      }
      const float mb = m_run == -INFINITY ? 0.f : m_run - kKv8PLift;
      bool p_free = i == 0;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t pk[32];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const float factor = f[half * 4 + p], off = lv[half * 4 + p] - mb;
          float sum[2];
#pragma unroll
          for (int ch = 0; ch < 2; ++ch) {
            // asked here, needed behind this half: P was last read by the product of the tile before; the next S
            if (p == 2 && ch == 1 && half == 0 && i > 0) p_free = mbar_test(odone, (i - 1) & 1);
            if (p == 2 && ch == 1 && half == 1) s_ready = mbar_test(sfull, (i + 1) & 1);
            float e[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = fast_exp2(fmaf(s[half * 64 + p * 16 + ch * 8 + k], factor, off));
            sum[ch] = ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
#pragma unroll
            for (int k = 0; k < 4; ++k) pk[p * 8 + ch * 4 + k] = pack_f16x2(e[2 * k], e[2 * k + 1]);
          }
          l_run = fmaf(sum[0] + sum[1], sc[half * 4 + p].z, l_run);
        }
        if (half == 0 && !__all_sync(0xffffffffu, p_free) && alive) alive = mbar_wait(odone, (i - 1) & 1, err);
        tc_fence_after();
        tmem_st32(p_tm + half * 32, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull + 8 * half);
      }
      put_scales(i + 1);
    }
    // ---- epilogue, once the products of the last key tiles have finished.  The warps of a CTA with one tile take half of the columns each, for
    // the sum of both accumulators.
    sums[t * kTcRows + r] = l_run;
    refs[t * kTcRows + r] = m_run;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const int tok = tt0 + rt;
    const bool real = rt < QT && tok < t_end;
    const size_t oidx = static_cast<size_t>(tok) * num_q_heads + h * gr + (r - rt * gr);
    const bool second = own == 1 && n_of[1] > 0;  // there is an accumulator 1 to be added
    float l = l_run, w0 = 1.f, w1 = 0.f;
    bool any0 = true, any1 = false;  // the accumulator holds something
    if (own == 1) {
      const float m0 = refs[r], m1 = refs[kTcRows + r];
      any0 = m0 > -INFINITY;
      any1 = m1 > -INFINITY;
      m_run = fmaxf(m0, m1);
      const float ref = m_run == -INFINITY ? 0.f : m_run;
      w0 = fast_exp2(m0 - ref);
      w1 = fast_exp2(m1 - ref);
      l = w0 * sums[r] + w1 * sums[kTcRows + r];
    }
    if (splits > 1 && real && (own == 2 || t == 0)) part_ml[oidx * splits + split] = make_float2(m_run, l);
    const int n_e = own == 2 ? n_own : n_of[0];
    if (n_e > 0) {
      const uint32_t acc = own == 2 ? o_acc : tmem_o + lane_off;
      const int cols = own == 2 ? D : D / 2, col0 = own == 2 ? 0 : t * (D / 2);
      if (alive) alive = mbar_wait(own == 2 ? odone : bar_odone, (n_e - 1) & 1, err);
      if (second && alive) alive = mbar_wait(bar_odone + 8, (n_of[1] - 1) & 1, err);
      tc_fence_after();
      const float inv = splits > 1 ? 1.f : 1.f / l, none = 0.f * l;  // none: 0, or NaN where the row's sum is
#pragma unroll 1
      for (int c0 = col0; c0 < col0 + cols; c0 += 32) {
        uint32_t o[32];
        tmem_ld32(acc + c0, o);
        tmem_ld_wait();
        // What is in an accumulator that holds nothing may not be a number, and its weight of 0 would not undo that.  A weight that vanished
        // beside the other's is taken: times a NaN it is one.
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(any0 ? __uint_as_float(o[c]) * (w0 * inv) : none);
        if (second) {
          uint32_t o1[32];
          tmem_ld32(acc + kTcKeys + c0, o1);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (any1) o[c] = __float_as_uint(fmaf(__uint_as_float(o1[c]), w1 * inv, __uint_as_float(o[c])));
        }
        if (real && alive) {
          if (splits > 1) {
            uint4* to = reinterpret_cast<uint4*>(part_o + (oidx * splits + split) * D + c0);
#pragma unroll
            for (int c = 0; c < 8; ++c) to[c] = make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
          } else {
            uint4* to = reinterpret_cast<uint4*>(out + oidx * D + c0);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t x[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) x[k] = pack_bf16x2(__uint_as_float(o[8 * c + 2 * k]), __uint_as_float(o[8 * c + 2 * k + 1]));
              to[c] = make_uint4(x[0], x[1], x[2], x[3]);
            }
          }
        }
      }
    }
    __syncwarp();
    asm volatile("bar.arrive 2, 384;" ::: "memory");  // rows written
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
#endif
}

// How a call is laid out: tiles of 128 score rows per kv head, how many CTAs of a head take two of them (the rule of the 16-bit kernel,
// paged_prefill_pairs.cu), and into how many parts of `split_tiles` key tiles the keys are cut.
struct Kv8PrefillPlan {
  int ctas, pairs, splits, split_tiles;
};
static int kv8_prefill_plan(int num_tokens, int first_pos, int hq, int hkv, Kv8PrefillPlan* p) {
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc) return rc;
  // The 16-bit kernel's rule, whose tile costs are not quite those here.  us with its choice, all single tiles, all pairs; 32 / 4 heads of 128:
  // 2048 tokens 50, 64, 51; 1500 behind 100 36, 45, 36; 1024 25.4, 23.9, 25.4; 600 16.6, 16.6, 19.3; 1024 behind 14336 233, 285, 233; 1500 behind
  // 14001 353, 417, 436; 300 behind 3000 36.1, 36.0, 37.8.  64 / 4: 512 behind 4096 79, 90, 79.  8 / 8: 700 behind 900 19.6, 19.6, 26.5.  32 / 4 of
  // 64: 2048 41, 52, 41; 16 / 2: 2048 26.6, 26.5, 35.1; 2048 behind 2048 63.7, 58.7, 63.7; 1024 behind 14336 126.5, 126.2, 122.0.
  p->pairs = b200_paged_attn_prefill_pairs(num_tokens, first_pos, hq, hkv, 0, sms, nullptr);
  if (p->pairs < 0) return p->pairs;
  const int qt = kTcRows / (hq / hkv), key_tiles = (first_pos + num_tokens - 1) / kTcKeys + 1;
  p->ctas = (num_tokens + qt - 1) / qt - p->pairs;
  const long long all = static_cast<long long>(p->ctas) * hkv;
  // As many parts as SMs are there for, down to one key tile: us with parts of at least 1, 2, 4, 8 key tiles, a token behind 600 (32 / 4
  // heads of 128) 9.3, 10.3, 11.4, 12.2, behind 3000 10.2, 10.3, 12.4, 16.5; 64 tokens behind 2000 (8 / 2 of 64) 11.4, 12.3, 13.4, 15.4;
  // 128 behind 1100 (8 / 1 of 128) 15.5, 14.4, 17.5, 17.2.  Where CTAs of pairs are 60 to 70 % of the SMs, three or four parts may gain: 700 behind
  // 8000 (32 / 4 of 128) 141 in one, 160, 126, 144 in two, three, four; 400 behind 12000 (64 / 4) 196, 216, 221, 190; but 1024 behind 14336 245, 272,
  // 291, 296, 512 behind 4096 (64 / 4) 79, 108, 126, 133.
  const int want = static_cast<int>(std::max(1ll, std::min<long long>(sms / all, key_tiles)));
  p->split_tiles = (key_tiles + want - 1) / want;
  p->splits = (key_tiles + p->split_tiles - 1) / p->split_tiles;
  return 0;
}

template <int D>
static int launch_kv8_prefill(const void* q, const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale,
                              const int* table_row, void* out, const AttnWorkspace& w, int num_tokens, int first_pos, int hq, int hkv,
                              int num_blocks, float scale, const Kv8PrefillPlan& p, cudaStream_t st) {
  CUtensorMap kmap;
  const uint64_t rows = static_cast<uint64_t>(num_blocks) * hkv * kKvPage;
  int rc = D == 128 ? get_tensor_map_2d(k_pool, rows, 128, 1, kKvPage, 128, &kmap) : get_tensor_map_2d_64(k_pool, rows, kKvPage, &kmap);
  if (rc) return rc;
  rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&kv8_attn_prefill_kernel<D>), Kv8PrefillCfg<D>::kSmemBytes);
  if (rc) return rc;
  B200_CUDA(launch_overlapped(kv8_attn_prefill_kernel<D>, dim3(p.ctas * p.splits * hkv), dim3(kKv8PrefillThreads), Kv8PrefillCfg<D>::kSmemBytes,
                              st, kmap, static_cast<const uint8_t*>(v_pool), static_cast<const uint8_t*>(k_scale),
                              static_cast<const uint8_t*>(v_scale), table_row, static_cast<const __nv_bfloat16*>(q),
                              static_cast<__nv_bfloat16*>(out), w.o, w.ml, w.err, num_tokens, first_pos, hq, hkv, num_blocks,
                              scale * 1.4426950408889634f, p.pairs, p.splits, p.split_tiles));
  if (p.splits > 1) return launch_kv8_join(D, w, out, num_tokens, hq, p.splits, st);
  return 0;
}

}  // namespace b200

using namespace b200;

extern "C" size_t b200_kv8_attn_prefill_workspace_bytes(int num_tokens, int first_position, int num_q_heads, int num_kv_heads, int head_dim) {
  if (num_tokens <= 0 || first_position < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || num_q_heads % num_kv_heads != 0 ||
      num_q_heads / num_kv_heads > kTcRows || static_cast<long long>(num_tokens) + first_position >= (1ll << 31) - kTcKeys)
    return 256;
  Kv8PrefillPlan p;
  if (kv8_prefill_plan(num_tokens, first_position, num_q_heads, num_kv_heads, &p) || p.splits == 1) return 256;
  return carve(nullptr, num_tokens, num_q_heads, head_dim, p.splits).bytes;
}

extern "C" int b200_kv8_attn_prefill(const void* q, const void* k_pool, const void* v_pool, const void* k_scale, const void* v_scale,
                                     const int32_t* block_table_row, void* out, void* workspace, size_t workspace_bytes, int num_tokens,
                                     int first_position, int num_q_heads, int num_kv_heads, int head_dim, int num_blocks,
                                     int max_pages_per_seq, float scale, void* stream) {
  B200_REQUIRE(q && k_pool && v_pool && k_scale && v_scale && block_table_row && out && workspace, "kv8_attn_prefill: null pointer");
  int rc = check_kv8("kv8_attn_prefill", num_tokens, num_q_heads, num_kv_heads, head_dim, num_blocks, max_pages_per_seq, q, k_pool, v_pool, out,
                     scale);
  if (rc) return rc;
  B200_REQUIRE(on_words(block_table_row), "kv8_attn_prefill: the table row must be 4-byte aligned");
  B200_REQUIRE(num_q_heads / num_kv_heads <= kTcRows, "kv8_attn_prefill: more than %d q heads per kv head", kTcRows);
  B200_REQUIRE(first_position >= 0 && static_cast<long long>(first_position) + num_tokens <= static_cast<long long>(max_pages_per_seq) * kKvPage,
               "kv8_attn_prefill: positions %d .. of %d tokens do not fit %d pages", first_position, num_tokens, max_pages_per_seq);
  B200_REQUIRE(static_cast<long long>(first_position) + num_tokens < (1ll << 31) - kTcKeys &&
                   static_cast<long long>(num_tokens) * num_q_heads < (1ll << 31),
               "kv8_attn_prefill: positions or rows past 2^31");
  rc = check_device(nullptr);
  if (rc) return rc;
  Kv8PrefillPlan p;
  rc = kv8_prefill_plan(num_tokens, first_position, num_q_heads, num_kv_heads, &p);
  if (rc) return rc;
  B200_REQUIRE(static_cast<long long>(p.ctas) * p.splits * num_kv_heads < (1ll << 31), "kv8_attn_prefill: grid too large");
  AttnWorkspace w = carve(workspace, num_tokens, num_q_heads, head_dim, p.splits);
  const size_t need = p.splits > 1 ? w.bytes : 256;
  if (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) {
    set_detail("kv8_attn_prefill: workspace of %zu bytes at %p, %zu on a 16-byte boundary are needed", workspace_bytes, workspace, need);
    return -kErrWorkspace;
  }
#define B200_KV8_ARGS q, k_pool, v_pool, k_scale, v_scale, block_table_row, out, w, num_tokens, first_position, num_q_heads, num_kv_heads, \
                      num_blocks, scale, p, as_stream(stream)
  return head_dim == 128 ? launch_kv8_prefill<128>(B200_KV8_ARGS) : launch_kv8_prefill<64>(B200_KV8_ARGS);
#undef B200_KV8_ARGS
}
