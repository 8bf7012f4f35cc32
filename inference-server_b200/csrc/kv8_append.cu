// Filling the 8-bit page cache (kv8.cuh): slots of new tokens from request lengths, and keys and values into their slots.
//
// The reference keeps both on the host and in 16 bits: block lists per request (src/inference_server/kv_cache/block_manager.py:51-94)
// and a copy of dense keys and values into fresh blocks (src/inference_server/kv_cache/cache_manager.py:185-214).

#include "host.h"
#include "kv8.cuh"

namespace b200 {

// ----------------------------------------------------------------- slot map --
//
// need_b = pages(ctx_b + new_b) - pages(ctx_b) pages go to sequence b out of the list of free pages, in the order of the sequences, by
// exclusive prefix sums; so do the rows of the new tokens.  Every CTA takes the sums of all sequences for itself (a few KB from L2, one
// scan of pairs packed into 64 bits) and keeps them in shared memory; then a row finds its sequence, and a fresh page its place in the
// table, by bisection.  So one launch does all of it, no CTA waits for another, and none reads what another writes: a row in a
// fresh page takes the page from the list and not from the table.  Bound by the chain of loads (lengths, then list or table): 3.3 us for a
// step of 256 sequences, 3.1 for 48 prompts of 20000 tokens, in a graph of calls; the scan is 256 sequences a round.
constexpr int kMapThreads = 256;
constexpr int kMapMaxSeqs = 4096;

// The last i in [0, n) with start[i] <= x, for ascending start with start[0] <= x.
__device__ __forceinline__ int bisect(const int* start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kMapThreads)
kv_slot_map_kernel(const int* __restrict__ ctx_lens, const int* __restrict__ new_lens, int* __restrict__ table,
                   const int* __restrict__ supply, const int* __restrict__ supply_used, int supply_len, int* __restrict__ lens,
                   int* __restrict__ row_start, int* __restrict__ row_seq, int* __restrict__ positions, int* __restrict__ slots,
                   int* __restrict__ used_out, int* __restrict__ err, int num_seqs, int num_rows, int num_blocks, int max_pages) {
  grid_dep_wait();
  grid_dep_launch();
  extern __shared__ int map_smem[];
  int* rows_at = map_smem;                 // [num_seqs + 1] first row of a sequence
  int* pages_at = map_smem + num_seqs + 1;  // [num_seqs + 1] first of its fresh pages
  __shared__ unsigned long long warp_sum[kMapThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool first_cta = blockIdx.x == 0;
  int used = *supply_used;
  if (used < 0 || used > supply_len) {  // no page can be told free
    if (first_cta && tid == 0) set_error(err, kErrDevNoPages);
    used = supply_len;
  }

  // pairs (new rows, fresh pages) in the two halves of 64 bits; neither sum passes 2^31 (checked on the host by the table's size)
  unsigned long long carry = 0;
  for (int b0 = 0; b0 < num_seqs; b0 += kMapThreads) {
    const int b = b0 + tid;
    int c = 0, n = 0;
    if (b < num_seqs) {
      c = ctx_lens[b];
      n = new_lens[b];
      if (c < 0 || n < 0 || c > max_pages * kKvPage || n > max_pages * kKvPage - c) {  // a sequence that does not fit gets nothing
        if (first_cta) set_error(err, kErrDevBadCtxLen);
        n = 0;
        c = min(max(c, 0), max_pages * kKvPage);
      }
      if (first_cta) lens[b] = c + n;
    }
    const int take = (c + n + kKvPage - 1) / kKvPage - (c + kKvPage - 1) / kKvPage;
    const unsigned long long mine = static_cast<unsigned long long>(take) << 32 | static_cast<unsigned>(n);
    unsigned long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    unsigned long long before = carry, all = carry;
#pragma unroll
    for (int w = 0; w < kMapThreads / 32; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    const unsigned long long at = before + sum - mine;
    if (b < num_seqs) {
      rows_at[b] = static_cast<int>(at);
      pages_at[b] = static_cast<int>(at >> 32);
      if (first_cta) row_start[b] = static_cast<int>(at);
    }
    carry = all;
    __syncthreads();
  }
  const int rows = static_cast<int>(carry), pages = static_cast<int>(carry >> 32);
  if (tid == 0) {
    rows_at[num_seqs] = rows;
    pages_at[num_seqs] = pages;
    if (first_cta) {
      row_start[num_seqs] = rows;
      if (rows > num_rows) set_error(err, kErrDevBadCtxLen);
      if (pages > supply_len - used) set_error(err, kErrDevNoPages);
      *used_out = used + min(pages, supply_len - used);
    }
  }
  __syncthreads();

  const int stride = gridDim.x * kMapThreads;
  const int handed = min(pages, supply_len - used);
  // A page that is not there, or is none, is -1 in the table: lens counts it, so the next call takes the entry for the sequence's own page,
  // and what a table row of earlier use names there belongs to another sequence by now.
  for (int p = blockIdx.x * kMapThreads + tid; p < pages; p += stride) {
    int id = p < handed ? supply[used + p] : -1;
    if (id < 0 || id >= num_blocks) {
      if (p < handed) set_error(err, kErrDevBadBlockId);
      id = -1;
    }
    // of sequences that begin at the same page the last is the one that gets it
    const int b = bisect(pages_at, num_seqs, p);
    const int have = (ctx_lens[b] + kKvPage - 1) / kKvPage;  // in range: a sequence that takes pages fits
    table[static_cast<size_t>(b) * max_pages + have + p - pages_at[b]] = id;
  }
  for (int r = blockIdx.x * kMapThreads + tid; r < num_rows; r += stride) {
    int seq = -1, pos = 0, slot = -1;
    if (r < rows) {
      seq = bisect(rows_at, num_seqs, r);
      const int c = ctx_lens[seq], have = (c + kKvPage - 1) / kKvPage;
      pos = c + r - rows_at[seq];
      const int page = pos / kKvPage;
      int id = -1;
      if (page < have) {
        id = table[static_cast<size_t>(seq) * max_pages + page];
        if (id < 0 || id >= num_blocks) set_error(err, kErrDevBadBlockId);
      } else if (pages_at[seq] + page - have < handed) {
        id = supply[used + pages_at[seq] + page - have];
      }
      if (id >= 0 && id < num_blocks) slot = id * kKvPage + pos % kKvPage;
    }
    row_seq[r] = seq;
    positions[r] = pos;
    slots[r] = slot;
  }
}

// ------------------------------------------------------------------- append --
//
// A run is a set of neighbouring rows whose slots lie in one page.  One warp takes a run's keys, or values, of one kv head: it holds up
// to 16 rows in registers, 16 bytes a lane and load, so that their largest magnitude and their rounding are one pass
// over memory, finds the page's scale and writes 8-bit rows.  Only where the scale of a page that already had tokens grows are its
// earlier rows read, rounded anew and written back.  Nothing else of the page is touched.
//
// A CTA looks after `window` rows: it does the runs that begin there, its warps sharing (run, head, K or V) items.  Few rows per window
// give a decode step, whose rows are runs of one, a CTA each; many rows per window keep a prompt, whose runs are 16 long, from
// launching CTAs that find nothing to begin.
//
// Bound by memory for prompts, whose rows are read once (8970 rows of 4 heads of 128 in bf16, 28 MB read and written, 8.8 us; 4.2 at the copy
// rate, the rest a launch and the chain slot -> rows -> largest magnitude -> scale -> stores), by that chain for steps (256 rows 3.0 us).
constexpr int kAppendWarps = 8;
constexpr int kAppendMaxWindow = 16;  // a run that begins in a window lies within the 32 rows that a warp's lanes look at

// 16 bytes of a row: 8 bf16 or 4 fp32 numbers.
template <typename T>
struct RowPiece {
  static constexpr int kNumbers = 16 / static_cast<int>(sizeof(T));
  uint4 w;
  __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(word(i));
    else return __uint_as_float(i & 1 ? word(i / 2) & 0xffff0000u : word(i / 2) << 16);
  }
  // Largest magnitudes so far, infinities and NaN among them: bits of an fp32 number, or of two bf16 numbers side by side.
  __device__ __forceinline__ uint32_t top(uint32_t m) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = sizeof(T) == 4 ? max(m, word(i) & 0x7fffffffu) : __vmaxu2(m, word(i) & 0x7fff7fffu);
    return m;
  }
  __device__ __forceinline__ static uint32_t top_of(uint32_t m) { return sizeof(T) == 4 ? m : max(m >> 16, m & 0xffffu) << 16; }
  __device__ __forceinline__ uint32_t finite_top(uint32_t m) const {
#pragma unroll
    for (int i = 0; i < kNumbers; ++i) {
      const uint32_t a = __float_as_uint(value(i)) & 0x7fffffffu;
      m = max(m, a < 0x7f800000u ? a : 0u);
    }
    return m;
  }
  // e4m3 codes of the numbers times `by`, which is a power of two: the product is exact, or underflows far below the smallest code.
  // An infinity has no e4m3 number and must not look like one: where there may be any (`ODD`) it becomes NaN.
  template <bool ODD>
  __device__ __forceinline__ void store(uint8_t* to, float by) const {
    uint32_t codes[kNumbers / 4];
#pragma unroll
    for (int k = 0; k < kNumbers / 4; ++k) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = value(4 * k + i);
        if (ODD && !(fabsf(x[i]) < INFINITY)) x[i] = NAN;
      }
      const float2 lo = mul_pair(x[0], x[1], by), hi = mul_pair(x[2], x[3], by);
      codes[k] = to_e4m3x4(lo.x, lo.y, hi.x, hi.y);
    }
    if constexpr (kNumbers == 8) *reinterpret_cast<uint2*>(to) = make_uint2(codes[0], codes[1]);
    else *reinterpret_cast<uint32_t*>(to) = codes[0];
  }
};

// Four codes times `by`, rounded again.
__device__ __forceinline__ uint32_t round_again(uint32_t codes, float by) {
  uint32_t lo, hi;
  e4m3x4_to_f16(codes, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return to_e4m3x4(a.x * by, a.y * by, b.x * by, b.y * by);
}

template <typename T, int D>
__global__ void __launch_bounds__(kAppendWarps * 32, D * sizeof(T) > 256 ? 2 : 4)
kv8_append_kernel(const T* __restrict__ k_new, const T* __restrict__ v_new, long long k_stride, long long v_stride,
                  uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool, uint8_t* __restrict__ k_scale, uint8_t* __restrict__ v_scale,
                  const int* __restrict__ slots, int* __restrict__ err, int num_rows, int num_kv_heads, int num_blocks, int window) {
  grid_dep_wait();
  grid_dep_launch();
  using Piece = RowPiece<T>;
  constexpr int kLanes = D / Piece::kNumbers, kAtOnce = 32 / kLanes, kSteps = kKvPage / kAtOnce;  // lanes of a row; rows of a step
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / kLanes, col = lane % kLanes * Piece::kNumbers;
  const int row0 = blockIdx.x * window;  // lane l looks at row row0 - 1 + l
  const int my_row = row0 - 1 + lane;
  int slot = -1;
  if (my_row >= 0 && my_row < num_rows) slot = slots[my_row];
  if (slot >= num_blocks * kKvPage) {
    set_error(err, kErrDevBadBlockId);
    slot = -1;
  }
  const int block = slot < 0 ? -1 : slot / kKvPage;
  const int left = __shfl_up_sync(0xffffffffu, block, 1);
  unsigned starts = __ballot_sync(0xffffffffu, lane >= 1 && lane <= window && block >= 0 && block != left);
  const int items = 2 * num_kv_heads, total = __popc(starts) * items;
  int item = warp;  // of the run of the lowest bit left in `starts`
#pragma unroll 1
  for (int it = warp; it < total; it += kAppendWarps, item += kAppendWarps) {
    for (; item >= items; item -= items) starts &= starts - 1;
    const int first = __ffs(starts) - 1;
    const int page = __shfl_sync(0xffffffffu, block, first);
    const unsigned same = __ballot_sync(0xffffffffu, block == page) >> first;
    int n = __ffs(~same) - 1;  // rows of the run among those of the lanes; first >= 1, so a bit of `same` is clear
    const int row = row0 - 1 + first, low0 = __shfl_sync(0xffffffffu, slot, first);
    // The usual run names one slot after the other.
    const bool inside = lane >= first && lane < first + n;
    bool plain = __all_sync(0xffffffffu, !inside || slot - lane == low0 - first) && n <= kKvPage;
    int low = low0 % kKvPage;
    if (!plain || first + n == 32) {
      low = __reduce_min_sync(0xffffffffu, inside ? slot % kKvPage : kKvPage);
      // slots named more than once can make a run longer than a page
      for (; row + n < num_rows && slots[row + n] >= 0 && slots[row + n] / kKvPage == page; ++n) {
        low = min(low, slots[row + n] % kKvPage);
        plain = false;
      }
    }

    const bool is_v = item >= num_kv_heads;
    const int h = is_v ? item - num_kv_heads : item;
    const long long stride = is_v ? v_stride : k_stride;
    const T* src = (is_v ? v_new : k_new) + row * stride + h * D + col;
    const size_t cell = static_cast<size_t>(page) * num_kv_heads + h;
    uint8_t* pool = (is_v ? v_pool : k_pool) + cell * (kKvPage * D) + col;
    uint8_t* scale = (is_v ? v_scale : k_scale) + cell;
    const int old = scale_exponent(*scale);

    Piece x[kSteps];
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      x[s].w = make_uint4(0u, 0u, 0u, 0u);
      if (s * kAtOnce + sub < n) x[s].w = *reinterpret_cast<const uint4*>(src + (s * kAtOnce + sub) * stride);
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) top = x[s].top(top);
#pragma unroll 1
    for (int i = kKvPage + sub; i < n; i += kAtOnce) top = Piece{*reinterpret_cast<const uint4*>(src + i * stride)}.top(top);
    top = __reduce_max_sync(0xffffffffu, Piece::top_of(top));
    if (top >= 0x7f800000u) {  // the largest finite magnitude instead
      plain = false;
      top = 0;
#pragma unroll 1
      for (int i = sub; i < n; i += kAtOnce) top = Piece{*reinterpret_cast<const uint4*>(src + i * stride)}.finite_top(top);
      top = __reduce_max_sync(0xffffffffu, top);
    }
    int e = fit_exponent(top);
    if (low > 0 && old >= e) {
      e = old;
    } else {  // a new page, or a larger scale for one that has tokens
      const float by = power_of_two(old - e);
      constexpr int kBatch = kSteps < 4 ? kSteps : 4;
#pragma unroll 1
      for (int r0 = sub; r0 < low; r0 += kBatch * kAtOnce) {
        uint32_t codes[kBatch][Piece::kNumbers / 4];
#pragma unroll
        for (int s = 0; s < kBatch; ++s)
          if (r0 + s * kAtOnce < low)
#pragma unroll
            for (int k = 0; k < Piece::kNumbers / 4; ++k)
              codes[s][k] = *reinterpret_cast<const uint32_t*>(pool + (r0 + s * kAtOnce) * D + 4 * k);
#pragma unroll
        for (int s = 0; s < kBatch; ++s)
          if (r0 + s * kAtOnce < low)
#pragma unroll
            for (int k = 0; k < Piece::kNumbers / 4; ++k)
              *reinterpret_cast<uint32_t*>(pool + (r0 + s * kAtOnce) * D + 4 * k) = round_again(codes[s][k], by);
      }
      __syncwarp();
      if (lane == 0) *scale = static_cast<uint8_t>(e + 127);
    }
    const float by = power_of_two(-e);
    if (plain) {
      uint8_t* to = pool + (low + sub) * D;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        if (s * kAtOnce + sub < n) x[s].template store<false>(to + s * kAtOnce * D, by);
    } else {  // one row after the other: of those that name one slot the last stays
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        if (sub == 0) Piece{*reinterpret_cast<const uint4*>(src + i * stride)}.template store<true>(pool + slots[row + i] % kKvPage * D, by);
      }
    }
  }
}

template <typename T, int D>
static int launch_append(const void* k_new, const void* v_new, long long ks, long long vs, void* k_pool, void* v_pool, void* k_scale,
                         void* v_scale, const int* slots, int* err, int rows, int hkv, int num_blocks, cudaStream_t st) {
  int sms = 0;
  int rc = device_sm_count(&sms);
  if (rc) return rc;
  // The fewest rows per CTA with which the grid fits the GPU at once.  us with 4, 8 and 16 CTAs per SM in its place: 8970 rows of 4 heads
  // of 128 in bf16 8.8, 11.4, 12.2; 61 short prompts of 2 heads of 64 in fp32 2.4, 3.1, 3.0.
  int window = 1;
  while (window < kAppendMaxWindow && (rows + window - 1) / window > 4 * sms) window *= 2;
  B200_CUDA(launch_overlapped(kv8_append_kernel<T, D>, dim3((rows + window - 1) / window), dim3(kAppendWarps * 32), 0, st,
                              static_cast<const T*>(k_new), static_cast<const T*>(v_new), ks, vs, static_cast<uint8_t*>(k_pool),
                              static_cast<uint8_t*>(v_pool), static_cast<uint8_t*>(k_scale), static_cast<uint8_t*>(v_scale), slots, err,
                              rows, hkv, num_blocks, window));
  return 0;
}

}  // namespace b200

using namespace b200;

extern "C" int b200_kv_slot_map(const int32_t* ctx_lens, const int32_t* new_lens, int32_t* block_table, const int32_t* supply,
                                const int32_t* supply_used, int supply_len, int32_t* lens, int32_t* row_start, int32_t* row_seq,
                                int32_t* positions, int32_t* slots, int32_t* supply_used_out, void* status_word, int num_seqs,
                                int num_rows, int num_blocks, int max_pages_per_seq, void* stream) {
  B200_REQUIRE(ctx_lens && new_lens && block_table && supply_used && lens && row_start && supply_used_out &&
                   (supply || supply_len == 0) && ((row_seq && positions && slots) || num_rows == 0),
               "kv_slot_map: null pointer");
  B200_REQUIRE(on_words(ctx_lens, new_lens, block_table, supply, supply_used, lens, row_start, row_seq, positions, slots, supply_used_out, status_word),
               "kv_slot_map: whole numbers and the status word must be 4-byte aligned");
  B200_REQUIRE(num_seqs > 0 && num_seqs <= kMapMaxSeqs, "kv_slot_map: %d sequences outside [1, %d]", num_seqs, kMapMaxSeqs);
  B200_REQUIRE(num_rows >= 0 && supply_len >= 0 && num_blocks > 0 && max_pages_per_seq > 0, "kv_slot_map: bad dimension");
  B200_REQUIRE(static_cast<long long>(num_seqs) * max_pages_per_seq * kKvPage < (1ll << 31) &&
                   static_cast<long long>(num_blocks) * kKvPage < (1ll << 31) && num_rows < (1 << 30),
               "kv_slot_map: tokens of the table, or slots of the pool, past 2^31");
  B200_REQUIRE(supply_used_out != supply_used && lens != ctx_lens && lens != new_lens,
               "kv_slot_map: an output is an input, which other blocks still read");
  int rc = check_device(nullptr);
  if (rc) return rc;
  int sms = 0;
  rc = device_sm_count(&sms);
  if (rc) return rc;
  const int want = (num_rows + kMapThreads - 1) / kMapThreads;
  const int ctas = want < 1 ? 1 : want > 2 * sms ? 2 * sms : want;
  const size_t smem = static_cast<size_t>(2 * (num_seqs + 1)) * sizeof(int);
  B200_CUDA(launch_overlapped(kv_slot_map_kernel, dim3(ctas), dim3(kMapThreads), smem, as_stream(stream), ctx_lens, new_lens, block_table,
                              supply, supply_used, supply_len, lens, row_start, row_seq, positions, slots, supply_used_out,
                              static_cast<int*>(status_word), num_seqs, num_rows, num_blocks, max_pages_per_seq));
  return 0;
}

extern "C" int b200_kv8_append(const void* k_new, const void* v_new, int64_t k_row_stride, int64_t v_row_stride, void* k_pool, void* v_pool,
                               void* k_scale, void* v_scale, const int32_t* slots, void* status_word, int num_rows, int num_kv_heads,
                               int head_dim, int num_blocks, int dtype, void* stream) {
  B200_REQUIRE(k_new && v_new && k_pool && v_pool && k_scale && v_scale && slots, "kv8_append: null pointer");
  B200_REQUIRE(on_words(slots, status_word), "kv8_append: slots and the status word must be 4-byte aligned");
  B200_REQUIRE(num_rows > 0 && num_kv_heads > 0 && num_blocks > 0, "kv8_append: non-positive dimension");
  B200_REQUIRE(head_dim == 64 || head_dim == 128, "kv8_append: head_dim %d is neither 64 nor 128", head_dim);
  B200_REQUIRE(dtype == 0 || dtype == 1, "kv8_append: dtype %d is neither 0 (bf16) nor 1 (f32)", dtype);
  B200_REQUIRE(static_cast<long long>(num_blocks) * kKvPage < (1ll << 31), "kv8_append: %d pages have more slots than 32 bits count", num_blocks);
  B200_REQUIRE(num_rows < (1 << 30) && num_kv_heads <= 1 << 20, "kv8_append: too many rows or heads");
  const int align = 16;  // bytes a lane loads at once
  const int elem = dtype == 0 ? 2 : 4;
  B200_REQUIRE(reinterpret_cast<uintptr_t>(k_new) % align == 0 && reinterpret_cast<uintptr_t>(v_new) % align == 0 &&
                   k_row_stride * elem % align == 0 && v_row_stride * elem % align == 0 && k_row_stride >= 0 && v_row_stride >= 0,
               "kv8_append: rows of k and v must start on multiples of %d bytes", align);
  B200_REQUIRE(reinterpret_cast<uintptr_t>(k_pool) % 16 == 0 && reinterpret_cast<uintptr_t>(v_pool) % 16 == 0,
               "kv8_append: pools must be 16-byte aligned");
  int rc = check_device(nullptr);
  if (rc) return rc;
#define B200_APPEND_ARGS k_new, v_new, k_row_stride, v_row_stride, k_pool, v_pool, k_scale, v_scale, slots, static_cast<int*>(status_word), \
                         num_rows, num_kv_heads, num_blocks, as_stream(stream)
  if (dtype == 0) return head_dim == 128 ? launch_append<__nv_bfloat16, 128>(B200_APPEND_ARGS) : launch_append<__nv_bfloat16, 64>(B200_APPEND_ARGS);
  return head_dim == 128 ? launch_append<float, 128>(B200_APPEND_ARGS) : launch_append<float, 64>(B200_APPEND_ARGS);
#undef B200_APPEND_ARGS
}
