// Decode attention over the 4-bit paged KV cache (format: kv4.cuh): head sizes 64, 128 and 256, 16-token pages,
// at most 16 query rows per (sequence, kv head) -- the G = hq / hkv heads of the group times the appended tokens.
//
// Floor: the cached bytes, 160 per token and kv head at D = 128 (K and V), once. At 44 bytes per ns and SM that
// leaves 112 clocks, 448 issue slots, per 16 tokens and SM. The nibbles decide whether that is met:
//
//   S^T = K Q^T   m16n8k16 with the 16 tokens of a page as M and 8 query rows as N: half the instructions of the
//                 usual orientation, whose M = 16 rows would be mostly padding. Two k-steps cover one quantisation
//                 group, so K needs no expansion: the fragments hold the integers bias + c that a nibble is
//                 under a suitable exponent (64 + c in fp16, 128 + c in bf16: one and-or), and the group's step
//                 multiplies the fp32 result. Bias and minimum are two more k-steps: lo_g and s_g against the group
//                 sums of q, split into two (bf16: three) terms of the rows' type. K is thus never rounded.
//   softmax       in the S^T accumulators: a lane has two query rows and 4 tokens of 16. The reference maximum is
//                 raised only when some score exceeds it by more than 8 (log2), so the usual step has no shuffle
//                 and no rescaling; P stays below 2^8 and the final division by the row sum makes it exact.
//   O^T += V^T P^T  M = 16 channels, N = 8 query rows; P^T fragments come from the S^T accumulators by one
//                 8 x 8 transpose (movmatrix) per 8 tokens. A fragments want pairs of tokens: two tokens' code
//                 words are interleaved by halves (prmt) and expanded, lo + s c rounded once to fp16. For bf16 rows
//                 lo and s are first scaled by a power of two that follows the largest of them, so that V and P keep
//                 11 bits. (The step cannot move to P as it does for K: p * s underflows fp16 for small s.)
//
// P is rounded to fp16; sums, maxima and accumulators are fp32.
//
// Measured, 32 / 8 heads of 128 (ten launches in a CUDA graph): 256 sequences of 512 to 2048, fp16 123 us (3.4 TB/s of the cached
// bytes, the 16-bit cache's kernel would read 3.2 times as many); 8 of 16300, bf16 53 us; one of 1000 9.9 us; 64 trees of four
// tokens behind 100 to 4000, fp16 98 us. No unit is full at 256 sequences: issue slots 56 %, integer pipe 47 %, DRAM 42 %, tensor pipe
// 20 %. It is latency: a warp issues every 6.4 clocks, 2.1 of them waiting for memory and copies, 1.3 for the previous instruction, and
// three consumer warps per scheduler do not cover that.
//
// Work: a unit is one (sequence, kv head, block of 8 or 16 query rows). All units' slots of 32 tokens (two pages),
// laid end to end, are cut into equal shares, one per persistent CTA, so ragged batches and single long sequences
// load every SM alike; a unit cut between CTAs leaves fp32 partial results that a second kernel joins. In a CTA
// a producer warp streams the share's pages (bulk copies into a ring of slots) and, per unit, its query rows and a
// descriptor, ahead of four consumer warps that take the slots round-robin. At the end of a unit one of them, in turn,
// joins the results of the four while the others go on (all four waiting for each other: 64 heads over 8, D = 128, two
// tokens each 100 us instead of 89; D = 256 with a window 68 us instead of 57).
// Every wait is bounded (common.cuh).
#include "kv4.cuh"

namespace mlcb {

constexpr int KV4_DEC_THREADS = 160;
constexpr int KV4_DEC_ITEMS = 1024;   // items per launch: their prefix sums sit in shared memory
constexpr int KV4_DEC_MIN_SHARE = 4;  // slots per CTA at least: one per consumer warp

struct Kv4DecParams {
  const void* q;
  const uint8_t* pages;
  void* out;
  float* lse;
  float* part_o;   // [2 CTAs][16][D] fp32: partial rows of a share's first and last unit
  float* part_ml;  // [2 CTAs][16][2]
  int* part_unit;  // [CTAs][4]: unit begun here and cut: rows (0: none), first token, kv head * 16 + first row, pieces
  const int *item_seq, *item_qstart, *item_ntok, *q_kvlen, *page_indptr, *page_indices;
  const int* q_kvstart;
  const unsigned long long* tree_mask;
  int* status;
  long long q_stride, num_pages;
  int hq, hkv, group, row_blocks, num_items, sink;
  float scale_log2;          // sm_scale * log2(e)
  float cap_k, cap_log2;     // soft cap: scores are kv4_softcap(raw, cap_k, cap_log2); 0 = none
};

// What one item visits: pages [0, npg) of its list, less those that lie outside every row's window.
struct Kv4Item {
  int qstart, ntok, npg;
  int blocks;               // blocks of query rows
  int sink_pg, skip;        // pages [sink_pg, sink_pg + skip) of the list are never fetched
  int all_from, all_to;     // positions [all_from, all_to) are seen by every row (so is the sink below the window)
  const int* list;
};

template <bool EXT, int ROWS>
__device__ __forceinline__ Kv4Item kv4_item(const Kv4DecParams& p, int item) {
  Kv4Item d;
  const int b = p.item_seq[item];
  d.qstart = p.item_qstart[item];
  d.ntok = p.item_ntok[item];
  d.blocks = max(1, min(p.row_blocks, (d.ntok * p.group + ROWS - 1) / ROWS));
  int reach = 0, to = 0x7fffffff, from = 0, first = 0x7fffffff;
  for (int i = 0; i < d.ntok; ++i) {
    const int n = p.q_kvlen[d.qstart + i];
    int end = n;
    if (EXT && p.tree_mask) {
      const unsigned long long tm = p.tree_mask[d.qstart + i];
      if (tm) end += 64 - __clzll(tm);
    }
    reach = max(reach, end);
    to = min(to, n);
    if (EXT && p.q_kvstart) {
      const int s = p.q_kvstart[d.qstart + i];
      from = max(from, s);
      first = min(first, s);
    }
  }
  d.all_from = from;
  d.all_to = to;
  d.sink_pg = 0;
  d.skip = 0;
  if (EXT && p.q_kvstart) {
    d.sink_pg = (p.sink + KV4_PAGE - 1) / KV4_PAGE;
    d.skip = max(0, min(first, reach) / KV4_PAGE - d.sink_pg);
  }
  const int p0 = p.page_indptr[b];
  const int held = p.page_indptr[b + 1] - p0;
  d.list = p.page_indices + p0;
  int upto = (reach + KV4_PAGE - 1) / KV4_PAGE;
  if (upto > held) {  // more positions than the sequence has pages for: never dereferenced
    if (p.status) atomicCAS(p.status, 0, ERR_BAD_INDEX);
    upto = held;
  }
  d.npg = max(0, upto - d.skip);
  return d;
}

// A unit's part inside one share, handed from the producer to the consumers through shared memory.
struct Kv4Piece {
  int qstart, ntok, hk, row0;
  int slot0, slots;         // slots of the unit: first, count (0: nothing visible)
  int npg, sink_pg, skip, all_from, all_to;
  int list0;                // the sequence's first entry of page_indices
  int part;                 // -1: the whole unit, written to out; else the row block of part_o it goes to
  int last;                 // the share ends here
};

__device__ __forceinline__ uint32_t kv4_movmatrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename T>
__device__ __forceinline__ void kv4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1, const float (&c)[4]);
template <>
__device__ __forceinline__ void kv4_mma<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
template <>
__device__ __forceinline__ void kv4_mma<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// Pairs of integers bias + c for the nibbles at bits 4 i of both halves.
template <typename T>
__device__ __forceinline__ void kv4_raw4(uint32_t w, uint32_t (&out)[4]);
template <>
__device__ __forceinline__ void kv4_raw4<__half>(uint32_t w, uint32_t (&out)[4]) {
  out[0] = kv4_and_or(w << 4, 0x00f000f0u, 0x54005400u);
  out[1] = kv4_and_or(w, 0x00f000f0u, 0x54005400u);
  out[2] = kv4_and_or(w >> 4, 0x00f000f0u, 0x54005400u);
  out[3] = kv4_and_or(w >> 8, 0x00f000f0u, 0x54005400u);
}
template <>
__device__ __forceinline__ void kv4_raw4<__nv_bfloat16>(uint32_t w, uint32_t (&out)[4]) {
  out[0] = kv4_and_or(w, 0x000f000fu, 0x43004300u);
  out[1] = kv4_and_or(w >> 4, 0x000f000fu, 0x43004300u);
  out[2] = kv4_and_or(w >> 8, 0x000f000fu, 0x43004300u);
  out[3] = kv4_and_or(w >> 12, 0x000f000fu, 0x43004300u);
}
template <typename T>
struct Kv4Bias;
template <>
struct Kv4Bias<__half> {
  static constexpr float BIAS = 64.f;
  static constexpr uint32_t ONES = 0x3c003c00u;
};
template <>
struct Kv4Bias<__nv_bfloat16> {
  static constexpr float BIAS = 128.f;
  static constexpr uint32_t ONES = 0x3f803f80u;
};

// s of a (lo, s) word as fp32
template <typename T>
__device__ __forceinline__ float kv4_step(uint32_t meta);
template <>
__device__ __forceinline__ float kv4_step<__half>(uint32_t meta) {
  return __high2float(*reinterpret_cast<const __half2*>(&meta));
}
template <>
__device__ __forceinline__ float kv4_step<__nv_bfloat16>(uint32_t meta) {
  return __uint_as_float(meta & 0xffff0000u);
}

// Row `row` (of the item's rows) of the output: acc[c] = channel 32 c + lane, scaled by 1 / L. A row that sees nothing
// is 0 with log-sum-exp -inf; NaN stays NaN.
template <typename T, int D>
__device__ __forceinline__ void kv4_finish_row(const Kv4DecParams& p, int qstart, int hk, int row, float M, float L,
                                               const float (&acc)[D / 32]) {
  const int lane = threadIdx.x & 31;
  const size_t at = static_cast<size_t>(qstart + row / p.group) * p.hq + hk * p.group + row % p.group;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T* dst = reinterpret_cast<T*>(p.out) + at * D;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) dst[c * 32 + lane] = Cvt<T>::from_f(acc[c] * inv);
  if (p.lse && lane == 0) p.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

// The rows of one piece by kv4_rows_exact. A call of its own, so that it takes no registers from the ordinary path.
template <typename T, int D, bool EXT>
__device__ __noinline__ void kv4_piece_exact(const Kv4DecParams& p, const Kv4Piece* piece, int rows) {
  const Kv4Piece pc = *piece;
  const int lane = threadIdx.x & 31, npg = pc.npg;
  auto at = [&](int i) {
    const int pi = pc.slot0 * 2 + i / KV4_PAGE;
    return pi >= npg ? -1 : (!EXT || pi < pc.sink_pg ? pi : pi + pc.skip) * KV4_PAGE + i % KV4_PAGE;
  };
#pragma unroll 1
  for (int first = 0; first < rows; first += KV4_EXACT) {
    int tok[KV4_EXACT], kvlen[KV4_EXACT], start[KV4_EXACT];
    size_t to[KV4_EXACT];  // the row of (token, head)
    unsigned long long tm[KV4_EXACT];
    const T* q[KV4_EXACT];
#pragma unroll
    for (int i = 0; i < KV4_EXACT; ++i) {
      const int row = pc.row0 + min(first + i, rows - 1), head = pc.hk * p.group + row % p.group;
      tok[i] = pc.qstart + row / p.group;
      to[i] = static_cast<size_t>(tok[i]) * p.hq + head;
      q[i] = reinterpret_cast<const T*>(p.q) + static_cast<size_t>(tok[i]) * p.q_stride + head * D;
      kvlen[i] = p.q_kvlen[tok[i]];
      start[i] = EXT && p.q_kvstart ? p.q_kvstart[tok[i]] : 0;
      tm[i] = EXT && p.tree_mask ? p.tree_mask[tok[i]] : 0ull;
    }
    auto sees = [&](int i, int pos) { return kv4_visible(pos, kvlen[i], start[i], p.sink, tm[i]); };
    float M[KV4_EXACT], L[KV4_EXACT], acc[KV4_EXACT][8];
    kv4_rows_exact<T, D>(p.pages, p.num_pages, p.page_indices + pc.list0, p.hkv, pc.hk, q, 1.f, p.scale_log2,
                         EXT ? p.cap_k : 0.f, EXT ? p.cap_log2 : 0.f, pc.slots * 2 * KV4_PAGE, at, sees, M, L, acc);
#pragma unroll
    for (int i = 0; i < KV4_EXACT; ++i) {
      if (first + i >= rows) continue;
      if (pc.part >= 0) {
        const size_t part = static_cast<size_t>(pc.part) * 16 + first + i;
        if (lane < D / 8) kv4_put8(p.part_o + part * D + lane * 8, acc[i]);
        if (lane == 0) reinterpret_cast<float2*>(p.part_ml)[part] = make_float2(M[i], L[i]);
      } else {
        if (lane < D / 8) kv4_put8(reinterpret_cast<T*>(p.out) + to[i] * D + lane * 8, acc[i], L[i] == 0.f ? 0.f : 1.f / L[i]);
        if (p.lse && lane == 0) p.lse[to[i]] = L[i] == 0.f ? -INFINITY : (M[i] + log2f(L[i])) * 0.6931471805599453f;
      }
    }
  }
}

template <int D, int NT>
struct Kv4DecShape {
  static constexpr int ROW = kv4_row_bytes(D);
  static constexpr int PAGE_BYTES = KV4_PAGE * ROW;            // K or V of one page and head
  static constexpr int SLOT_BYTES = 4 * PAGE_BYTES;            // K, V of two pages
  static constexpr int SLOTS = D == 256 ? 4 : 8;               // a multiple of the four consumer warps
  static constexpr int ROWS = 8 * NT;
  // resident per SM: what the registers allow without spilling much (D = 128, one n-tile: 3 120 us, 4 129 us)
  static constexpr int CTAS = D == 64 ? (NT == 1 ? 4 : 3) : D == 128 ? (NT == 1 ? 3 : 2) : 2;
  // Query rows of a piece; two pieces are held. The pitch spreads a fragment's eight rows over the banks.
  static constexpr int Q_PITCH = D * 2 + 16;
  static constexpr int Q_BYTES = ROWS * Q_PITCH;
  // three warps' partial O in fragment order (16 bytes per lane, pair of tiles and column), and their (m, l), of two pieces
  static constexpr int MERGE_BYTES = 6 * (ROWS * D * 4 + ROWS * 8);
  static constexpr int OFF_Q = SLOTS * SLOT_BYTES;
  static constexpr int OFF_MERGE = OFF_Q + 2 * Q_BYTES;
  static constexpr int OFF_BAR = OFF_MERGE + MERGE_BYTES;
  static constexpr int OFF_PIECE = OFF_BAR + 8 * (2 * SLOTS + 6);
  static constexpr int OFF_SCAN = OFF_PIECE + 2 * 64;          // item prefix sums, sized by the launch
  static_assert(sizeof(Kv4Piece) <= 64, "a piece descriptor has 64 bytes");
};

// EXT: masks or a soft cap. GUARD: bf16 items of several tokens, whose rows see different positions (kv4.cuh).
template <typename T, int D, int NT, bool EXT, bool GUARD>
__global__ void __launch_bounds__(KV4_DEC_THREADS, Kv4DecShape<D, NT>::CTAS) kv4_decode_kernel(const __grid_constant__ Kv4DecParams p) {
  using Shape = Kv4DecShape<D, NT>;
  constexpr int ROW = Shape::ROW, PB = Shape::PAGE_BYTES, SLOTS = Shape::SLOTS, ROWS = Shape::ROWS;
  constexpr int GROUPS = D / KV4_GROUP;
  constexpr int VW = D / 64;   // V code words per lane and token
  constexpr bool BF16 = Kv4Type<T>::IS_BF16;
  pdl_launch_dependents();
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* merge = smem + Shape::OFF_MERGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Shape::OFF_BAR);
  uint64_t* empty = full + SLOTS;
  uint64_t* piece_full = empty + SLOTS;   // [2]
  uint64_t* piece_empty = piece_full + 2; // [2]
  uint64_t* merge_full = piece_empty + 2; // [2]
  Kv4Piece* pieces = reinterpret_cast<Kv4Piece*>(smem + Shape::OFF_PIECE);  // [2], 64 bytes apart
  int* scan = reinterpret_cast<int*>(smem + Shape::OFF_SCAN);               // [num_items + 1]
  __shared__ int abort_word;
  __shared__ int wide[2];  // bf16: a piece's rows do not share a scale (kv4.cuh)
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < SLOTS) {
    mbar_init(&full[threadIdx.x], 1);
    mbar_init(&empty[threadIdx.x], 1);
  }
  if (threadIdx.x < 2) {
    mbar_init(&piece_full[threadIdx.x], 1);
    mbar_init(&piece_empty[threadIdx.x], 4);
    mbar_init(&merge_full[threadIdx.x], 3);
  }
  mbar_fence_init();
  if (threadIdx.x == 0) {
    abort_word = 0;
    // "nothing cut here" until the producer's last piece says otherwise: the second kernel takes counts and addresses from this
    // word, and runs as well after a wait that ran out has ended the producer early
    p.part_unit[blockIdx.x * 4] = 0;
  }
  // slots of every item over its row blocks (an item without a visible position takes one, so that its rows get written)
  for (int i = threadIdx.x; i < p.num_items; i += KV4_DEC_THREADS) {
    const Kv4Item d = kv4_item<EXT, ROWS>(p, i);
    scan[i] = max(1, (d.npg + 1) >> 1) * d.blocks;
  }
  __syncthreads();
  if (warp == 0) {
    int sum = 0;
    for (int base = 0; base < p.num_items; base += 32) {
      const int n = base + lane < p.num_items ? scan[base + lane] : 0;
      int x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (base + lane < p.num_items) scan[base + lane] = sum + x - n;
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) scan[p.num_items] = sum;
  }
  __syncthreads();
  const long long total = static_cast<long long>(scan[p.num_items]) * p.hkv;
  const long long share = max((total + gridDim.x - 1) / gridDim.x, static_cast<long long>(KV4_DEC_MIN_SHARE));
  const long long begin = blockIdx.x * share, end = min(total, begin + share);
  if (begin >= end) return;

  if (warp == 4) {
    // ---------------------------------------------------------------- producer
    int lo = 0, hi = p.num_items - 1;  // the item that holds slot `begin`
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (static_cast<long long>(scan[mid]) * p.hkv <= begin) lo = mid;
      else hi = mid - 1;
    }
    int item = lo;
    long long at = begin;
    uint32_t g = 0, k = 0;
    bool ok = true;
    Kv4Item d = kv4_item<EXT, ROWS>(p, item);
    while (at < end && ok) {
      if (at >= static_cast<long long>(scan[item + 1]) * p.hkv) d = kv4_item<EXT, ROWS>(p, ++item);
      const int n = (scan[item + 1] - scan[item]) / d.blocks;
      const int local = static_cast<int>(at - static_cast<long long>(scan[item]) * p.hkv);
      const int unit = local / n, slot0 = local % n;
      const int take = static_cast<int>(min(static_cast<long long>(n - slot0), end - at));
      const bool begins = slot0 == 0, ends = slot0 + take == n;
      const int hk = unit / d.blocks, row0 = unit % d.blocks * ROWS;
      const int rows = min(ROWS, d.ntok * p.group - row0);
      // ---- descriptor and query rows
      const int e = k & 1;
      if (k >= 2) {
        ok = mbar_wait(&piece_empty[e], ((k >> 1) & 1) ^ 1, abort_flag, p.status, ERR_WAIT_PRODUCER);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      if (lane == 0) {
        Kv4Piece* pc = reinterpret_cast<Kv4Piece*>(reinterpret_cast<uint8_t*>(pieces) + e * 64);
        pc->qstart = d.qstart;
        pc->ntok = d.ntok;
        pc->hk = hk;
        pc->row0 = row0;
        pc->slot0 = slot0;
        pc->slots = min(take, (d.npg + 1) / 2 - slot0);
        pc->npg = d.npg;
        pc->sink_pg = d.sink_pg;
        pc->skip = d.skip;
        pc->all_from = d.all_from;
        pc->all_to = d.all_to;
        pc->list0 = static_cast<int>(d.list - p.page_indices);
        wide[e] = 0;
        pc->part = begins && ends ? -1 : static_cast<int>(blockIdx.x) * 2 + (begins ? 1 : 0);
        pc->last = at + take >= end;
        if (at + take >= end) {
          // pieces of a unit that begins here and runs on: this share's and those of the CTAs after it
          const long long rest = n - take;
          int* pu = p.part_unit + blockIdx.x * 4;
          pu[0] = begins && !ends ? max(0, rows) : 0;
          pu[1] = d.qstart;
          pu[2] = hk * 16 + row0;
          pu[3] = 1 + static_cast<int>((rest + share - 1) / share);
        }
        mbar_expect_tx(&piece_full[e], max(0, rows) * D * 2);
      }
      __syncwarp();
      if (lane < rows) {
        const int row = row0 + lane;
        const uint8_t* src = reinterpret_cast<const uint8_t*>(p.q) +
                             (static_cast<size_t>(d.qstart + row / p.group) * p.q_stride +
                              static_cast<size_t>(hk * p.group + row % p.group) * D) * 2;
        bulk_load(smem + Shape::OFF_Q + e * Shape::Q_BYTES + lane * Shape::Q_PITCH, src, D * 2, &piece_full[e]);
      }
      ++k;
      // ---- pages: lane i holds the address of page base + i (one coalesced load of page numbers per 32) and issues
      // its two copies, K and V, when its slot's turn comes
      const int pg0 = slot0 * 2, pg1 = min(d.npg, (slot0 + take) * 2);
      for (int base = pg0; base < pg1 && ok; base += 32) {
        const int m = min(32, pg1 - base);
        const uint8_t* src = p.pages;
        if (lane < m) {
          const int li = base + lane;
          int pg = d.list[li < d.sink_pg ? li : li + d.skip];
          if (pg >= p.num_pages) {
            if (p.status) atomicCAS(p.status, 0, ERR_BAD_INDEX);
            pg = 0;
          }
          // a negative page was released by a sliding window: every position of it is masked
          src += (static_cast<size_t>(max(pg, 0)) * 2 * p.hkv + hk) * PB;
        }
        for (int i = 0; i < m; i += 2, ++g) {
          const int s = g % SLOTS;
          if (g >= SLOTS) {
            ok = mbar_wait(&empty[s], ((g / SLOTS) & 1) ^ 1, abort_flag, p.status, ERR_WAIT_PRODUCER);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
          if (lane == i) mbar_expect_tx(&full[s], min(2, m - i) * 2 * PB);
          __syncwarp();
          if ((lane ^ i) < 2 && lane < m) {
            uint8_t* dst = smem + s * Shape::SLOT_BYTES + (lane & 1) * 2 * PB;
            bulk_load(dst, src, PB, &full[s]);
            bulk_load(dst + PB, src + static_cast<size_t>(p.hkv) * PB, PB, &full[s]);
          }
        }
      }
      at += take;
    }
    // all copies have landed before this warp leaves, also those that the consumers gave up waiting for
    for (uint32_t n = g < SLOTS ? 0 : g - SLOTS; n < g; ++n) kv4_drain(&full[n % SLOTS], (n / SLOTS) & 1);
    for (uint32_t n = k < 2 ? 0 : k - 2; n < k; ++n) kv4_drain(&piece_full[n & 1], (n >> 1) & 1);
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int r = lane >> 2, t = lane & 3;
  uint32_t g0 = 0;
  for (uint32_t k = 0;; ++k) {
    const int e = k & 1;
    bool ok = mbar_wait(&piece_full[e], (k >> 1) & 1, abort_flag, p.status, ERR_WAIT_TMA);
    ok = __all_sync(0xffffffffu, ok);
    const Kv4Piece pc = *reinterpret_cast<const Kv4Piece*>(reinterpret_cast<const uint8_t*>(pieces) + e * 64);
    if (!ok) break;  // a wait of some role ran out: the others find out by the abort flag
    const int rows = min(ROWS, pc.ntok * p.group - pc.row0);  // 0: an item without tokens
    const int npg = pc.npg;
    // Q^T fragments: lane (r, t) has channels 8 t .. 8 t + 7 of every group of row r (+ 8 per n-tile), two k-steps each.
    // They stay in shared memory, one 16-byte load per group and slot. Rows behind the last hold anything: a column of
    // the products is its own, and theirs are never written out.
    const uint8_t* q_rows = smem + Shape::OFF_Q + e * Shape::Q_BYTES + r * Shape::Q_PITCH + t * 16;
    // B fragments of the minimum / bias k-steps: sums of q over groups 2 t and 2 t + 1 of row r, leading and trailing term
    // (bf16: and a third, with -bias times it), each row scaled by a power of two so that its largest sum is in
    // [2^12, 2^13): fp16 would lose the trailing terms of small queries and the sums of large ones. `undo` is the inverse
    // for this lane's score columns, rows 2 t and 2 t + 1.
    uint32_t ql[NT][BF16 ? 4 : 2];
    float undo[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int grp = 0; grp < GROUPS; ++grp) {
        const uint4 v = *reinterpret_cast<const uint4*>(q_rows + nt * 8 * Shape::Q_PITCH + grp * 64);
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        float c[4];
        constexpr uint32_t ones = Kv4Bias<T>::ONES;
        kv4_mma<T>(c, ones, ones, ones, ones, v.x, v.y, zero);
        kv4_mma<T>(c, ones, ones, ones, ones, v.z, v.w, c);
        // c[0], c[1] are columns 2 t, 2 t + 1; column r sits in the lanes with t = r / 2
        const float x = __shfl_sync(0xffffffffu, c[0], (lane & 28) | (r >> 1));
        const float y = __shfl_sync(0xffffffffu, c[1], (lane & 28) | (r >> 1));
        if (grp / 2 == t) sum[grp & 1] = (r & 1) ? y : x;
      }
      float most = fmaxf(fabsf(sum[0]), fabsf(sum[1]));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int up = min(12 + 127 - static_cast<int>(__float_as_uint(most) >> 23), 126);  // >= -116
      sum[0] *= exp2f(static_cast<float>(up));
      sum[1] *= exp2f(static_cast<float>(up));
#pragma unroll
      for (int c = 0; c < 2; ++c) undo[nt][c] = exp2f(static_cast<float>(-__shfl_sync(0xffffffffu, up, (2 * t + c) * 4)));
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        const float h0 = Cvt<T>::to_f(Cvt<T>::from_f(sum[0])), h1 = Cvt<T>::to_f(Cvt<T>::from_f(sum[1]));
        ql[nt][k2] = Kv4Type<T>::pack(h0, h1);
        sum[0] -= h0;
        sum[1] -= h1;
      }
      if constexpr (BF16) {
        ql[nt][2] = Kv4Type<T>::pack(sum[0], sum[1]);
        ql[nt][3] = Kv4Type<T>::pack(sum[0] * -Kv4Bias<T>::BIAS, sum[1] * -Kv4Bias<T>::BIAS);
      }
    }
    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2];
    int v_exp = -1000;  // bf16: V is scaled by 2^-v_exp into fp16's range
    int v_all = -1000, v_part = -1000;  // the largest need of positions that every row sees (a lane's), and of others
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // A column behind the last row has an infinite maximum, weights of 0 and never asks for a rescaling: it holds the
      // products of whatever the shared memory held, which must not decide when the warp's live rows are rounded.
#pragma unroll
      for (int c = 0; c < 2; ++c) m[nt][c] = nt * 8 + 2 * t + c < rows ? -INFINITY : INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
    }
    for (int i = (warp - static_cast<int>(g0 & 3u)) & 3; i < pc.slots && ok; i += 4) {
      const uint32_t g = g0 + static_cast<uint32_t>(i);
      const int s = g % SLOTS;
      ok = mbar_wait(&full[s], (g / SLOTS) & 1, abort_flag, p.status, ERR_WAIT_TMA);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint8_t* slot = smem + s * Shape::SLOT_BYTES;
      // ---- S^T = K Q^T
      float sc[2][NT][4];
      uint32_t m0[2][GROUPS], m1[2][GROUPS];  // (lo, s) of tokens r and r + 8
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
        const uint8_t* k0 = slot + pg * 2 * PB + r * ROW + D / 2;
        // k-slots 2 t, 2 t + 1 (and those + 8) are groups 2 t, 2 t + 1: minima in one product, steps in the other. Where
        // there are fewer groups than slots ql is 0 and any group's words do.
        const int go = (2 * t) % GROUPS * 4;
        const uint2 x = *reinterpret_cast<const uint2*>(k0 + go), y = *reinterpret_cast<const uint2*>(k0 + 8 * ROW + go);
        const uint32_t lo0 = __byte_perm(x.x, x.y, 0x5410), lo1 = __byte_perm(y.x, y.y, 0x5410);
        const uint32_t st0 = __byte_perm(x.x, x.y, 0x7632), st1 = __byte_perm(y.x, y.y, 0x7632);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float zero[4] = {0.f, 0.f, 0.f, 0.f};
          float a[4], b[4];
          kv4_mma<T>(a, lo0, lo1, lo0, lo1, ql[nt][0], ql[nt][1], zero);
          kv4_mma<T>(b, st0, st1, st0, st1, ql[nt][0], ql[nt][1], zero);
          if constexpr (BF16) kv4_mma<T>(a, lo0, lo1, st0, st1, ql[nt][2], ql[nt][3], a);
#pragma unroll
          for (int c = 0; c < 4; ++c) sc[pg][nt][c] = fmaf(b[c], -Kv4Bias<T>::BIAS, a[c]) * undo[nt][c & 1];
        }
        kv4_words<GROUPS>(k0, m0[pg]);
        kv4_words<GROUPS>(k0 + 8 * ROW, m1[pg]);
      }
#pragma unroll
      for (int grp = 0; grp < GROUPS; ++grp) {
        uint4 q[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) q[nt] = *reinterpret_cast<const uint4*>(q_rows + nt * 8 * Shape::Q_PITCH + grp * 64);
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
          const uint8_t* k0 = slot + pg * 2 * PB + r * ROW + grp * 16 + t * 4;
          uint32_t e0[4], e1[4];
          kv4_raw4<T>(*reinterpret_cast<const uint32_t*>(k0), e0);
          kv4_raw4<T>(*reinterpret_cast<const uint32_t*>(k0 + 8 * ROW), e1);
          const float s0 = kv4_step<T>(m0[pg][grp]), s1 = kv4_step<T>(m1[pg][grp]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float zero[4] = {0.f, 0.f, 0.f, 0.f};
            float c[4];
            kv4_mma<T>(c, e0[0], e1[0], e0[1], e1[1], q[nt].x, q[nt].y, zero);
            kv4_mma<T>(c, e0[2], e1[2], e0[3], e1[3], q[nt].z, q[nt].w, c);
            sc[pg][nt][0] = fmaf(s0, c[0], sc[pg][nt][0]);
            sc[pg][nt][1] = fmaf(s0, c[1], sc[pg][nt][1]);
            sc[pg][nt][2] = fmaf(s1, c[2], sc[pg][nt][2]);
            sc[pg][nt][3] = fmaf(s1, c[3], sc[pg][nt][3]);
          }
        }
      }
      // ---- scale, cap, mask. A slot that every row sees in full (all but the ends of a sequence or window) skips
      // the per-element test; the others also drop V of tokens that no row sees, whatever their bytes hold.
      const int pi = (pc.slot0 + i) * 2;
      const bool two = pi + 1 < npg;
      const int at0 = (!EXT || pi < pc.sink_pg ? pi : pi + pc.skip) * KV4_PAGE;
      const int at1 = two ? (!EXT || pi + 1 < pc.sink_pg ? pi + 1 : pi + 1 + pc.skip) * KV4_PAGE : 0x3fffffff;
      bool plain = at1 + KV4_PAGE <= pc.all_to;
      if (EXT) plain = plain && (at0 >= pc.all_from || at0 + KV4_PAGE <= p.sink) && (at1 >= pc.all_from || at1 + KV4_PAGE <= p.sink);
      uint32_t seen = 0xffffffffu;
#pragma unroll
      for (int pg = 0; pg < 2; ++pg)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float v = sc[pg][nt][c];
            sc[pg][nt][c] = EXT && p.cap_log2 != 0.f ? kv4_softcap(v, p.cap_k, p.cap_log2) : v * p.scale_log2;
          }
      if (!plain) {
        auto sees = [&](int pos, int tok) {
          return kv4_visible(pos, p.q_kvlen[tok], EXT && p.q_kvstart ? p.q_kvstart[tok] : 0, p.sink,
                             EXT && p.tree_mask ? p.tree_mask[tok] : 0ull);
        };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int row = nt * 8 + 2 * t + c;
            const bool live = row < rows;
            const int tok = pc.qstart + (live ? (pc.row0 + row) / p.group : 0);
#pragma unroll
            for (int pg = 0; pg < 2; ++pg)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (!live || !sees((pg ? at1 : at0) + r + h * 8, tok)) sc[pg][nt][c + 2 * h] = -INFINITY;
          }
        const int pos = (lane < 16 ? at0 : at1) + (lane & 15);  // lane = token of the slot
        bool any = false, every = true;
        for (int q = 0; q < pc.ntok; ++q) {
          const bool it = sees(pos, pc.qstart + q);
          any = any || it;
          every = every && it;
        }
        seen = __ballot_sync(0xffffffffu, any);
        if (GUARD && pc.ntok > 1) {
          // what only some rows see must not crowd out what others see when V is scaled (kv4.cuh)
          uint32_t vm[GROUPS], most = 0;
          kv4_words<GROUPS>(slot + ((lane >> 4) * 2 + 1) * PB + (lane & 15) * ROW + D / 2, vm);
#pragma unroll
          for (int grp = 0; grp < GROUPS; ++grp) most = __vmaxu2(most, vm[grp] & 0xffff7fffu);
          const int one = any ? kv4_need(most) : KV4_NEEDS_NONE;
          v_part = max(v_part, __reduce_max_sync(0xffffffffu, one > KV4_NEEDS_NONE && !every ? one : -1000));
          const int low = __reduce_min_sync(0xffffffffu, one > KV4_NEEDS_NONE ? one : 1000);
          if (v_part > max(__reduce_max_sync(0xffffffffu, v_all), low) + KV4_WIDE && lane == 0) wide[e] = 1;
        }
      }
      // ---- running maximum (raised lazily) and P
      bool raise = false;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          top[nt][c] = fmaxf(fmaxf(sc[0][nt][c], sc[0][nt][c + 2]), fmaxf(sc[1][nt][c], sc[1][nt][c + 2]));
          raise = raise || top[nt][c] > m[nt][c] + 8.f;
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = top[nt][c];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float mn = fmaxf(m[nt][c], x);
            const float a = m[nt][c] == -INFINITY ? 1.f : exp2f(m[nt][c] - mn);  // nothing accumulated before
            m[nt][c] = mn;
            l[nt][c] *= a;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              o[nt][j][c] *= a;
              o[nt][j][c + 2] *= a;
            }
          }
      }
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float2 shift = make_float2(m[nt][0] == -INFINITY ? 0.f : -m[nt][0], m[nt][1] == -INFINITY ? 0.f : -m[nt][1]);
        float2 ls = make_float2(l[nt][0], l[nt][1]);
#pragma unroll
        for (int pg = 0; pg < 2; ++pg)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 x = kv4_add2(make_float2(sc[pg][nt][2 * h], sc[pg][nt][2 * h + 1]), shift);
            const float2 w = make_float2(exp2f(x.x), exp2f(x.y));
            ls = kv4_add2(ls, w);
            pb[pg][nt][h] = kv4_movmatrix(Kv4Type<__half>::pack(w.x, w.y));
          }
        l[nt][0] = ls.x;
        l[nt][1] = ls.y;
      }
      // ---- O^T += V^T P^T: this lane expands channels [r D / 8, (r + 1) D / 8) of tokens 2t, 2t+1, 2t+8, 2t+9
      uint32_t meta[2][4];
#pragma unroll
      for (int pg = 0; pg < 2; ++pg)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          meta[pg][x] = *reinterpret_cast<const uint32_t*>(slot + (pg * 2 + 1) * PB + (2 * t + (x & 1) + (x >> 1) * 8) * ROW +
                                                           D / 2 + (r * (D / 8) / KV4_GROUP) * 4);
          if (!plain && !((seen >> (pg * 16 + 2 * t + (x & 1) + (x >> 1) * 8)) & 1u)) meta[pg][x] = 0u;
        }
      float shrink = 1.f;
      if constexpr (BF16) {
        // A larger value raises v_exp for good (O is rescaled). The largest lies between 2^9 and 2^14 then (v_exp is a multiple
        // of 4): values keep their 11 bits down to 2^-23 of it.
        uint32_t top = 0;
#pragma unroll
        for (int pg = 0; pg < 2; ++pg)
#pragma unroll
          for (int x = 0; x < 4; ++x) top = __vmaxu2(top, meta[pg][x] & 0xffff7fffu);
        const int need = kv4_need(top);
        if (GUARD && plain) v_all = max(v_all, need);
        if (__any_sync(0xffffffffu, need > v_exp)) {
          const int e2 = (__reduce_max_sync(0xffffffffu, need) + 1027) / 4 * 4 - 1024;  // in steps of 4
          const float f = v_exp == -1000 ? 1.f : exp2f(static_cast<float>(max(v_exp - e2, -126)));
          v_exp = max(e2, -120);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
#pragma unroll
              for (int c = 0; c < 4; ++c) o[nt][j][c] *= f;
        }
        shrink = exp2f(static_cast<float>(-v_exp));
      }
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
        const uint8_t* vb = slot + (pg * 2 + 1) * PB + 2 * t * ROW + r * (D / 16);
        uint32_t w[4][VW];
#pragma unroll
        for (int x = 0; x < 4; ++x) kv4_words<VW>(vb + ((x & 1) + (x >> 1) * 8) * ROW, w[x]);
        uint32_t lo[2], st[2];  // of token pairs (2t, 2t+1) and (2t+8, 2t+9), in fp16
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t ma = meta[pg][2 * x], mb = meta[pg][2 * x + 1];
          if constexpr (BF16) {
            lo[x] = Kv4Type<__half>::pack(__uint_as_float(ma << 16) * shrink, __uint_as_float(mb << 16) * shrink);
            st[x] = Kv4Type<__half>::pack(__uint_as_float(ma & 0xffff0000u) * shrink, __uint_as_float(mb & 0xffff0000u) * shrink);
          } else {
            lo[x] = __byte_perm(ma, mb, 0x5410);
            st[x] = __byte_perm(ma, mb, 0x7632);
          }
        }
#pragma unroll
        for (int i2 = 0; i2 < VW; ++i2) {
          uint32_t a0[4], a1[4], a2[4], a3[4];
          Kv4Type<__half>::expand4(__byte_perm(w[0][i2], w[1][i2], 0x5410), st[0], lo[0], a0);
          Kv4Type<__half>::expand4(__byte_perm(w[0][i2], w[1][i2], 0x7632), st[0], lo[0], a1);
          Kv4Type<__half>::expand4(__byte_perm(w[2][i2], w[3][i2], 0x5410), st[1], lo[1], a2);
          Kv4Type<__half>::expand4(__byte_perm(w[2][i2], w[3][i2], 0x7632), st[1], lo[1], a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              kv4_mma<__half>(o[nt][i2 * 4 + x], a0[x], a1[x], a2[x], a3[x], pb[pg][nt][0], pb[pg][nt][1], o[nt][i2 * 4 + x]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
    g0 += static_cast<uint32_t>(max(0, pc.slots));
    if (!ok) break;
    // ---------------------------------------------------------------- merge the four warps of the unit
    // The warps take turns: three leave their results in shared memory in fragment order and go on to the next piece, the
    // fourth adds them to its own in a fixed order. A lane keeps its place, so the accesses are whole 512-byte rows and
    // the arithmetic stays in registers. A piece's buffers and barrier come round with its descriptor's: all four warps
    // have released piece k - 2, and with it read its buffers, before piece k is handed out.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 4);
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 8);
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 16);
      }
    if constexpr (BF16) {
      if (GUARD && v_part > -1000) {
        const int all = __reduce_max_sync(0xffffffffu, v_all);
        if (all > KV4_NEEDS_NONE && v_part > all + KV4_WIDE && lane == 0) wide[e] = 1;
      }
      const float f = exp2f(static_cast<float>(max(v_exp, -126)));  // untouched (-1000): o is 0
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[nt][j][c] *= f;
    }
    auto give = [&](int b) {
      float4* dst = reinterpret_cast<float4*>(merge + b * (ROWS * D * 4)) + lane;
      float* ml = reinterpret_cast<float*>(merge + 6 * ROWS * D * 4 + b * ROWS * 8);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
          dst[(nt * (D / 16) + j) * 32] = make_float4(o[nt][j][0], o[nt][j][1], o[nt][j][2], o[nt][j][3]);
        if (r == 0)
          reinterpret_cast<float4*>(ml)[nt * 4 + t] = make_float4(m[nt][0], l[nt][0], m[nt][1], l[nt][1]);
      }
    };
    auto take = [&](int b) {
      const float4* src = reinterpret_cast<const float4*>(merge + b * (ROWS * D * 4)) + lane;
      const float* ml = reinterpret_cast<const float*>(merge + 6 * ROWS * D * 4 + b * ROWS * 8);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float4 x = reinterpret_cast<const float4*>(ml)[nt * 4 + t];
        const float M0 = fmaxf(m[nt][0], x.x), M1 = fmaxf(m[nt][1], x.z);
        const float a0 = m[nt][0] == -INFINITY ? 0.f : exp2f(m[nt][0] - M0), a1 = m[nt][1] == -INFINITY ? 0.f : exp2f(m[nt][1] - M1);
        const float b0 = x.x == -INFINITY ? 0.f : exp2f(x.x - M0), b1 = x.z == -INFINITY ? 0.f : exp2f(x.z - M1);
        l[nt][0] = l[nt][0] * a0 + x.y * b0;
        l[nt][1] = l[nt][1] * a1 + x.w * b1;
        m[nt][0] = M0;
        m[nt][1] = M1;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          const float4 y = src[(nt * (D / 16) + j) * 32];
          o[nt][j][0] = o[nt][j][0] * a0 + y.x * b0;
          o[nt][j][1] = o[nt][j][1] * a1 + y.y * b1;
          o[nt][j][2] = o[nt][j][2] * a0 + y.z * b0;
          o[nt][j][3] = o[nt][j][3] * a1 + y.w * b1;
        }
      }
    };
    const int turn = (warp - static_cast<int>(k & 3u)) & 3;  // 0: this warp joins
    if (turn) {
      give(e * 3 + turn - 1);
      __syncwarp();
      if (lane == 0) mbar_arrive(&merge_full[e]);
    } else {
      ok = mbar_wait(&merge_full[e], (k >> 1) & 1, abort_flag, p.status, ERR_WAIT_EPILOGUE);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      __syncwarp();
      if (GUARD && wide[e]) {
        if constexpr (GUARD)
          kv4_piece_exact<T, D, EXT>(p, reinterpret_cast<const Kv4Piece*>(reinterpret_cast<const uint8_t*>(pieces) + e * 64), rows);
      } else {
#pragma unroll 1
        for (int b = 0; b < 3; ++b) take(e * 3 + b);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int row = nt * 8 + 2 * t + c;
            if (row >= rows) continue;
            if (pc.part >= 0) {
              const size_t at = static_cast<size_t>(pc.part) * 16 + row;
              float2* dst = reinterpret_cast<float2*>(p.part_o + at * D + r * (D / 8));
#pragma unroll
              for (int j = 0; j < D / 16; ++j) dst[j] = make_float2(o[nt][j][c], o[nt][j][c + 2]);
              if (r == 0) reinterpret_cast<float2*>(p.part_ml)[at] = make_float2(m[nt][c], l[nt][c]);
            } else {
              // a row that sees nothing is 0; NaN stays NaN
              const float L = l[nt][c], inv = L == 0.f ? 0.f : 1.f / L;
              const size_t at = static_cast<size_t>(pc.qstart + (pc.row0 + row) / p.group) * p.hq + pc.hk * p.group +
                                (pc.row0 + row) % p.group;
              uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + at * D + r * (D / 8));
#pragma unroll
              for (int j = 0; j < D / 16; ++j) dst[j] = Kv4Type<T>::pack(o[nt][j][c] * inv, o[nt][j][c + 2] * inv);
              if (p.lse && r == 0) p.lse[at] = L == 0.f ? -INFINITY : (m[nt][c] + log2f(L)) * 0.6931471805599453f;
            }
          }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&piece_empty[e]);
    if (pc.last) break;
  }
}

// Joins the pieces of the units that were cut: block c has the unit that began in CTA c's share, if any. Its first
// piece is that CTA's last, the others are the first pieces of the CTAs after it.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_decode_merge_kernel(const Kv4DecParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 pu = reinterpret_cast<const int4*>(p.part_unit)[blockIdx.x];
  const int rows = pu.x, qstart = pu.y, hk = pu.z >> 4, row0 = pu.z & 15, pieces = pu.w;
  for (int row = warp; row < rows; row += 4) {
    auto block = [&](int i) { return (i == 0 ? blockIdx.x * 2 + 1 : (blockIdx.x + i) * 2) * static_cast<size_t>(16) + row; };
    // running maximum over batches of four pieces, whose loads are issued together
    float M = -INFINITY, L = 0.f, acc[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) acc[c] = 0.f;
    for (int base = 0; base < pieces; base += 4) {
      float2 ml[4];
      float v[4][D / 32];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f);
        if (base + i < pieces) {
          const size_t b = block(base + i);
          ml[i] = reinterpret_cast<const float2*>(p.part_ml)[b];
#pragma unroll
          for (int c = 0; c < D / 32; ++c) v[i][c] = p.part_o[b * D + c * 32 + lane];
        }
      }
      const float Mn = fmaxf(M, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)));
      const float f = M == -INFINITY ? 0.f : exp2f(M - Mn);
      L *= f;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) acc[c] *= f;
      M = Mn;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (base + i >= pieces) continue;
        const float w = ml[i].x == -INFINITY ? 0.f : exp2f(ml[i].x - M);
        L += ml[i].y * w;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) acc[c] = fmaf(v[i][c], w, acc[c]);
      }
    }
    kv4_finish_row<T, D>(p, qstart, hk, row0 + row, M, L, acc);
  }
}

template <typename T, int D, int NT, bool EXT, bool GUARD>
int kv4_decode_launch(Kv4DecParams p, int num_items, int max_ctas, cudaStream_t stream) {
  using Shape = Kv4DecShape<D, NT>;
  auto kern = kv4_decode_kernel<T, D, NT, EXT, GUARD>;
  const int batch = num_items < KV4_DEC_ITEMS ? num_items : KV4_DEC_ITEMS;
  const int most = Shape::OFF_SCAN + (KV4_DEC_ITEMS + 1) * 4;
  static int per_sm[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return static_cast<int>(err);
  dev &= 63;
  if (!per_sm[dev]) {
    err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (err != cudaSuccess) return static_cast<int>(err);
    int n = 0;
    err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, KV4_DEC_THREADS, most);
    if (err != cudaSuccess) return static_cast<int>(err);
    per_sm[dev] = n > 0 ? n : 1;
  }
  int ctas = per_sm[dev] * sm_count();
  if (ctas > max_ctas) ctas = max_ctas;
  for (int first = 0; first < num_items; first += batch) {
    Kv4DecParams part = p;
    part.item_seq += first;
    part.item_qstart += first;
    part.item_ntok += first;
    part.num_items = num_items - first < batch ? num_items - first : batch;
    kern<<<ctas, KV4_DEC_THREADS, Shape::OFF_SCAN + (part.num_items + 1) * 4, stream>>>(part);
    err = cudaGetLastError();  // the second kernel reads what this one wrote
    if (err != cudaSuccess) return static_cast<int>(err);
    count_launch();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(128);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    err = cudaLaunchKernelEx(&cfg, kv4_decode_merge_kernel<T, D>, part);
    if (err != cudaSuccess) return static_cast<int>(err);
    count_launch();
  }
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int D, int NT>
int kv4_decode_kind(const Kv4DecParams& p, bool ext, bool several, int num_items, int max_ctas, cudaStream_t stream) {
  if constexpr (Kv4Type<T>::IS_BF16) {
    // Items of one token skip the guard: 256 sequences of 512 to 2048, bf16, 133 us without and 141 with it; 64 causal verify
    // chunks of four tokens 117 without (and wrong beside an infinity) and 121 with it.
    if (several)
      return ext ? kv4_decode_launch<T, D, NT, true, true>(p, num_items, max_ctas, stream)
                 : kv4_decode_launch<T, D, NT, false, true>(p, num_items, max_ctas, stream);
  }
  return ext ? kv4_decode_launch<T, D, NT, true, false>(p, num_items, max_ctas, stream)
             : kv4_decode_launch<T, D, NT, false, false>(p, num_items, max_ctas, stream);
}

template <typename T, int D>
int kv4_decode_shape(Kv4DecParams& p, int rows, bool ext, int num_items, int max_ctas, cudaStream_t stream) {
  // Up to 8 query rows need one n-tile. 9 to 16 rows take two, which share the expanded V; at D = 256 the
  // accumulators of two would not fit the register file, and two units read the same pages instead.
  const bool several = rows > p.group;  // tokens in an item
  if constexpr (D < 256) {
    if (rows > 8) {
      p.row_blocks = 1;
      return kv4_decode_kind<T, D, 2>(p, ext, several, num_items, max_ctas, stream);
    }
  }
  p.row_blocks = (rows + 7) / 8;
  return kv4_decode_kind<T, D, 1>(p, ext, several, num_items, max_ctas, stream);
}

}  // namespace mlcb

using namespace mlcb;

// One layer's cache [num_pages, 2, hkv, 16, row]. Items are (sequence, query-token range) pairs of at most `rows`
// <= 16 query rows (tokens * hq / hkv) each. Scratch for max_ctas CTAs: part_o [2 max_ctas, 16, d] and part_ml
// [2 max_ctas, 16, 2] fp32, part_unit [max_ctas, 4] int32; it is written before it is read. Returns -1 shape,
// -2 alignment, -3 type, -4 missing scratch.
MLCB_API int mlcb_kv4_decode(const void* q, const void* pages, void* out, float* lse, const int* item_seq,
                             const int* item_qstart, const int* item_ntok, const int* q_kvlen, const int* page_indptr,
                             const int* page_indices, int num_items, int rows, long long q_stride, int hq, int hkv, int d,
                             long long num_pages, float sm_scale, int dtype, int max_ctas, float* part_o, float* part_ml,
                             int* part_unit, int* status, cudaStream_t stream, const int* q_kvstart,
                             const unsigned long long* tree_mask, int sink, float softcap) {
  if (num_items <= 0) return 0;
  if (hkv <= 0 || hq <= 0 || hq % hkv || rows < 1 || rows > 16 || (d != 64 && d != 128 && d != 256)) return -1;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pages) | reinterpret_cast<uintptr_t>(part_unit)) & 15)
    return -2;
  if (q_stride % 8) return -2;
  if (dtype != 0 && dtype != 1) return -3;
  if (max_ctas < 1 || !part_o || !part_ml || !part_unit) return -4;
  Kv4DecParams p;
  p.q = q;
  p.pages = static_cast<const uint8_t*>(pages);
  p.out = out;
  p.lse = lse;
  p.part_o = part_o;
  p.part_ml = part_ml;
  p.part_unit = part_unit;
  p.item_seq = item_seq;
  p.item_qstart = item_qstart;
  p.item_ntok = item_ntok;
  p.q_kvlen = q_kvlen;
  p.page_indptr = page_indptr;
  p.page_indices = page_indices;
  p.q_kvstart = q_kvstart;
  p.tree_mask = tree_mask;
  p.status = status;
  p.q_stride = q_stride;
  p.num_pages = num_pages;
  p.hq = hq;
  p.hkv = hkv;
  p.group = hq / hkv;
  p.row_blocks = 1;
  p.num_items = num_items;
  p.sink = q_kvstart ? sink : 0;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.cap_k = softcap > 0.f ? 2.f * 1.4426950408889634f * sm_scale / softcap : 0.f;
  p.cap_log2 = softcap > 0.f ? softcap * 1.4426950408889634f : 0.f;
  const bool ext = q_kvstart || tree_mask || softcap > 0.f;
  if (dtype == 0) {
    if (d == 64) return kv4_decode_shape<__half, 64>(p, rows, ext, num_items, max_ctas, stream);
    if (d == 128) return kv4_decode_shape<__half, 128>(p, rows, ext, num_items, max_ctas, stream);
    return kv4_decode_shape<__half, 256>(p, rows, ext, num_items, max_ctas, stream);
  }
  if (d == 64) return kv4_decode_shape<__nv_bfloat16, 64>(p, rows, ext, num_items, max_ctas, stream);
  if (d == 128) return kv4_decode_shape<__nv_bfloat16, 128>(p, rows, ext, num_items, max_ctas, stream);
  return kv4_decode_shape<__nv_bfloat16, 256>(p, rows, ext, num_items, max_ctas, stream);
}
