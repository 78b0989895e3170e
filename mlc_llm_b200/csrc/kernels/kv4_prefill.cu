// Prefill attention over the 4-bit paged KV cache (format: kv4.cuh) on the 5th-gen tensor cores: head sizes 64, 96,
// 128 and 256, 16-token pages, any mask of the 16-bit kernels.
//
// A CTA owns up to 256 query rows of one kv head -- (token, q head) pairs, the G = hq / hkv heads of the group side
// by side -- as two accumulator tiles of 128 rows, and walks the cached positions in blocks of 128:
//
//   raw       a warp copies the blocks' packed rows (80 bytes per token at D = 128) into a ring of shared memory
//   expand    four warps turn them into fp16 K and V tiles in the layout the tensor core reads (128-byte swizzle; V
//             MN-major), lo + s c rounded once. One expansion feeds both query tiles; it hides under the rest (without
//             it 2.16 ms for 2.30, measured at a step before). bf16 rows are scaled by a power of two per block (V: of
//             the largest block so far; queries: per row) into fp16's range, so that K, V and P keep 11 bits.
//   S = Q K^T    tcgen05.mma, both operands in shared memory, D in TMEM (128 columns per tile)
//   softmax      one thread per row, 32 columns of TMEM at a time, in two passes: the block's maximum, then its weights
//                against a running reference that is raised (and O rescaled) only when a score exceeds it by more
//                than 8 (log2). One vote per block: with one per 32 columns the code between the votes could not be
//                interleaved, and a block took 2630 clocks instead of 2100. P (fp16) overwrites S in TMEM.
//   O += P V     tcgen05.mma, A = P in TMEM, B = V in shared memory, D accumulates in TMEM for the whole loop
//
// While the softmax of one tile runs, the tensor core works on the other tile. With D = 256 one tile fills TMEM (O
// takes 256 columns): blocks are 64 positions, S has two buffers, and the scores of block j + 1 are computed before
// the softmax of block j ends.
//
// Few long rows (a short chunk behind a long prefix) are split over the cached positions; fp32 partial rows are
// joined by a second kernel. Bounds: the tensor core (4 D flops per query row and position) and, as slow, the exponentials
// (one per row and position: 2048 clocks each per block at 16 per clock and SM and 8 K flops per clock).
//
// Measured, 32 / 8 heads of 128: 16384 causal tokens fp16 2.08 ms (1057 TFLOP/s), bf16 2.20 ms (one launch; back to back the power
// limit makes it 2.2 to 2.3 ms); chunks of 2000, 1500, 700 and 1800 new tokens behind 7000, 0, 0 and 3200, bf16 454 us; four
// of 512 to 2048 behind up to 8192 (641 Gflop) 710 us (903 TFLOP/s); 4 x 1024 fp16 76 us. A block takes some 4200
// clocks: a tile's softmax (2050 to 2330, latency of one warp per scheduler and tile) and then its products and hand-overs (1670
// to 2050), one after the other: P overwrites the tile's only S, so that the next scores are computed behind P V. (Two S buffers
// of 64 columns per tile, as with D = 256, would overlap them; not built.)
// Tried and slower at 16384 (2.15 ms then): 16 softmax warps 2.23, eight expanding warps 3.26, P handed over in halves 2.21;
// a quarter of the exponentials as polynomials 2.13 against 2.07.
//
// Roles: 4 warps per query tile (softmax, epilogue), 4 expanding warps, 1 copying warp, 1 issuing warp. Every wait is
// bounded (common.cuh).
#include "kv4.cuh"

namespace mlcb {

struct Kv4PreParams {
  const void* q;
  const uint8_t* pages;
  void* out;
  float* lse;
  float* part_o;   // [tiles, hkv, splits, rows, D] fp32 (splits > 1)
  float* part_ml;  // [tiles, hkv, splits, rows, 2]
  const int *tile_seq, *tile_qstart, *tile_ntok, *q_kvlen, *page_indptr, *page_indices;
  const int* q_kvstart;
  const unsigned long long* tree_mask;
  int* status;
  long long q_stride, num_pages;
  int hq, hkv, group, sink, splits, num_tiles;
  int parts;               // CTAs per tile: 2 where a tile has more than the 128 rows of a D = 256 CTA
  uint32_t q_flip;         // sign bits of a pair where sm_scale is negative: scale_log2 is its magnitude
  float scale_log2;        // sm_scale * log2(e)
  float cap_k, cap_log2;   // soft cap: scores are kv4_softcap(raw, cap_k, cap_log2); 0 = none
};

// One lane of a converged warp, in the form the compiler knows to be a single thread: what the elected lane does with
// warp-uniform values stays in uniform registers, which the tensor-core instructions take their operands from. (Issued
// under `lane == 0` an instruction took about 130 clocks, more than most of the products.)
__device__ __forceinline__ bool kv4_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

template <int D>
struct Kv4PreShape {
  static constexpr int SUB = D == 256 ? 1 : 2;           // query tiles of 128 rows
  static constexpr int BLK = D == 256 ? 64 : 128;        // cached positions per block
  static constexpr int HALVES = (D + 63) / 64;           // 64-channel atoms of a row
  static constexpr int ROW = kv4_row_bytes(D);
  static constexpr int PAGE_BYTES = KV4_PAGE * ROW;
  static constexpr int TILE_BYTES = BLK * HALVES * 128;  // one expanded K or V tile
  static constexpr int TILES = 4;                        // K, V, K, V
  static constexpr int Q_BYTES = 128 * HALVES * 128;     // one query tile
  static constexpr int RAW_BYTES = BLK * ROW;            // a raw slot: packed K or V rows of a block
  static constexpr int RAW_SLOTS = 3;
  static constexpr int CHUNKS = BLK / 32;                // a warp expands 32 positions; with two chunks for the four
  static constexpr int SHARES = 4 / CHUNKS;              // warps, two warps share the channels of each
  static constexpr int OFF_TILE = SUB * Q_BYTES;
  static constexpr int OFF_RAW = OFF_TILE + TILES * TILE_BYTES;
  static constexpr int SMEM = OFF_RAW + RAW_SLOTS * RAW_BYTES + 1024;
  // Two query tiles: four warpgroups that share the launch's 4 x 128 registers per thread as 168 + 168 + 96 + 80 (the
  // last holds the copying and the issuing warp and two idle ones). One tile: 320 threads have registers to spare.
  // Without the split (448 threads of 128) at a step before: 548 us for 484 (bf16), 2.15 ms for 2.07 (16384, fp16).
  static constexpr bool SPLIT = SUB == 2;
  static constexpr int THREADS = SPLIT ? 512 : SUB * 128 + 128 + 64;
  static constexpr int O_COL = SUB == 2 ? 256 : 128;     // TMEM: S tiles first, then O
  static constexpr int O_STEP = 128;
};

// D[tmem] (+)= A[tmem] * B[smem]; 16-bit inputs, fp32 accumulate. A holds two K-adjacent values per 32-bit column.
__device__ __forceinline__ void kv4_umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void kv4_tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void kv4_tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void kv4_tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int N, bool UP>
__device__ __forceinline__ void kv4_set_regs() {
  if constexpr (UP) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// What a CTA needs to know of its tile, found by all threads together.
struct Kv4Tile {
  int reach[2];     // per query tile: positions any of its rows sees end here
  int all_to[2];    // per query tile: every row sees [all_from, all_to)
  int all_from[2];
  int first;        // no row sees a position in [sink, first)
};

template <typename T, int D, bool EXT>
__global__ void __launch_bounds__(Kv4PreShape<D>::THREADS, 1) kv4_prefill_kernel(const Kv4PreParams p) {
  using Shape = Kv4PreShape<D>;
  constexpr int SUB = Shape::SUB, BLK = Shape::BLK, ROW = Shape::ROW;
  constexpr int GROUPS = D / KV4_GROUP;
  constexpr bool BF16 = Kv4Type<T>::IS_BF16;
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[2 * Shape::RAW_SLOTS + 2 * Shape::TILES + 10];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ Kv4Tile info;
  __shared__ int exps[4][2];  // bf16: exponents of a block's K and V; blocks j - 3 .. j are live
  __shared__ int wide_from;   // bf16: the first block at which the rows of the tile share no scale (kv4.cuh)
  uint64_t* raw_full = bars;
  uint64_t* raw_empty = raw_full + Shape::RAW_SLOTS;
  uint64_t* tile_full = raw_empty + Shape::RAW_SLOTS;
  uint64_t* tile_empty = tile_full + Shape::TILES;
  // per query tile; with D = 256 per S buffer, because a fast warp may finish block j + 1 before a slow one block j
  uint64_t* s_full = tile_empty + Shape::TILES;  // [2]
  uint64_t* p_full = s_full + 2;                 // [2]
  uint64_t* o_done = p_full + 2;                 // [SUB]
  uint64_t* pv_done = o_done + 2;                // D = 256 only
  uint64_t* q_ready = pv_done + 1;
  uint64_t* mma_idle = q_ready + 1;              // every product of this CTA is over
  uint64_t* looked = mma_idle + 1;               // wide_from is final
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.group;
  // long tiles first, of all heads: the last tiles of a sequence see the most positions, and plans put the longest last (all
  // tiles of one head before those of the next: 4 x 1024 causal tokens 82 us instead of 74)
  const int hk = blockIdx.x % p.hkv, split = blockIdx.x / p.hkv % p.splits;
  const int work = p.num_tiles * p.parts - 1 - static_cast<int>(blockIdx.x) / p.hkv / p.splits;
  const int tile = work / p.parts, row0 = work % p.parts * 128;  // first row of the tile that is this CTA's
  const int seq = p.tile_seq[tile], qstart = p.tile_qstart[tile], ntok = p.tile_ntok[tile];
  const int valid_rows = max(0, min(ntok * G - row0, SUB * 128));
  const int p0 = p.page_indptr[seq];
  const int held = p.page_indptr[seq + 1] - p0;

  // rows of several tokens see different positions: the copying warp looks out for sizes that no common scale serves (kv4.cuh)
  const bool guard = BF16 && ntok > 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < Shape::RAW_SLOTS; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], guard ? 5 : 4);
    }
    for (int i = 0; i < Shape::TILES; ++i) {
      mbar_init(&tile_full[i], 4);
      mbar_init(&tile_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(pv_done, 1);
    mbar_init(q_ready, 4 * SUB);
    mbar_init(mma_idle, 1);
    mbar_init(looked, 1);
    abort_word = 0;
    wide_from = 0x7fffffff;
    mbar_fence_init();
    for (int i = 0; i < 2; ++i) {
      info.reach[i] = 0;
      info.all_to[i] = 0x7fffffff;
      info.all_from[i] = 0;
    }
    info.first = 0x7fffffff;
  }
  constexpr int ISSUER = SUB * 4 + 5, COPIER = SUB * 4 + 4;
  if (warp == ISSUER) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  __syncthreads();
  // (the second CTA of a short tile has no rows: where G does not divide 128, row0 / G * G is below row0, and its token may be
  // behind the last one of the call)
  const int past = valid_rows > 0 ? row0 + valid_rows : 0;
  for (int i = row0 / G + threadIdx.x; i * G < past; i += Shape::THREADS) {
    const int n = p.q_kvlen[qstart + i];
    int end = n, from = 0;
    if (EXT && p.tree_mask) {
      const unsigned long long tm = p.tree_mask[qstart + i];
      if (tm) end += 64 - __clzll(tm);
    }
    if (EXT && p.q_kvstart) from = p.q_kvstart[qstart + i];
#pragma unroll
    for (int s = 0; s < SUB; ++s)
      if (i * G < row0 + (s + 1) * 128 && (i + 1) * G > row0 + s * 128) {  // a token's heads may straddle the two tiles
        atomicMax(&info.reach[s], end);
        atomicMin(&info.all_to[s], n);
        atomicMax(&info.all_from[s], from);
      }
    atomicMin(&info.first, from);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int* list = p.page_indices + p0;
  const long long room = static_cast<long long>(held) * KV4_PAGE;
  if (threadIdx.x == 0 && p.status && max(info.reach[0], info.reach[1]) > room) atomicCAS(p.status, 0, ERR_BAD_INDEX);
  // Blocks a tile visits: all up to its reach, less the run of whole blocks between the sink and the first position
  // that any row sees; of those, this split's share.
  int sink_blks = 0, skip = 0, most = 0, nblk[2] = {0, 0};
  {
    int low = 0x7fffffff;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      nblk[s] = static_cast<int>((min(static_cast<long long>(info.reach[s]), room) + BLK - 1) / BLK);
      if (s * 128 < valid_rows) low = min(low, info.reach[s]);
    }
    if (EXT && p.q_kvstart) {
      sink_blks = (p.sink + BLK - 1) / BLK;
      skip = max(0, min(info.first, low) / BLK - sink_blks);
    }
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      nblk[s] = max(0, nblk[s] - skip);
      most = max(most, nblk[s]);
    }
  }
  const int per = (most + p.splits - 1) / p.splits, j0 = split * per;
#pragma unroll
  for (int s = 0; s < SUB; ++s) nblk[s] = max(0, min(nblk[s] - j0, per));
  const int nmax = SUB == 2 ? max(nblk[0], nblk[1]) : nblk[0];
  auto base_of = [&](int j) { return (!EXT || j0 + j < sink_blks ? j0 + j : j0 + j + skip) * BLK; };

  if (warp >= COPIER) {
   if constexpr (Shape::SPLIT) kv4_set_regs<80, false>();
   if (warp == COPIER) {
    // ---------------------------------------------------------------- packed rows -> raw ring
    bool ok = true;
    int m = 0, seen = 0;  // raw slots so far, and those of them that were looked at
    int v_part = -1000, v_all = -1000;  // the largest needs of V: of positions that only some rows see, and of others behind those
    const int all_to = min(info.all_to[0], info.all_to[1]), all_from = max(info.all_from[0], info.all_from[1]);
    auto look = [&](int n) {
      const int s = n % Shape::RAW_SLOTS, j = n >> 1, base = base_of(j);
      const bool plain = base + BLK <= all_to && (!EXT || base >= all_from || base + BLK <= p.sink);
      if (!plain || ((n & 1) && v_part > -1000)) {  // most blocks are seen by every row, and nothing else came before them
        if (!__all_sync(0xffffffffu, mbar_wait(&raw_full[s], (n / Shape::RAW_SLOTS) & 1, abort_flag, p.status, ERR_WAIT_TMA))) return false;
        const int reach = static_cast<int>(min(static_cast<long long>(max(info.reach[0], info.reach[1])), room));
        const int first = EXT && p.q_kvstart ? info.first : 0;
        int all = KV4_NEEDS_NONE, part = -1000, low = 1000;  // of the block: seen by every row, others, the smallest
        for (int t = lane; t < BLK; t += 32) {
          const int pos = base + t;
          const uint32_t* pr = reinterpret_cast<const uint32_t*>(smem + Shape::OFF_RAW + s * Shape::RAW_BYTES + t * ROW + D / 2);
          uint32_t top = 0;
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) top = __vmaxu2(top, pr[g] & 0xffff7fffu);
          const int need = kv4_need(top);
          if (need <= KV4_NEEDS_NONE || pos >= reach || (pos < first && pos >= p.sink)) continue;
          if (plain) all = max(all, need);
          else if (pos >= all_to || (EXT && pos < all_from && pos >= p.sink)) part = max(part, need);
          low = min(low, need);
        }
        __syncwarp();
        all = __reduce_max_sync(0xffffffffu, all);
        part = __reduce_max_sync(0xffffffffu, part);
        low = __reduce_min_sync(0xffffffffu, low);
        bool wide = part > low + KV4_WIDE;  // K has an exponent per block
        if (n & 1) {                        // V that of the largest so far
          if (plain && all > KV4_NEEDS_NONE) v_all = max(v_all, all);
          v_part = max(v_part, part);
          wide = low < 1000 && v_part > max(v_all, plain ? -1000 : low) + KV4_WIDE;
        }
        if (wide && lane == 0 && wide_from > j) wide_from = j;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&raw_empty[s]);
      return true;
    };
    for (int j = 0; j < nmax && ok; ++j) {
      const int pg0 = base_of(j) / KV4_PAGE;
      int mine = 0;  // lane i: page number of the block's page i
      if (lane < BLK / KV4_PAGE && pg0 + lane < held) {
        mine = list[pg0 + lane];
        if (mine >= p.num_pages) {
          if (p.status) atomicCAS(p.status, 0, ERR_BAD_INDEX);
          mine = 0;
        }
        if (mine < 0) mine = 0;  // released by a sliding window: every position of it is masked
      }
      const int here = max(0, min(BLK / KV4_PAGE, held - pg0));  // pages of this block that exist
      for (int kv = 0; kv < 2; ++kv, ++m) {
        const int s = m % Shape::RAW_SLOTS;
        if (m >= Shape::RAW_SLOTS) {
          ok = mbar_wait(&raw_empty[s], ((m / Shape::RAW_SLOTS) & 1) ^ 1, abort_flag, p.status, ERR_WAIT_PRODUCER);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        if (lane == 0) mbar_expect_tx(&raw_full[s], here * Shape::PAGE_BYTES);
        __syncwarp();
        if (lane < here) {
          const size_t block = (static_cast<size_t>(mine) * 2 + kv) * p.hkv + hk;
          bulk_load(smem + Shape::OFF_RAW + s * Shape::RAW_BYTES + lane * Shape::PAGE_BYTES,
                    p.pages + block * Shape::PAGE_BYTES, Shape::PAGE_BYTES, &raw_full[s]);
        }
        if (guard && m + 1 - seen == Shape::RAW_SLOTS) {
          ok = look(seen++);
          if (!ok) break;
        }
      }
    }
    if (guard) {
      while (ok && seen < m) ok = look(seen++);
      if (ok && lane == 0) mbar_arrive(looked);
    }
    for (int n = max(0, m - Shape::RAW_SLOTS); n < m; ++n) kv4_drain(&raw_full[n % Shape::RAW_SLOTS], (n / Shape::RAW_SLOTS) & 1);
   } else if (warp == ISSUER) {
    // ---------------------------------------------------------------- tensor core
    if (nmax > 0) {
      const uint32_t idesc_qk = umma_idesc(0, 128, BLK, 0, 0);
      const uint32_t idesc_pv = umma_idesc(0, 128, D, 0, 1);
      bool ok = __all_sync(0xffffffffu, mbar_wait(q_ready, 0, abort_flag, p.status, ERR_WAIT_PRODUCER));
      auto tile_wait = [&](int n) {
        return __all_sync(0xffffffffu, mbar_wait(&tile_full[n % Shape::TILES], (n / Shape::TILES) & 1, abort_flag, p.status,
                                                 ERR_WAIT_DEQUANT)) != 0;
      };
      auto s_col = [&](int i, int j) { return tmem + (SUB == 2 ? i * 128 : (j & 1) * BLK); };
      auto qk = [&](int i, int j) {
        const uint64_t da = umma_smem_desc(smem_u32(smem + i * Shape::Q_BYTES), 16, 1024);
        const uint64_t db = umma_smem_desc(smem_u32(smem + Shape::OFF_TILE + (2 * j) % Shape::TILES * Shape::TILE_BYTES), 16, 1024);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t a = da + ((kk >> 2) * (128 * 128) + (kk & 3) * 32) / 16;
          const uint64_t b = db + ((kk >> 2) * (BLK * 128) + (kk & 3) * 32) / 16;
          umma_f16(s_col(i, j), a, b, idesc_qk, kk ? 1u : 0u);
        }
        umma_commit(&s_full[SUB == 2 ? i : j & 1]);
      };
      auto pv = [&](int i, int j) {
        const uint64_t dv = umma_smem_desc(smem_u32(smem + Shape::OFF_TILE + (2 * j + 1) % Shape::TILES * Shape::TILE_BYTES), BLK * 128, 1024);
#pragma unroll
        for (int kk = 0; kk < BLK / 16; ++kk) {
          // V: MN-major, 64-wide atoms along channels (LBO), 8-position groups (SBO)
          const uint64_t b = dv + kk * 2048 / 16;
          kv4_umma_ts(tmem + Shape::O_COL + i * Shape::O_STEP, s_col(i, j) + kk * 8, b, idesc_pv, (j | kk) ? 1u : 0u);
        }
        if (SUB == 1) umma_commit(pv_done);
      };
      auto one = [&](auto&& f) {
        if (kv4_elect()) f();
        __syncwarp();
      };
      ok = ok && tile_wait(0);
      if (ok) {
        tc_fence_after();
        one([&] {
#pragma unroll
          for (int i = 0; i < SUB; ++i)
            if (nblk[i] > 0) qk(i, 0);
          umma_commit(&tile_empty[0]);
        });
      }
      for (int j = 0; j < nmax && ok; ++j) {
        if (SUB == 1 && j + 1 < nmax) {
          ok = tile_wait(2 * j + 2);
          if (!ok) break;
          tc_fence_after();
          one([&] {
            qk(0, j + 1);
            umma_commit(&tile_empty[(2 * j + 2) % Shape::TILES]);
          });
        }
        ok = tile_wait(2 * j + 1);
#pragma unroll
        for (int i = 0; i < SUB; ++i) {
          if (!ok || j >= nblk[i]) continue;
          ok = SUB == 2 ? mbar_wait(&p_full[i], j & 1, abort_flag, p.status, ERR_WAIT_EPILOGUE)
                        : mbar_wait(&p_full[j & 1], (j >> 1) & 1, abort_flag, p.status, ERR_WAIT_EPILOGUE);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) continue;
          tc_fence_after();
          one([&] {
            pv(i, j);
            if (j + 1 == nblk[i]) umma_commit(&o_done[i]);
          });
          if (SUB == 2 && j + 1 < nblk[i]) {
            ok = tile_wait(2 * j + 2);
            if (!ok) continue;
            tc_fence_after();
            one([&] { qk(i, j + 1); });
          }
        }
        if (!ok) break;
        one([&] {
          umma_commit(&tile_empty[(2 * j + 1) % Shape::TILES]);
          if (SUB == 2 && j + 1 < nmax) umma_commit(&tile_empty[(2 * j + 2) % Shape::TILES]);
        });
      }
      one([&] { umma_commit(mma_idle); });
      kv4_drain(mma_idle, 0);
    }
   }
  } else if (warp >= SUB * 4) {
    // ---------------------------------------------------------------- expanding warps
    if constexpr (Shape::SPLIT) kv4_set_regs<96, false>();
    // A warp takes 32 positions of a block, lane = position, so the loads (row pitch 5/8 D bytes) and the swizzled
    // 16-byte stores are free of bank conflicts.
    const int w = warp - SUB * 4;
    const int chunk = w % Shape::CHUNKS, token = chunk * 32 + lane;
    constexpr int MINE = (GROUPS + Shape::SHARES - 1) / Shape::SHARES;
    const int g0 = w / Shape::CHUNKS * MINE;
    const int reach = max(info.reach[0], SUB == 2 ? info.reach[1] : 0);
    const int first = EXT && p.q_kvstart ? info.first : 0;
    int v_most = -120;
    bool ok = true;
    for (int n = 0; n < 2 * nmax && ok; ++n) {
      const int j = n >> 1;
      const int b = n % Shape::TILES;
      if (n >= Shape::TILES) {
        ok = mbar_wait(&tile_empty[b], ((n / Shape::TILES) & 1) ^ 1, abort_flag, p.status, ERR_WAIT_MMA);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      const int s = n % Shape::RAW_SLOTS;
      ok = mbar_wait(&raw_full[s], (n / Shape::RAW_SLOTS) & 1, abort_flag, p.status, ERR_WAIT_TMA);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint8_t* src = smem + Shape::OFF_RAW + s * Shape::RAW_BYTES + token * ROW;
      uint8_t* row = smem + Shape::OFF_TILE + b * Shape::TILE_BYTES + token * 128;
      // a position that no row sees counts as 0 whatever its bytes hold (its weight is 0, but 0 * NaN is not)
      const int at = base_of(j) + token;
      const bool live = at < reach && at < room && (at >= first || at < p.sink);
      const uint32_t* pairs = reinterpret_cast<const uint32_t*>(src + D / 2);
      uint32_t meta[MINE];
#pragma unroll
      for (int i = 0; i < MINE; ++i) meta[i] = live ? pairs[g0 + i] : 0u;
      float shrink = 1.f;
      if constexpr (BF16) {
        // One exponent per block for K, and for V that of the largest block so far, so that weights need no scale. Every warp
        // looks at all positions of the block: all come to the same exponent without meeting. (With one per 32 positions and
        // the weights carrying the difference P lost bits, and it took 2 % longer.) In steps of 4: the largest value lies between
        // 2^9 and 2^14 then, and values below 2^-23 of it lose bits.
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < Shape::CHUNKS; ++c) {
          const int t = c * 32 + lane, pos = base_of(j) + t;
          const uint8_t* pr = smem + Shape::OFF_RAW + s * Shape::RAW_BYTES + t * ROW + D / 2;
          uint32_t m[GROUPS];
          if constexpr (ROW % 16 == 0) {
            kv4_words<GROUPS>(pr, m);
          } else {
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) m[g] = reinterpret_cast<const uint32_t*>(pr)[g];
          }
          uint32_t most = 0;
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) most = __vmaxu2(most, m[g] & 0xffff7fffu);
          if (pos < reach && pos < room && (pos >= first || pos < p.sink)) top = __vmaxu2(top, most);
        }
        int e = max((__reduce_max_sync(0xffffffffu, kv4_need(top)) + 1027) / 4 * 4 - 1024, -120);
        if (n & 1) e = v_most = max(v_most, e);
        if (w == 0 && lane == 0) exps[j & 3][n & 1] = e;
        shrink = exp2f(static_cast<float>(-e));
      }
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const int g = g0 + i;
        uint32_t c[4], lo2, s2;
        if constexpr (ROW % 16 == 0) {
          kv4_words<4>(src + g * 16, c);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x) c[x] = reinterpret_cast<const uint32_t*>(src)[g * 4 + x];
        }
        if constexpr (BF16) {
          const float lo = __uint_as_float(meta[i] << 16) * shrink, st = __uint_as_float(meta[i] & 0xffff0000u) * shrink;
          lo2 = Kv4Type<__half>::pack(lo, lo);
          s2 = Kv4Type<__half>::pack(st, st);
        } else {
          lo2 = __byte_perm(meta[i], meta[i], 0x1010);
          s2 = __byte_perm(meta[i], meta[i], 0x3232);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint32_t v[4];
          Kv4Type<__half>::expand4(c[x], s2, lo2, v);
          const int unit = (g & 1) * 4 + x;  // 16-byte unit of the 64-channel atom
          *reinterpret_cast<uint4*>(row + (g >> 1) * (BLK * 128) + ((unit ^ (token & 7)) << 4)) =
              make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&raw_empty[s]);
        mbar_arrive(&tile_full[b]);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax / epilogue
    if constexpr (Shape::SPLIT) kv4_set_regs<168, true>();
    const int sub = warp >> 2;
    const int row = threadIdx.x & 127;                 // row of the tile
    const int grow = sub * 128 + row;                  // row of the CTA
    const bool row_valid = grow < valid_rows;
    const bool warp_active = sub * 128 + (warp & 3) * 32 < valid_rows;
    // row / G of rows below 2^20: (row + 1/2) / G is half a step of 1 / G away from any whole number
    const float per_group = 1.f / static_cast<float>(G);
    auto token_of = [&](int r) { return static_cast<int>((static_cast<float>(r) + 0.5f) * per_group); };
    const int ahead_of_row = row_valid ? token_of(row0 + grow) : 0;
    const int tok = qstart + ahead_of_row, head = hk * G + (row_valid ? row0 + grow - ahead_of_row * G : 0);
    const int kvlen = row_valid ? p.q_kvlen[tok] : 0;
    int start = 0;
    unsigned long long tm = 0ull;
    if (EXT && row_valid) {
      if (p.q_kvstart) start = p.q_kvstart[tok];
      if (p.tree_mask) tm = p.tree_mask[tok];
    }
    float row_scale = 1.f;  // of the scores, undoing that of the staged query row
    {
      // Query rows: the warp loads its 32 whole, neighbouring lanes neighbouring bytes, a batch of loads at a time (one
      // thread per row and load after load took 9000 clocks for 32 KB).
      constexpr int UNITS = D / 8, BATCH = UNITS % 8 ? 6 : 8;  // 16-byte units of a row
      static_assert(UNITS % BATCH == 0, "whole batches");
      uint8_t* tile = smem + sub * Shape::Q_BYTES;
      auto place = [&](int r, int c) { return reinterpret_cast<uint4*>(tile + r * 128 + (c >> 3) * (128 * 128) + (((c & 7) ^ (r & 7)) << 4)); };
      const uint8_t* q0 = reinterpret_cast<const uint8_t*>(p.q) + (static_cast<size_t>(qstart) * p.q_stride + static_cast<size_t>(hk) * G * D) * 2;
#pragma unroll 1
      for (int b = 0; b < UNITS; b += BATCH) {
        uint4 v[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {  // rows behind the last are copies of it; a CTA without rows has none to read
          const int at = (b + i) * 32 + lane, r = row0 + min(sub * 128 + (warp & 3) * 32 + at / UNITS, valid_rows - 1);
          const int ahead = token_of(r);
          v[i] = make_uint4(0, 0, 0, 0);
          if (valid_rows > 0) v[i] = reinterpret_cast<const uint4*>(q0 + (ahead * p.q_stride + (r - ahead * G) * D) * 2)[at % UNITS];
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const int at = (b + i) * 32 + lane;
          if constexpr (!BF16) {
            v[i].x ^= p.q_flip;
            v[i].y ^= p.q_flip;
            v[i].z ^= p.q_flip;
            v[i].w ^= p.q_flip;
          }
          *place((warp & 3) * 32 + at / UNITS, at % UNITS) = v[i];
        }
      }
      __syncwarp();
      if constexpr (BF16) {
        // into fp16 with the row's largest magnitude in [2^10, 2^11); infinity and NaN stay what they are
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < UNITS; ++c) {
          const uint4 v = *place(row, c);
          top = __vmaxu2(__vmaxu2(top, __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu)), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
        }
        const int e = max(static_cast<int>(max(top & 0xffffu, top >> 16) >> 7) - 127 - 10, -120);
        const float q_scale = exp2f(static_cast<float>(-e));
        row_scale = exp2f(static_cast<float>(e));
#pragma unroll 4
        for (int c = 0; c < UNITS; ++c) {
          uint4 v = *place(row, c);
          uint32_t* x = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] ^= p.q_flip;
            x[i] = Kv4Type<__half>::pack(__uint_as_float(x[i] << 16) * q_scale, __uint_as_float(x[i] & 0xffff0000u) * q_scale);
          }
          *place(row, c) = v;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    const int mine = sub ? nblk[1] : nblk[0], all_to = info.all_to[sub], all_from = info.all_from[sub];
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_o = tmem + lanes + Shape::O_COL + sub * Shape::O_STEP;
    float m_ref = -INFINITY, l = 0.f;
    int v_exp = -1000;  // bf16: O holds sums of V * 2^-v_exp
    bool ok = true;
    for (int j = 0; j < mine && ok; ++j) {
      // bf16: the exponents of the block's K and V (the warps that expanded V wrote both before they released it)
      int k_exp = 0, v_top = v_exp;
      if constexpr (BF16) {
        const int n = 2 * j + 1;
        ok = mbar_wait(&tile_full[n % Shape::TILES], (n / Shape::TILES) & 1, abort_flag, p.status, ERR_WAIT_DEQUANT);
        k_exp = exps[j & 3][0];
        v_top = exps[j & 3][1];  // not below v_exp
      }
      ok = ok && (SUB == 2 ? mbar_wait(&s_full[sub], j & 1, abort_flag, p.status, ERR_WAIT_MMA)
                           : mbar_wait(&s_full[j & 1], (j >> 1) & 1, abort_flag, p.status, ERR_WAIT_MMA));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_s = tmem + lanes + (SUB == 2 ? sub * 128 : (j & 1) * BLK);
      if (warp_active) {
        const int base = base_of(j);
        const bool plain = base + BLK <= all_to && (!EXT || base >= all_from || base + BLK <= p.sink);
        const bool capped = EXT && p.cap_log2 != 0.f;
        // ---- maximum of the block's scores, 32 columns at a time (log2 units). Capped and masked ones are written back.
        const float undo = BF16 ? row_scale * exp2f(static_cast<float>(k_exp)) : row_scale;
        // (not 0 where zeros scaled it away: a hidden score is -inf * scale)
        const float scale = capped ? 1.f : fmaxf(p.scale_log2 * undo, 1e-30f);
        float mx = -INFINITY;
        uint32_t r[2][32];
        __syncwarp();
        tmem_ld32(t_s, r[0]);
#pragma unroll
        for (int c = 0; c < BLK / 32; ++c) {
          uint32_t (&x)[32] = r[c & 1];
          tmem_ld_wait();
          if (c + 1 < BLK / 32) tmem_ld32(t_s + (c + 1) * 32, r[(c + 1) & 1]);
          if (capped) {
            const float k = p.cap_k * undo;
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(kv4_softcap(__uint_as_float(x[i]), k, p.cap_log2));
          }
          if (!plain) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!kv4_visible(base + c * 32 + i, kvlen, start, EXT ? p.sink : 0, tm)) x[i] = 0xff800000u;
          }
          if (capped || !plain) kv4_tmem_st32(t_s + c * 32, x);
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            top[0] = fmaxf(top[0], fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
            top[1] = fmaxf(top[1], fmaxf(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])));
          }
          mx = fmaxf(mx, fmaxf(top[0], top[1]));
        }
        mx *= scale;
        if (capped || !plain) kv4_tmem_st_wait();
        tmem_ld32(t_s, r[0]);
        // ---- raise the reference (and the exponent of V) where the block needs it
        if (__any_sync(0xffffffffu, mx > m_ref + 8.f || v_top > v_exp)) {
          const float m_new = fmaxf(m_ref, mx);
          const float alpha = m_ref == -INFINITY ? 0.f : exp2f(m_ref - m_new);
          // (the first block finds O undefined and leaves it alone; rows that saw nothing so far hold zeros)
          const float o_alpha = BF16 ? alpha * exp2f(static_cast<float>(max(v_exp - v_top, -126))) : alpha;
          v_exp = v_top;
          if (j > 0) {
            if (SUB == 1) {  // the scores of this block were computed before the last P V ended
              ok = mbar_wait(pv_done, (j - 1) & 1, abort_flag, p.status, ERR_WAIT_MMA);
              ok = __all_sync(0xffffffffu, ok);
              tc_fence_after();
            }
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld32(t_o + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * o_alpha);
              kv4_tmem_st32(t_o + c, o);
            }
          }
          l *= m_ref == -INFINITY ? 1.f : alpha;
          m_ref = m_new;
        }
        // ---- weights against the reference; they overwrite columns that were read before
        const float shift = m_ref == -INFINITY ? 0.f : -m_ref;
#pragma unroll
        for (int c = 0; c < BLK / 32; ++c) {
          uint32_t (&x)[32] = r[c & 1];
          tmem_ld_wait();
          if (c + 1 < BLK / 32) tmem_ld32(t_s + (c + 1) * 32, r[(c + 1) & 1]);
          float2 acc = make_float2(0.f, 0.f);
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 v = make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
            const float2 y = kv4_fma2(v, make_float2(scale, scale), make_float2(shift, shift));
            const float2 e = make_float2(exp2f(y.x), exp2f(y.y));
            acc = kv4_add2(acc, e);
            w[i] = Kv4Type<__half>::pack(e.x, e.y);
          }
          l += acc.x + acc.y;
          kv4_tmem_st16(t_s + c * 16, w);
        }
        kv4_tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[SUB == 2 ? sub : j & 1]);
    }
    // ---- epilogue: O / l, or the partial row
    if (ok && mine > 0) {
      ok = mbar_wait(&o_done[sub], 0, abort_flag, p.status, ERR_WAIT_MMA);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok && guard) ok = __all_sync(0xffffffffu, mbar_wait(looked, 0, abort_flag, p.status, ERR_WAIT_PRODUCER));
    const bool exact = BF16 && ok && wide_from < mine;
    if (ok && warp_active && exact) {
      if constexpr (BF16) {
        const int wrow0 = sub * 128 + (warp & 3) * 32;
        const int end = min(wrow0 + 32, valid_rows);
        auto at = [&](int i) {
          const int pos = base_of(i / BLK) + i % BLK;
          return pos < room ? pos : -1;
        };
#pragma unroll 1
        for (int first = wrow0; first < end; first += KV4_EXACT) {
          int len[KV4_EXACT], from[KV4_EXACT];
          size_t to[KV4_EXACT];  // the row of (token, head)
          unsigned long long bits[KV4_EXACT];
          const T* q[KV4_EXACT];
#pragma unroll
          for (int i = 0; i < KV4_EXACT; ++i) {
            const int r = row0 + min(first + i, end - 1), ahead = token_of(r), t = qstart + ahead, h = hk * G + r - ahead * G;
            to[i] = static_cast<size_t>(t) * p.hq + h;
            q[i] = reinterpret_cast<const T*>(p.q) + static_cast<size_t>(t) * p.q_stride + h * D;
            len[i] = p.q_kvlen[t];
            from[i] = EXT && p.q_kvstart ? p.q_kvstart[t] : 0;
            bits[i] = EXT && p.tree_mask ? p.tree_mask[t] : 0ull;
          }
          auto sees = [&](int i, int pos) { return kv4_visible(pos, len[i], from[i], EXT ? p.sink : 0, bits[i]); };
          float M[KV4_EXACT], L[KV4_EXACT], acc[KV4_EXACT][8];
          kv4_rows_exact<T, D>(p.pages, p.num_pages, list, p.hkv, hk, q, p.q_flip ? -1.f : 1.f, p.scale_log2, EXT ? p.cap_k : 0.f,
                               EXT ? p.cap_log2 : 0.f, mine * BLK, at, sees, M, L, acc);
#pragma unroll
          for (int i = 0; i < KV4_EXACT; ++i) {
            if (first + i >= end) continue;
            if (p.splits > 1) {
              const size_t prow = ((static_cast<size_t>(work) * p.hkv + hk) * p.splits + split) * (SUB * 128) + first + i;
              if (lane < D / 8) kv4_put8(p.part_o + prow * D + lane * 8, acc[i]);
              if (lane == 0) {
                p.part_ml[prow * 2] = M[i];
                p.part_ml[prow * 2 + 1] = L[i];
              }
            } else {
              if (lane < D / 8) kv4_put8(reinterpret_cast<T*>(p.out) + to[i] * D + lane * 8, acc[i], L[i] == 0.f ? 0.f : 1.f / L[i]);
              if (lane == 0 && p.lse) p.lse[to[i]] = L[i] == 0.f ? -INFINITY : (M[i] + log2f(L[i])) * 0.6931471805599453f;
            }
          }
        }
      }
    }
    if (ok && warp_active && !exact) {
      tc_fence_after();
      const float grow_v = BF16 && mine > 0 ? exp2f(static_cast<float>(v_exp)) : 1.f;
      const float inv = l == 0.f ? 0.f : 1.f / l * grow_v;  // a row that sees nothing is 0; NaN stays NaN
      const size_t prow = ((static_cast<size_t>(work) * p.hkv + hk) * p.splits + split) * (SUB * 128) + grow;
      // By way of shared memory (this tile's queries are used up), so that neighbouring lanes write neighbouring bytes:
      // 32 columns of the warp's rows, 8 units of 16 bytes each as fp32, 4 in the output's type.
      const bool partial = p.splits > 1;
      uint8_t* stage = smem + sub * Shape::Q_BYTES + (warp & 3) * 4096;
      const int wrow0 = sub * 128 + (warp & 3) * 32;
      uint8_t* part = reinterpret_cast<uint8_t*>(p.part_o) + (prow - lane) * D * 4;
      uint8_t* dst[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = row0 + wrow0 + i * 8 + (lane >> 2);
        const int ahead = token_of(r);
        dst[i] = reinterpret_cast<uint8_t*>(p.out) + (static_cast<size_t>(qstart + ahead) * p.hq + hk * G + r - ahead * G) * D * 2 + (lane & 3) * 16;
        if (r - row0 >= valid_rows) dst[i] = nullptr;
      }
      uint32_t o2[2][32];
      __syncwarp();
      tmem_ld32(t_o, o2[0]);
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t (&o)[32] = o2[(c / 32) & 1];
        tmem_ld_wait();
        if (c + 32 < D) tmem_ld32(t_o + c + 32, o2[(c / 32 + 1) & 1]);
        __syncwarp();
        if (mine == 0) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0;
        }
        if (partial) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) =
                make_float4(__uint_as_float(o[4 * i]) * grow_v, __uint_as_float(o[4 * i + 1]) * grow_v,
                            __uint_as_float(o[4 * i + 2]) * grow_v, __uint_as_float(o[4 * i + 3]) * grow_v);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            if (wrow0 + r < valid_rows)
              *reinterpret_cast<uint4*>(part + static_cast<size_t>(r) * D * 4 + c * 4 + (lane & 7) * 16) =
                  *reinterpret_cast<const uint4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              v[k] = Kv4Type<T>::pack(__uint_as_float(o[i * 8 + 2 * k]) * inv, __uint_as_float(o[i * 8 + 2 * k + 1]) * inv);
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + (lane >> 2);
            if (dst[i])
              *reinterpret_cast<uint4*>(dst[i] + c * 2) =
                  *reinterpret_cast<const uint4*>(stage + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
          }
        }
      }
      if (row_valid) {
        if (p.splits > 1) {
          p.part_ml[prow * 2] = m_ref;
          p.part_ml[prow * 2 + 1] = l;
        } else if (p.lse) {
          p.lse[static_cast<size_t>(tok) * p.hq + head] = l == 0.f ? -INFINITY : (m_ref + log2f(l)) * 0.6931471805599453f;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == ISSUER) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the splits: one warp per row, grid (tiles, hkv).
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_prefill_merge_kernel(const Kv4PreParams p) {
  constexpr int ROWS = Kv4PreShape<D>::SUB * 128;
  const int tile = blockIdx.x / p.parts, row0 = blockIdx.x % p.parts * 128;
  const int hk = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int qstart = p.tile_qstart[tile], rows = min(ROWS, p.tile_ntok[tile] * p.group - row0);
  for (int row = blockIdx.z * 8 + warp; row < rows; row += 8 * gridDim.z) {
    const size_t first = (static_cast<size_t>(blockIdx.x) * p.hkv + hk) * p.splits * ROWS + row;
    float M = -INFINITY, L = 0.f, acc[D / 32];
    for (int s = 0; s < p.splits; ++s) M = fmaxf(M, p.part_ml[(first + s * ROWS) * 2]);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) acc[c] = 0.f;
    for (int s = 0; s < p.splits; ++s) {
      const size_t b = first + s * ROWS;
      const float ms = p.part_ml[b * 2], ls = p.part_ml[b * 2 + 1];
      const float w = ms == -INFINITY ? 0.f : exp2f(ms - M);
      L += ls != ls ? ls : ls * w;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) acc[c] = fmaf(p.part_o[b * D + c * 32 + lane], w, acc[c]);
    }
    const size_t at = static_cast<size_t>(qstart + (row0 + row) / p.group) * p.hq + hk * p.group + (row0 + row) % p.group;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* dst = reinterpret_cast<T*>(p.out) + at * D;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dst[c * 32 + lane] = Cvt<T>::from_f(acc[c] * inv);
    if (p.lse && lane == 0) p.lse[at] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
  }
}

template <typename T, int D, bool EXT>
int kv4_prefill_launch(const Kv4PreParams& p, cudaStream_t stream) {
  using Shape = Kv4PreShape<D>;
  auto kern = kv4_prefill_kernel<T, D, EXT>;
  static bool attr_set[64] = {};
  if (first_use_on_device(attr_set)) {
    const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM);
    if (err != cudaSuccess) return static_cast<int>(err);
  }
  kern<<<p.num_tiles * p.parts * p.splits * p.hkv, Shape::THREADS, Shape::SMEM, stream>>>(p);
  count_launch();
  if (p.splits > 1) {
    kv4_prefill_merge_kernel<T, D><<<dim3(p.num_tiles * p.parts, p.hkv, 8), 256, 0, stream>>>(p);
    count_launch();
  }
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
int kv4_prefill_shape(const Kv4PreParams& p, int d, bool ext, cudaStream_t stream) {
  if (d == 64) return ext ? kv4_prefill_launch<T, 64, true>(p, stream) : kv4_prefill_launch<T, 64, false>(p, stream);
  if (d == 96) return ext ? kv4_prefill_launch<T, 96, true>(p, stream) : kv4_prefill_launch<T, 96, false>(p, stream);
  if (d == 128) return ext ? kv4_prefill_launch<T, 128, true>(p, stream) : kv4_prefill_launch<T, 128, false>(p, stream);
  return ext ? kv4_prefill_launch<T, 256, true>(p, stream) : kv4_prefill_launch<T, 256, false>(p, stream);
}

}  // namespace mlcb

using namespace mlcb;

// One layer's cache [num_pages, 2, hkv, 16, row]. Tiles are (sequence, query-token range) pairs with tokens * hq / hkv
// <= tile_rows <= 256. splits > 1 needs fp32 scratch for 256 rows per (tile, kv head, split): part_o [.., 256, d] and
// part_ml [.., 256, 2]. Returns -1 shape, -2 alignment, -3 type, -4 missing scratch.
MLCB_API int mlcb_kv4_prefill(const void* q, const void* pages, void* out, float* lse, const int* tile_seq,
                              const int* tile_qstart, const int* tile_ntok, const int* q_kvlen, const int* page_indptr,
                              const int* page_indices, int num_tiles, int tile_rows, long long q_stride, int hq, int hkv,
                              int d, long long num_pages, float sm_scale, int dtype, int splits, float* part_o,
                              float* part_ml, int* status, cudaStream_t stream, const int* q_kvstart,
                              const unsigned long long* tree_mask, int sink, float softcap) {
  if (num_tiles <= 0) return 0;
  if (hkv <= 0 || hkv > 65535 || hq <= 0 || hq % hkv || (d != 64 && d != 96 && d != 128 && d != 256)) return -1;
  if (tile_rows < 1 || tile_rows > 256) return -1;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(pages)) & 15) return -2;
  if (q_stride % 8) return -2;
  if (dtype != 0 && dtype != 1) return -3;
  if (splits < 1 || (splits > 1 && (!part_o || !part_ml)) || static_cast<long long>(num_tiles) * splits * 2 * hkv > 0x7fffffffLL) return -4;
  Kv4PreParams p;
  p.q = q;
  p.pages = static_cast<const uint8_t*>(pages);
  p.out = out;
  p.lse = lse;
  p.part_o = part_o;
  p.part_ml = part_ml;
  p.tile_seq = tile_seq;
  p.tile_qstart = tile_qstart;
  p.tile_ntok = tile_ntok;
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
  p.sink = q_kvstart ? sink : 0;
  p.splits = splits;
  p.num_tiles = num_tiles;
  p.parts = d == 256 && tile_rows > 128 ? 2 : 1;
  p.q_flip = sm_scale < 0.f ? 0x80008000u : 0u;
  p.scale_log2 = fmaxf(fabsf(sm_scale) * 1.4426950408889634f, 1e-30f);  // a hidden score is -inf * scale: not 0
  p.cap_k = softcap > 0.f ? 2.f * 1.4426950408889634f * fabsf(sm_scale) / softcap : 0.f;
  p.cap_log2 = softcap > 0.f ? softcap * 1.4426950408889634f : 0.f;
  const bool ext = q_kvstart || tree_mask || softcap > 0.f;
  return dtype == 0 ? kv4_prefill_shape<__half>(p, d, ext, stream) : kv4_prefill_shape<__nv_bfloat16>(p, d, ext, stream);
}
