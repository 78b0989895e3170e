// Decode attention over the 4-bit paged KV cache (format: kv4.cuh): head sizes 64, 128 and 256, 16-token pages,
// at most 16 query rows per (sequence, kv head) -- the G = hq / hkv heads of the group times the appended tokens.
//
// Floor: the cached bytes, 160 per token and kv head at D = 128 (K and V), once. At 44 bytes per ns and SM that
// leaves 112 clocks, 448 issue slots, per 16 tokens and SM, of which expanding the nibbles takes about 200; the
// kernel therefore wastes nothing on the query side:
//
//   S^T = K Q^T   m16n8k16 with the 16 tokens of a page as M and 8 query rows as N: half the instructions of the
//                 usual orientation, whose M = 16 rows are mostly padding. A lane's A fragments are two tokens
//                 and one quarter of the channels -- at D = 128 exactly one quantisation group, so a row is one
//                 16-byte load of codes and one (lo, s) word. The order of channels along K is free (Q is loaded
//                 in the same order), which makes the lane's channels contiguous.
//   softmax       in the S^T accumulators: a lane has two query rows and 4 tokens of 16. The reference maximum is
//                 raised only when some score exceeds it by more than 8 (log2), so the usual step has no shuffle
//                 and no rescaling; P stays below 2^8 and the final division by the row sum makes it exact.
//   O^T += V^T P^T  M = 16 channels, N = 8 query rows; P^T fragments come from the S^T accumulators by one
//                 8 x 8 transpose (movmatrix) per 8 tokens. A fragments want pairs of tokens: two tokens' code
//                 words are interleaved by halves (prmt) and expanded with the same masks.
//
// K and V are rounded to the type of the rows after lo + s c (one rounding), P to the same type; sums, maxima and
// accumulators are fp32.
//
// Work: a unit is one (sequence, kv head, row block of 8 or 16, KV split). CTAs are persistent; a producer warp
// streams the units' pages back to back through a ring of 32-token slots (two pages, up to four bulk copies) so
// that loads never stop between units, four consumer warps take the slots round-robin and merge at the end of
// each unit. Every wait is bounded (common.cuh).
#include "kv4.cuh"

namespace mlcb {

constexpr int KV4_PAGE = 16;
constexpr int KV4_DEC_THREADS = 160;

struct Kv4DecParams {
  const void* q;
  const uint8_t* pages;
  void* out;
  float* lse;
  float* part_o;   // [items, hkv, splits, 16, D] fp32 (splits > 1)
  float* part_ml;  // [items, hkv, splits, 16, 2]
  const int *item_seq, *item_qstart, *item_ntok, *q_kvlen, *page_indptr, *page_indices;
  const int* q_kvstart;
  const unsigned long long* tree_mask;
  int* status;
  long long q_stride, num_pages;
  int hq, hkv, group, splits, row_blocks, num_units, sink;
  float scale_log2;          // sm_scale * log2(e)
  float cap_k, cap_log2;     // soft cap: scores are kv4_softcap(raw, cap_k, cap_log2); 0 = none
};

// Visibility of position `pos` to a query token (the rule of the 16-bit kernels): below kvlen all positions from
// `start` on and the first `sink`; from kvlen on the set bits of the tree mask.
__device__ __forceinline__ bool kv4_visible(int pos, int kvlen, int start, int sink, unsigned long long tm) {
  if (pos < kvlen) return pos >= start || pos < sink;
  const int r = pos - kvlen;
  return r < 64 && ((tm >> r) & 1ull);
}

struct Kv4Unit {
  int item, hk, split, rb, qstart, ntok, valid_rows;
  int pg_begin, npg;        // pages of this unit, counted over the pages the item visits
  int sink_pg, skip;        // pages [sink_pg, sink_pg + skip) lie outside every row's window: never fetched
  int all_from, all_to;     // positions that every row sees: [all_from, all_to), and [0, all_sink) below the window
  const int* list;
  __device__ __forceinline__ int page_index(int i) const {
    const int li = pg_begin + i;
    return li < sink_pg ? li : li + skip;
  }
};

template <bool EXT>
__device__ __forceinline__ Kv4Unit kv4_unit(const Kv4DecParams& p, int u) {
  Kv4Unit d;
  d.split = u % p.splits;
  int r = u / p.splits;
  d.rb = r % p.row_blocks;
  r /= p.row_blocks;
  d.hk = r % p.hkv;
  d.item = r / p.hkv;
  const int b = p.item_seq[d.item];
  d.qstart = p.item_qstart[d.item];
  d.ntok = p.item_ntok[d.item];
  d.valid_rows = d.ntok * p.group;
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
    d.skip = max(0, first / KV4_PAGE - d.sink_pg);
  }
  const int p0 = p.page_indptr[b];
  const int held = p.page_indptr[b + 1] - p0;
  d.list = p.page_indices + p0;
  int upto = (reach + KV4_PAGE - 1) / KV4_PAGE;
  if (upto > held) {  // more positions than the sequence has pages for: never dereferenced
    if (p.status) atomicCAS(p.status, 0, ERR_BAD_INDEX);
    upto = held;
  }
  const int total = max(0, upto - d.skip);
  const int per = ((total + p.splits - 1) / p.splits + 1) & ~1;  // whole slots
  d.pg_begin = d.split * per;
  d.npg = max(0, min(total, d.pg_begin + per) - d.pg_begin);
  return d;
}

__device__ __forceinline__ uint32_t kv4_movmatrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename T>
__device__ __forceinline__ void kv4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1);
template <>
__device__ __forceinline__ void kv4_mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void kv4_mma<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                       uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// N code words from shared memory (rows are 16-, 8- or 4-byte aligned for N = 4, 2, 1).
template <int N>
__device__ __forceinline__ void kv4_words(const uint8_t* p, uint32_t (&w)[N]) {
  if (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x;
      w[4 * i + 1] = v.y;
      w[4 * i + 2] = v.z;
      w[4 * i + 3] = v.w;
    }
  } else if (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

template <int D, int NT>
struct Kv4DecShape {
  static constexpr int ROW = kv4_row_bytes(D);
  static constexpr int PAGE_BYTES = KV4_PAGE * ROW;            // K or V of one page and head
  static constexpr int SLOT_BYTES = 4 * PAGE_BYTES;            // K, V of two pages
  static constexpr int SLOTS = D == 256 ? 4 : 8;               // a multiple of the four consumer warps
  static constexpr int ROWS = 8 * NT;
  static constexpr int MERGE_BYTES = 4 * ROWS * (D + 2) * 4;   // four warps' O rows and (m, l) pairs
  static constexpr int SMEM = SLOTS * SLOT_BYTES + MERGE_BYTES + 16 * SLOTS + 16;
};

template <typename T, int D, int NT, bool EXT>
__global__ void __launch_bounds__(KV4_DEC_THREADS, 2) kv4_decode_kernel(const Kv4DecParams p) {
  using Shape = Kv4DecShape<D, NT>;
  constexpr int ROW = Shape::ROW, PB = Shape::PAGE_BYTES, SLOTS = Shape::SLOTS, ROWS = Shape::ROWS;
  constexpr int KW = D / 32;   // K code words per lane and token
  constexpr int VW = D / 64;   // V code words per lane and token
  pdl_launch_dependents();
  extern __shared__ __align__(128) uint8_t smem[];
  float* sm_o = reinterpret_cast<float*>(smem + SLOTS * Shape::SLOT_BYTES);  // [4][ROWS][D]
  float* sm_ml = sm_o + 4 * ROWS * D;                                       // [4][ROWS][2]
  uint64_t* full = reinterpret_cast<uint64_t*>(sm_ml + 4 * ROWS * 2);
  uint64_t* empty = full + SLOTS;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + SLOTS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < SLOTS) {
    mbar_init(&full[threadIdx.x], 1);
    mbar_init(&empty[threadIdx.x], 1);
    mbar_fence_init();
  }
  if (threadIdx.x == 0) *abort_flag = 0;
  __syncthreads();

  if (warp == 4) {
    // ---------------------------------------------------------------- producer
    // Lane i holds the page number of the unit's page base + i (one coalesced load per 32 pages); lanes 0..3 each
    // issue one copy of a slot (K and V of its two pages).
    uint32_t g = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < p.num_units && ok; u += gridDim.x) {
      const Kv4Unit d = kv4_unit<EXT>(p, u);
      for (int base = 0; base < d.npg && ok; base += 32) {
        int mine = 0;
        if (base + lane < d.npg) {
          mine = d.list[d.page_index(base + lane)];
          if (mine >= p.num_pages) {
            if (p.status) atomicCAS(p.status, 0, ERR_BAD_INDEX);
            mine = 0;
          }
          if (mine < 0) mine = 0;  // released by a sliding window: every position of it is masked
        }
        const int n = min(32, d.npg - base);
        for (int i = 0; i < n; i += 2, ++g) {
          const int s = g % SLOTS;
          if (g >= SLOTS) {
            ok = mbar_wait(&empty[s], ((g / SLOTS) & 1) ^ 1, abort_flag, p.status, ERR_WAIT_PRODUCER);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
          const int here = min(2, n - i);
          if (lane == 0) mbar_expect_tx(&full[s], here * 2 * PB);
          __syncwarp();
          const int pg = __shfl_sync(0xffffffffu, mine, i + ((lane >> 1) & 1));
          if (lane < 2 * here) {
            const size_t block = (static_cast<size_t>(pg) * 2 + (lane & 1)) * p.hkv + d.hk;
            bulk_load(smem + s * Shape::SLOT_BYTES + lane * PB, p.pages + block * PB, PB, &full[s]);
          }
        }
      }
    }
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int r = lane >> 2, t = lane & 3;
  uint32_t g0 = 0;
  for (int u = blockIdx.x; u < p.num_units; u += gridDim.x) {
    const Kv4Unit d = kv4_unit<EXT>(p, u);
    const int row0 = d.rb * ROWS;                           // first query row of this unit
    const int rows = min(ROWS, d.valid_rows - row0);        // may be <= 0: an empty row block
    // Q^T fragments: lane (r, t) holds row r (+ 8 per n-tile), channels [t D / 4, (t + 1) D / 4)
    uint32_t qb[NT][D / 16][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = nt * 8 + r;
      const bool live = row < rows;
      const int tok = d.qstart + (live ? (row0 + row) / p.group : 0), head = d.hk * p.group + (live ? (row0 + row) % p.group : 0);
      const uint8_t* src = reinterpret_cast<const uint8_t*>(p.q) +
                           (static_cast<size_t>(tok) * p.q_stride + static_cast<size_t>(head) * D + t * (D / 4)) * 2;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint4 v = live ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0);
        qb[nt][2 * i][0] = v.x;
        qb[nt][2 * i][1] = v.y;
        qb[nt][2 * i + 1][0] = v.z;
        qb[nt][2 * i + 1][1] = v.w;
      }
    }
    // this lane's score columns: rows 2 t and 2 t + 1 of each n-tile
    int kvlen[NT][2], start[NT][2];
    unsigned long long tm[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = nt * 8 + 2 * t + c;
        const bool live = row < rows;
        const int tok = d.qstart + (live ? (row0 + row) / p.group : 0);
        kvlen[nt][c] = live ? p.q_kvlen[tok] : 0;
        start[nt][c] = EXT && live && p.q_kvstart ? p.q_kvstart[tok] : 0;
        tm[nt][c] = EXT && live && p.tree_mask ? p.tree_mask[tok] : 0ull;
      }
    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
    }
    const int nslots = (d.npg + 1) >> 1;
    bool ok = true;
    for (int i = (warp - static_cast<int>(g0 & 3u)) & 3; i < nslots && ok; i += 4) {
      const uint32_t g = g0 + static_cast<uint32_t>(i);
      const int s = g % SLOTS;
      ok = mbar_wait(&full[s], (g / SLOTS) & 1, abort_flag, p.status, ERR_WAIT_TMA);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint8_t* slot = smem + s * Shape::SLOT_BYTES;
      const bool two = 2 * i + 1 < d.npg;
      const int at[2] = {d.page_index(2 * i) * KV4_PAGE, two ? d.page_index(2 * i + 1) * KV4_PAGE : 0x3fffffff};
      // ---- S^T = K Q^T
      float sc[2][NT][4];
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
        const uint8_t* k0 = slot + pg * 2 * PB + r * ROW;
        const uint8_t* k1 = k0 + 8 * ROW;
        uint32_t w0[KW], w1[KW];
        kv4_words<KW>(k0 + t * (D / 8), w0);
        kv4_words<KW>(k1 + t * (D / 8), w1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[pg][nt][0] = sc[pg][nt][1] = sc[pg][nt][2] = sc[pg][nt][3] = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const int grp = (t * (D / 4) + w * 8) / KV4_GROUP;
          const uint32_t m0 = *reinterpret_cast<const uint32_t*>(k0 + D / 2 + grp * 4);
          const uint32_t m1 = *reinterpret_cast<const uint32_t*>(k1 + D / 2 + grp * 4);
          uint32_t e0[4], e1[4];
          Kv4Type<T>::expand4(w0[w], __byte_perm(m0, m0, 0x3232), __byte_perm(m0, m0, 0x1010), e0);
          Kv4Type<T>::expand4(w1[w], __byte_perm(m1, m1, 0x3232), __byte_perm(m1, m1, 0x1010), e1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            kv4_mma<T>(sc[pg][nt], e0[0], e1[0], e0[1], e1[1], qb[nt][2 * w][0], qb[nt][2 * w][1]);
            kv4_mma<T>(sc[pg][nt], e0[2], e1[2], e0[3], e1[3], qb[nt][2 * w + 1][0], qb[nt][2 * w + 1][1]);
          }
        }
      }
      // ---- scale, cap, mask. A slot that every row sees in full (all but the ends of a sequence or window) skips
      // the per-element test; the others also drop V of tokens that no row sees, whatever their bytes hold.
      bool plain = two;
#pragma unroll
      for (int pg = 0; pg < 2; ++pg)
        plain = plain && at[pg] + KV4_PAGE <= d.all_to && (!EXT || at[pg] >= d.all_from || at[pg] + KV4_PAGE <= p.sink);
      uint32_t seen = 0xffffffffu;
#pragma unroll
      for (int pg = 0; pg < 2; ++pg)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float v = sc[pg][nt][c];
            v = EXT && p.cap_log2 != 0.f ? kv4_softcap(v, p.cap_k, p.cap_log2) : v * p.scale_log2;
            sc[pg][nt][c] = v;
          }
      if (!plain) {
#pragma unroll
        for (int pg = 0; pg < 2; ++pg)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (!kv4_visible(at[pg] + r + (c >> 1) * 8, kvlen[nt][c & 1], start[nt][c & 1], p.sink, tm[nt][c & 1]))
                sc[pg][nt][c] = -INFINITY;
        const int pos = (lane < 16 ? at[0] : at[1]) + (lane & 15);  // lane = token of the slot
        bool any = false;
        for (int q = 0; q < d.ntok; ++q)
          any = any || kv4_visible(pos, p.q_kvlen[d.qstart + q], EXT && p.q_kvstart ? p.q_kvstart[d.qstart + q] : 0, p.sink,
                                   EXT && p.tree_mask ? p.tree_mask[d.qstart + q] : 0ull);
        seen = __ballot_sync(0xffffffffu, any);
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
        const float ms0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], ms1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
          const float e0 = exp2f(sc[pg][nt][0] - ms0), e1 = exp2f(sc[pg][nt][1] - ms1);
          const float e2 = exp2f(sc[pg][nt][2] - ms0), e3 = exp2f(sc[pg][nt][3] - ms1);
          l[nt][0] += e0 + e2;
          l[nt][1] += e1 + e3;
          pb[pg][nt][0] = kv4_movmatrix(Kv4Type<T>::pack(e0, e1));
          pb[pg][nt][1] = kv4_movmatrix(Kv4Type<T>::pack(e2, e3));
        }
      }
      // ---- O^T += V^T P^T: this lane expands channels [r D / 8, (r + 1) D / 8) of tokens 2t, 2t+1, 2t+8, 2t+9
#pragma unroll
      for (int pg = 0; pg < 2; ++pg) {
        const uint8_t* vb = slot + (pg * 2 + 1) * PB;
        uint32_t w[4][VW], meta[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int token = 2 * t + (k & 1) + (k >> 1) * 8;
          kv4_words<VW>(vb + token * ROW + r * (D / 16), w[k]);
          meta[k] = *reinterpret_cast<const uint32_t*>(vb + token * ROW + D / 2 + (r * (D / 8) / KV4_GROUP) * 4);
          if (!((seen >> (pg * 16 + token)) & 1u)) meta[k] = 0u;
        }
        const uint32_t lo_ab = __byte_perm(meta[0], meta[1], 0x5410), s_ab = __byte_perm(meta[0], meta[1], 0x7632);
        const uint32_t lo_cd = __byte_perm(meta[2], meta[3], 0x5410), s_cd = __byte_perm(meta[2], meta[3], 0x7632);
#pragma unroll
        for (int i2 = 0; i2 < VW; ++i2) {
          uint32_t a0[4], a1[4], a2[4], a3[4];
          Kv4Type<T>::expand4(__byte_perm(w[0][i2], w[1][i2], 0x5410), s_ab, lo_ab, a0);
          Kv4Type<T>::expand4(__byte_perm(w[0][i2], w[1][i2], 0x7632), s_ab, lo_ab, a1);
          Kv4Type<T>::expand4(__byte_perm(w[2][i2], w[3][i2], 0x5410), s_cd, lo_cd, a2);
          Kv4Type<T>::expand4(__byte_perm(w[2][i2], w[3][i2], 0x7632), s_cd, lo_cd, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              kv4_mma<T>(o[nt][i2 * 4 + k], a0[k], a1[k], a2[k], a3[k], pb[pg][nt][0], pb[pg][nt][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
    g0 += static_cast<uint32_t>(nslots);
    // ---------------------------------------------------------------- merge the four warps of the unit
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = l[nt][c];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int row = nt * 8 + 2 * t + c;
        if (r == 0) {
          sm_ml[(warp * ROWS + row) * 2] = m[nt][c];
          sm_ml[(warp * ROWS + row) * 2 + 1] = x;
        }
        if (row < rows) {
          float* dst = sm_o + (warp * ROWS + row) * D + r * (D / 8);
#pragma unroll
          for (int j = 0; j < D / 16; ++j) *reinterpret_cast<float2*>(dst + 2 * j) = make_float2(o[nt][j][c], o[nt][j][c + 2]);
        }
      }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    for (int row = warp; row < rows; row += 4) {
      float M = -INFINITY, L = 0.f, wgt[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_ml[(w * ROWS + row) * 2]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float mw = sm_ml[(w * ROWS + row) * 2];
        wgt[w] = mw == -INFINITY ? 0.f : exp2f(mw - M);
        const float lw = sm_ml[(w * ROWS + row) * 2 + 1];
        L += lw != lw ? lw : lw * wgt[w];
      }
      float acc[D / 32];
#pragma unroll
      for (int c = 0; c < D / 32; ++c) acc[c] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int c = 0; c < D / 32; ++c) acc[c] = fmaf(sm_o[(w * ROWS + row) * D + c * 32 + lane], wgt[w], acc[c]);
      const int tok = d.qstart + (row0 + row) / p.group, head = d.hk * p.group + (row0 + row) % p.group;
      if (p.splits > 1) {
        const size_t base = ((static_cast<size_t>(d.item) * p.hkv + d.hk) * p.splits + d.split) * 16 + row0 + row;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) p.part_o[base * D + c * 32 + lane] = acc[c];
        if (lane == 0) {
          p.part_ml[base * 2] = M;
          p.part_ml[base * 2 + 1] = L;
        }
      } else {
        const float inv = L == 0.f ? 0.f : 1.f / L;  // a row that sees nothing is 0; NaN stays NaN
        T* dst = reinterpret_cast<T*>(p.out) + (static_cast<size_t>(tok) * p.hq + head) * D;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) dst[c * 32 + lane] = Cvt<T>::from_f(acc[c] * inv);
        if (p.lse && lane == 0)
          p.lse[static_cast<size_t>(tok) * p.hq + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
      }
    }
    // the scratch area is rewritten by the next unit; after the barrier all four warps read the same abort flag,
    // so they leave together if a wait of any of them ran out
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (*abort_flag) break;
  }
}

// Joins the splits of every (item, kv head): one warp per row.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_decode_merge_kernel(const Kv4DecParams p) {
  const int item = blockIdx.x, hk = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int qstart = p.item_qstart[item], valid_rows = p.item_ntok[item] * p.group;
  for (int row = warp; row < valid_rows; row += 4) {
    const size_t first = (static_cast<size_t>(item) * p.hkv + hk) * p.splits * 16 + row;
    float M = -INFINITY;
    for (int s = 0; s < p.splits; ++s) M = fmaxf(M, p.part_ml[(first + s * 16) * 2]);
    float L = 0.f, acc[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) acc[c] = 0.f;
    for (int s = 0; s < p.splits; ++s) {
      const float ms = p.part_ml[(first + s * 16) * 2], ls = p.part_ml[(first + s * 16) * 2 + 1];
      const float w = ms == -INFINITY ? 0.f : exp2f(ms - M);
      L += ls != ls ? ls : ls * w;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) acc[c] = fmaf(p.part_o[(first + s * 16) * D + c * 32 + lane], w, acc[c]);
    }
    const int tok = qstart + row / p.group, head = hk * p.group + row % p.group;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* dst = reinterpret_cast<T*>(p.out) + (static_cast<size_t>(tok) * p.hq + head) * D;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dst[c * 32 + lane] = Cvt<T>::from_f(acc[c] * inv);
    if (p.lse && lane == 0)
      p.lse[static_cast<size_t>(tok) * p.hq + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
  }
}

template <typename T, int D, int NT, bool EXT>
int kv4_decode_launch(const Kv4DecParams& p, int num_items, cudaStream_t stream) {
  using Shape = Kv4DecShape<D, NT>;
  auto kern = kv4_decode_kernel<T, D, NT, EXT>;
  static int per_sm[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return static_cast<int>(err);
  dev &= 63;
  if (!per_sm[dev]) {
    err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM);
    if (err != cudaSuccess) return static_cast<int>(err);
    int n = 0;
    err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, KV4_DEC_THREADS, Shape::SMEM);
    if (err != cudaSuccess) return static_cast<int>(err);
    per_sm[dev] = n > 0 ? n : 1;
  }
  const int most = per_sm[dev] * sm_count();
  kern<<<p.num_units < most ? p.num_units : most, KV4_DEC_THREADS, Shape::SMEM, stream>>>(p);
  count_launch();
  if (p.splits > 1) {
    kv4_decode_merge_kernel<T, D><<<dim3(num_items, p.hkv), 128, 0, stream>>>(p);
    count_launch();
  }
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int D>
int kv4_decode_shape(Kv4DecParams& p, int rows, bool ext, int num_items, cudaStream_t stream) {
  // Up to 8 query rows need one n-tile. 9 to 16 rows take two, which share the expanded K and V; at D = 256 the
  // accumulators of two would not fit the register file, and two units read the same pages instead.
  if (D < 256 && rows > 8) {
    p.row_blocks = 1;
    p.num_units = num_items * p.hkv * p.splits;
    return ext ? kv4_decode_launch<T, D, (D < 256 ? 2 : 1), true>(p, num_items, stream)
               : kv4_decode_launch<T, D, (D < 256 ? 2 : 1), false>(p, num_items, stream);
  }
  p.row_blocks = (rows + 7) / 8;
  p.num_units = num_items * p.hkv * p.splits * p.row_blocks;
  return ext ? kv4_decode_launch<T, D, 1, true>(p, num_items, stream) : kv4_decode_launch<T, D, 1, false>(p, num_items, stream);
}

}  // namespace mlcb

using namespace mlcb;

// One layer's cache [num_pages, 2, hkv, 16, row]. Items are (sequence, query-token range) pairs of at most `rows`
// <= 16 query rows (tokens * hq / hkv) each. splits > 1 needs fp32 scratch part_o [items, hkv, splits, 16, d] and
// part_ml [.., 16, 2]. Returns -1 shape, -2 alignment, -3 type, -4 missing scratch, -5 too many units.
MLCB_API int mlcb_kv4_decode(const void* q, const void* pages, void* out, float* lse, const int* item_seq,
                             const int* item_qstart, const int* item_ntok, const int* q_kvlen, const int* page_indptr,
                             const int* page_indices, int num_items, int rows, long long q_stride, int hq, int hkv, int d,
                             long long num_pages, float sm_scale, int dtype, int splits, float* part_o, float* part_ml,
                             int* status, cudaStream_t stream, const int* q_kvstart, const unsigned long long* tree_mask,
                             int sink, float softcap) {
  if (num_items <= 0) return 0;
  if (hkv <= 0 || hq <= 0 || hq % hkv || rows < 1 || rows > 16 || (d != 64 && d != 128 && d != 256)) return -1;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(pages)) & 15) return -2;
  if (q_stride % 8) return -2;
  if (dtype != 0 && dtype != 1) return -3;
  if (splits < 1 || (splits > 1 && (!part_o || !part_ml))) return -4;
  if (static_cast<long long>(num_items) * hkv * splits * 2 > 0x7fffffffLL || hkv > 65535) return -5;
  Kv4DecParams p;
  p.q = q;
  p.pages = static_cast<const uint8_t*>(pages);
  p.out = out;
  p.lse = lse;
  p.part_o = part_o;
  p.part_ml = part_ml;
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
  p.splits = splits;
  p.sink = q_kvstart ? sink : 0;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.cap_k = softcap > 0.f ? 2.f * 1.4426950408889634f * sm_scale / softcap : 0.f;
  p.cap_log2 = softcap > 0.f ? softcap * 1.4426950408889634f : 0.f;
  const bool ext = q_kvstart || tree_mask || softcap > 0.f;
  if (dtype == 0) {
    if (d == 64) return kv4_decode_shape<__half, 64>(p, rows, ext, num_items, stream);
    if (d == 128) return kv4_decode_shape<__half, 128>(p, rows, ext, num_items, stream);
    return kv4_decode_shape<__half, 256>(p, rows, ext, num_items, stream);
  }
  if (d == 64) return kv4_decode_shape<__nv_bfloat16, 64>(p, rows, ext, num_items, stream);
  if (d == 128) return kv4_decode_shape<__nv_bfloat16, 128>(p, rows, ext, num_items, stream);
  return kv4_decode_shape<__nv_bfloat16, 256>(p, rows, ext, num_items, stream);
}
