// The 4-bit KV cache format, shared by its writer, its reader and the attention kernels.
//
// A cache row holds the D values of one (token, K or V, kv head). They are cut into groups of 32 channels; a
// group keeps its minimum lo and a step s = T((max - lo) * r), both in the type T of the rows (fp16 / bf16), and a 4-bit
// code c = clamp(rint((x - lo) / s), 0, 15) per value. The group stands for lo + s * c. r is 1 / 15 in fp32: the product is
// an fp32 rounding away from the quotient, costs one instruction, and is what dividing a CUDA tensor by 15.0 computes.
//
//   row bytes:  D / 2 code bytes | D / 32 x (lo, s)          (80 bytes for D = 128, against 256 in 16 bits)
//   code word:  8 channels in 32 bits; nibble i of the low half is channel 2 i, of the high half channel 2 i + 1
//
// The nibble order is the one the tensor-core kernels want: (w >> 4 i) & 0x000f000f is a pair of adjacent
// channels, and the same mask on two tokens' interleaved halves is a pair of adjacent tokens. Pages are
// [2, kv heads, page, row] like the 16-bit cache's, so the 16 rows of a head are one contiguous run.
#pragma once
#include "common.cuh"

namespace mlcb {

constexpr int KV4_GROUP = 32;
constexpr int KV4_PAGE = 16;  // tokens per page of the tensor-core kernels
__host__ __device__ constexpr int kv4_row_bytes(int d) { return d / 2 + d / KV4_GROUP * 4; }

// (w & mask) | bits in one instruction.
__device__ __forceinline__ uint32_t kv4_and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
  return r;
}

// Values are clamped to this bound before quantisation (NaN becomes 0), so that lo + 15 s stays finite in T
// however s was rounded: fp16 65440 (max + 131008 / 2048 < 65520), bf16 2^126.
template <typename T>
struct Kv4Type;
template <>
struct Kv4Type<__half> {
  static constexpr bool IS_BF16 = false;
  static constexpr float BOUND = 65440.f;
  // out[i] = pair of s * c_i + lo for the nibbles at bits 4 i of both halves. A nibble under the exponent of
  // 1024 (bits 0-3) or of 64 (bits 4-7) is the exact number 1024 + c or 64 + c: no int-to-float conversion, one
  // shift per word, and one rounding in the final fma.
  static __device__ __forceinline__ void expand4(uint32_t w, uint32_t s2, uint32_t lo2, uint32_t (&out)[4]) {
    const uint32_t w8 = w >> 8;
    const uint32_t x[4] = {kv4_and_or(w, 0x000f000fu, 0x64006400u), kv4_and_or(w, 0x00f000f0u, 0x54005400u),
                           kv4_and_or(w8, 0x000f000fu, 0x64006400u), kv4_and_or(w8, 0x00f000f0u, 0x54005400u)};
    const uint32_t bias[2] = {0x64006400u, 0x54005400u};
    const __half2 s = *reinterpret_cast<const __half2*>(&s2), lo = *reinterpret_cast<const __half2*>(&lo2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 c = __hsub2(*reinterpret_cast<const __half2*>(&x[i]), *reinterpret_cast<const __half2*>(&bias[i & 1]));
      const __half2 v = __hfma2(c, s, lo);
      out[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct Kv4Type<__nv_bfloat16> {
  static constexpr bool IS_BF16 = true;
  static constexpr float BOUND = 8.507059173023461586e37f;  // 2^126
  // as above; bf16 has 7 mantissa bits, so only the nibble at bits 0-3 fits (under the exponent of 128)
  static __device__ __forceinline__ void expand4(uint32_t w, uint32_t s2, uint32_t lo2, uint32_t (&out)[4]) {
    const uint32_t bias = 0x43004300u;
    const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&s2);
    const __nv_bfloat162 lo = *reinterpret_cast<const __nv_bfloat162*>(&lo2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = kv4_and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);
      const __nv_bfloat162 c =
          __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&bias));
      const __nv_bfloat162 v = __hfma2(c, s, lo);
      out[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

// Code of channel `ch` (0..7) of a word.
__device__ __forceinline__ int kv4_code(uint32_t w, int ch) { return (w >> ((ch & 1) * 16 + (ch >> 1) * 4)) & 15; }

// cap * tanh(x / cap) through exp2: tanh(y) = 1 - 2 / (1 + e^2y), off by about 1e-7 * cap, where the hardware's
// tanh approximation is off by 5e-4 of the value. `k` = 2 log2(e) * scale / cap. (e^2y = inf gives cap; NaN stays.)
__device__ __forceinline__ float kv4_softcap(float raw, float k, float cap) {
  return cap - __fdividef(2.f * cap, 1.f + exp2f(raw * k));
}

// Visibility of position `pos` to a query token (the rule of the 16-bit kernels): below kvlen all positions from
// `start` on and the first `sink`; from kvlen on the set bits of the tree mask.
__device__ __forceinline__ bool kv4_visible(int pos, int kvlen, int start, int sink, unsigned long long tm) {
  if (pos < kvlen) return pos >= start || pos < sink;
  const int r = pos - kvlen;
  return r < 64 && ((tm >> r) & 1ull);
}

// (a.x, a.y) * (b.x, b.y) + (c.x, c.y), and a sum of pairs, in one instruction each.
__device__ __forceinline__ float2 kv4_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 kv4_add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.ftz.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}

// N words from shared memory (the address is aligned to 16, 8 or 4 bytes for N = 4, 2, 1).
template <int N>
__device__ __forceinline__ void kv4_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x;
      w[4 * i + 1] = v.y;
      w[4 * i + 2] = v.z;
      w[4 * i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// bf16 rows are scaled by a power of two into fp16's range, one for many positions. What a position needs: with
// |lo| < 2^(e + 13) and s < 2^(e + 9) its scaled values, at most |lo| + 15 s, stay below 2^14. `top` is the largest pair
// (|lo|, s) of its groups, halves apart.
__device__ __forceinline__ int kv4_need(uint32_t top) {
  return max(static_cast<int>(top >> 23) - 9, static_cast<int>((top & 0xffffu) >> 7) - 13) - 126;
}
constexpr int KV4_NEEDS_NONE = -135;  // of zeros (and of what is as small: below 2^-113)
// What that rounds away is small against the largest value. A row is entitled to that of the largest value that it sees, which
// positions that only other rows see must not push out of fp16's range: later tokens, other branches of a draft tree, tokens below
// its window, an infinity among them. Where those need 2^KV4_WIDE times more than what the row is sure to see, all rows of the tile
// are computed again by kv4_rows_exact. Below that the largest value that a row sees keeps its 11 bits, and others are off by
// 2^-22 of it at most.
constexpr int KV4_WIDE = 12;

// KV4_EXACT query rows over positions at(i), 0 <= i < to (-1: none there), of which row r sees sees(r, position), in fp32 from the
// packed rows as they are, by one warp: lane = position for the scores, then lane = code word for the values, SHARE positions side
// by side. Gives per row the maximum (log2), the sum of the weights against it, and in the first D / 8 lanes the weighted sums of
// channels 8 lane .. 8 lane + 7. The rows share what is read and unpacked (64 verify chunks of four tokens at 4000 positions, 32 / 8
// heads of 128: 10 ms, one row at a time 30). It reads global memory with nothing to hide that behind, 40 to 100 times slower than
// the tensor cores, and is no path for ordinary values: 16 rows take 2 us per position, so that a million positions in one CTA would
// exhaust the waits of its other warps.
constexpr int KV4_EXACT = 4;
template <typename T, int D, typename At, typename Sees>
__device__ __forceinline__ void kv4_rows_exact(const uint8_t* pages, long long num_pages, const int* list, int hkv, int hk,
                                               const T* const (&q)[KV4_EXACT], float sign, float scale_log2, float cap_k, float cap_log2,
                                               int to, At&& at, Sees&& sees, float (&m)[KV4_EXACT], float (&l)[KV4_EXACT],
                                               float (&acc)[KV4_EXACT][8]) {
  constexpr int GROUPS = D / KV4_GROUP, ROW = kv4_row_bytes(D), WORDS = D / 8, SHARE = 32 / WORDS, R = KV4_EXACT;
  const int lane = threadIdx.x & 31, word = lane % WORDS;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[r][j] = 0.f;
  }
  const size_t to_v = static_cast<size_t>(hkv) * KV4_PAGE * ROW;
#pragma unroll 1
  for (int base = 0; base < to; base += 32) {
    const int pos = base + lane < to ? at(base + lane) : -1;
    bool see[R];
    unsigned long long key = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      see[r] = pos >= 0 && sees(r, pos);
      if (see[r]) key = 1;
    }
    if (key) {
      const int pg = list[pos / KV4_PAGE];
      key = 0;
      if (pg >= 0 && pg < num_pages)  // others are reported where the pages are copied
        key = reinterpret_cast<unsigned long long>(pages + ((static_cast<size_t>(pg) * 2 * hkv + hk) * KV4_PAGE + pos % KV4_PAGE) * ROW);
    }
    if (!__any_sync(0xffffffffu, key != 0)) continue;
    float score[R];
#pragma unroll
    for (int r = 0; r < R; ++r) score[r] = 0.f;
    if (key) {
      const uint32_t* row = reinterpret_cast<const uint32_t*>(key);
#pragma unroll 1
      for (int g = 0; g < GROUPS; ++g) {
        const uint32_t meta = row[WORDS + g];
        const T* pair = reinterpret_cast<const T*>(&meta);
        const float lo = Cvt<T>::to_f(pair[0]), st = Cvt<T>::to_f(pair[1]);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t w = row[g * 4 + x];
          float k[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) k[j] = fmaf(st, static_cast<float>(kv4_code(w, j)), lo);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const uint4 v = reinterpret_cast<const uint4*>(q[r])[g * 4 + x];
            const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
            for (int j = 0; j < 8; ++j) score[r] = fmaf(Cvt<T>::to_f(e[j]), k[j], score[r]);
          }
        }
      }
    }
    float weight[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float sc = score[r] * sign;
      sc = cap_log2 != 0.f ? kv4_softcap(sc, cap_k, cap_log2) : sc * scale_log2;
      if (!see[r] || !key) sc = -INFINITY;
      const float mn = fmaxf(m[r], warp_max(sc)), f = m[r] == -INFINITY ? 0.f : exp2f(m[r] - mn);
      weight[r] = see[r] && key ? exp2f(sc - (mn == -INFINITY ? 0.f : mn)) : 0.f;
      m[r] = mn;
      l[r] = l[r] * f + weight[r];
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[r][j] *= f;
    }
#pragma unroll 2
    for (int x = 0; x < 32; x += SHARE) {
      const int from = (x + lane / WORDS) & 31;
      float w[R];
#pragma unroll
      for (int r = 0; r < R; ++r) w[r] = __shfl_sync(0xffffffffu, weight[r], from);
      const unsigned long long row = __shfl_sync(0xffffffffu, key, from);
      if (lane >= SHARE * WORDS || !row) continue;
      const uint32_t* v = reinterpret_cast<const uint32_t*>(row + to_v);
      const uint32_t code = v[word], meta = v[WORDS + word / 4];
      const T* pair = reinterpret_cast<const T*>(&meta);
      const float lo = Cvt<T>::to_f(pair[0]), st = Cvt<T>::to_f(pair[1]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = fmaf(st, static_cast<float>(kv4_code(code, j)), lo);
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][j] = fmaf(w[r], y, acc[r][j]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] = warp_sum(l[r]);
#pragma unroll
    for (int o = SHARE / 2 * WORDS; o >= WORDS; o /= 2)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[r][j] += __shfl_down_sync(0xffffffffu, acc[r][j], o);
  }
}
// 8 neighbouring channels of a row, as fp32 and in the rows' type.
__device__ __forceinline__ void kv4_put8(float* dst, const float (&v)[8]) {
  reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename T>
__device__ __forceinline__ void kv4_put8(T* dst, const float (&v)[8], float by) {
  *reinterpret_cast<uint4*>(dst) = make_uint4(Kv4Type<T>::pack(v[0] * by, v[1] * by), Kv4Type<T>::pack(v[2] * by, v[3] * by),
                                              Kv4Type<T>::pack(v[4] * by, v[5] * by), Kv4Type<T>::pack(v[6] * by, v[7] * by));
}

// Waits until phase `parity` of a barrier is over, no matter whether a wait of some role ran out: before a CTA gives up its
// shared memory and TMEM, the copies and products in flight have to land. They do so by themselves; the limit (about 50 ms)
// is for a phase that the hardware never ends.
__device__ __forceinline__ void kv4_drain(uint64_t* bar, uint32_t parity) {
  for (int i = 0; i < 256 && !mbar_try_wait_parked(bar, parity); ++i) {
  }
}

}  // namespace mlcb
