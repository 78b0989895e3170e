// Writing and reading the 4-bit paged KV cache (format: kv4.cuh), and its generic attention kernel.
//
// Reference counterpart: the append and attention functions of the paged KV cache (nn/kv_cache.py:16-93), whose
// pages hold 16-bit values only.
#include "kv4.cuh"

#include <type_traits>

namespace mlcb {

// ------------------------------------------------------------------ append
// Rotates the q and k heads of one token's fused projection row in place (as rope_append_kernel does) and writes
// its k and v heads, quantised, to the token's slot.
//
// The angle pos * inv_freq, its sine and cosine and the rotation of k are computed in 64 bits. In 32 bits the
// angle alone is off by 4e-3 at position 131071, and a key that lands on the other side of a rounding border
// becomes another code, 1/15 of its group's range away. 64-bit arithmetic costs little here: 64 angles and
// 1024 keys per token for 8 heads of 128.
// q only feeds products and is rotated in 32 bits with the 64-bit sines.
//
// A block takes one token and `parts` of its kv heads (and their share of the q heads): with one part the
// angles are computed once per token, which is what many tokens want; few tokens are cut into more parts so that
// more SMs share the row. Four neighbouring lanes own a group of 32 channels (one 16-byte load each).
constexpr int KV4_APPEND_THREADS = 256;

// Sine and cosine of x radians. x / pi is taken in two terms, so that the error stays that of one rounding near 1 however
// far the position is: with one term it is x 2^-53, which at 131071 moved a key of some million across a rounding border.
__device__ __forceinline__ void kv4_sincos(double x, double& s, double& c) {
  constexpr double INV_PI = 0.3183098861837907, INV_PI_REST = -1.9678676675182486e-17;
  const double turns = x * INV_PI;
  const double rest = fma(x, INV_PI_REST, fma(x, INV_PI, -turns));
  sincospi(fma(-2.0, rint(0.5 * turns), turns) + rest, &s, &c);
}

template <typename T>
__device__ __forceinline__ float kv4_sane(float v) {
  // fmaxf / fminf would turn NaN into a bound
  return v != v ? 0.f : fminf(fmaxf(v, -Kv4Type<T>::BOUND), Kv4Type<T>::BOUND);
}

// Magnitude bits of KV4 bounds: larger ones (infinity and NaN among them) are clamped before quantisation.
template <typename T>
constexpr uint32_t KV4_BOUND_BITS = 0;
template <>
constexpr uint32_t KV4_BOUND_BITS<__half> = 0x7bfdu;          // 65440
template <>
constexpr uint32_t KV4_BOUND_BITS<__nv_bfloat16> = 0x7e80u;   // 2^126

// The codes by the letter of the format: correctly rounded divisions.
__device__ __noinline__ uint32_t kv4_codes_exact(const float (&f)[8], float lo, float s) {
  uint32_t w = 0;
  for (int j = 0; j < 8; ++j) {
    const int c = min(15, __float2int_rn(__fdiv_rn(__fsub_rn(f[j], lo), s)));  // f >= lo: never negative
    w |= static_cast<uint32_t>(c) << ((j & 1) * 16 + (j >> 1) * 4);
  }
  return w;
}

// Quantises the 8 values of `val` (lanes 4 i .. 4 i + 3 hold one group) and stores code word and minimum / step.
// A code is rint of a quotient in [0, 15.1]. The reciprocal gives that quotient to 4e-6, so that only one within 6e-5
// of a half-way point could round elsewhere: those words, and ones whose step is too coarse for the range (subnormal),
// take the exact path. A division per value cost 3 200 of a token's 7 400 warp instructions.
template <typename T>
__device__ __forceinline__ void kv4_store8(const uint4& val, uint8_t* row, int chunk, int code_bytes) {
  const uint32_t bits[4] = {val.x, val.y, val.z, val.w};
  const T* e = reinterpret_cast<const T*>(bits);
  uint32_t mag = 0;
  float f[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) mag = __vmaxu2(mag, bits[j] & 0x7fff7fffu);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = Cvt<T>::to_f(e[j]);
  if (max(mag & 0xffffu, mag >> 16) > KV4_BOUND_BITS<T>) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = kv4_sane<T>(f[j]);
  }
  float lo = fminf(fminf(fminf(f[0], f[1]), fminf(f[2], f[3])), fminf(fminf(f[4], f[5]), fminf(f[6], f[7])));
  float hi = fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
  const unsigned quad = 0xfu << (threadIdx.x & 28);
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(quad, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(quad, hi, o));
  }
  const float range = __fsub_rn(hi, lo);
  const T st = Cvt<T>::from_f(__fmul_rn(range, 1.f / 15.f));
  const float s = Cvt<T>::to_f(st);
  uint32_t w = 0;
  if (s > 0.f) {
    const float inv = __fdividef(1.f, s);
    const float magic = 12582912.f;  // 1.5 * 2^23: a sum with it is rounded to a whole number, held in its low bits
    float far = 0.f;
    uint32_t sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = __fmul_rn(__fsub_rn(f[j], lo), inv);
      const float y = __fadd_rn(t, magic);
      far = fmaxf(far, fabsf(__fsub_rn(t, __fsub_rn(y, magic))));
      sum += __float_as_uint(y) << ((j & 1) * 16 + (j >> 1) * 4);
    }
    // the magic number's own bits, 0x4b400000 << 0, 4, 8, 12 (16 and more shift them out): 0x4b400000 * 0x1111 mod 2^32
    w = sum - 0x4b400000u * 0x1111u;
    const bool sure = far < 0.5f - 6e-5f && __fmul_rn(range, inv) < 15.4f;  // not so for NaN
    if (!sure) w = kv4_codes_exact(f, lo, s);
  }
  reinterpret_cast<uint32_t*>(row)[chunk] = w;
  if ((chunk & 3) == 0) {
    T meta[2] = {Cvt<T>::from_f(lo), st};
    reinterpret_cast<uint32_t*>(row + code_bytes)[chunk >> 2] = *reinterpret_cast<uint32_t*>(meta);
  }
}

template <typename T>
__global__ void __launch_bounds__(KV4_APPEND_THREADS)
kv4_append_kernel(T* __restrict__ qkv, uint8_t* __restrict__ pages, const int* __restrict__ pos,
                  const int* __restrict__ slot, const float* __restrict__ inv_freq, int hq, int hkv, int d,
                  int rot_dim, int page, double attn_factor, long long num_slots, int* status) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int half = rot_dim / 2;
  double* sn = reinterpret_cast<double*>(smem);  // [half]
  double* cs = sn + half;
  T* krow = reinterpret_cast<T*>(cs + half);     // [kv heads of this part][d]
  const int t = blockIdx.x, parts = gridDim.y, part = blockIdx.y;
  const int k0 = hkv * part / parts, k1 = hkv * (part + 1) / parts;
  const int q0 = hq * part / parts, q1 = hq * (part + 1) / parts;
  T* row = qkv + static_cast<size_t>(t) * (hq + 2 * hkv) * d;
  if (half) {
    const double p = static_cast<double>(pos[t]);
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
      double s, c;
      kv4_sincos(p * static_cast<double>(inv_freq[j]), s, c);
      sn[j] = s * attn_factor;
      cs[j] = c * attn_factor;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (q1 - q0) * half; i += blockDim.x) {
      T* hp = row + (q0 + i / half) * static_cast<size_t>(d);
      const int j = i % half;
      const float a = Cvt<T>::to_f(hp[j]), b = Cvt<T>::to_f(hp[j + half]);
      const float c = static_cast<float>(cs[j]), s = static_cast<float>(sn[j]);
      hp[j] = Cvt<T>::from_f(a * c - b * s);
      hp[j + half] = Cvt<T>::from_f(b * c + a * s);
    }
  }
  // keys: rotated into shared memory (and back into the row), the unrotated tail copied
  for (int i = threadIdx.x; i < (k1 - k0) * (d - half); i += blockDim.x) {
    const int h = i / (d - half), j = i % (d - half);
    T* hp = row + (hq + k0 + h) * static_cast<size_t>(d);
    T* kp = krow + h * d;
    if (j < half) {
      const double a = static_cast<double>(Cvt<T>::to_f(hp[j])), b = static_cast<double>(Cvt<T>::to_f(hp[j + half]));
      const T lo = Cvt<T>::from_f(static_cast<float>(a * cs[j] - b * sn[j]));
      const T hi = Cvt<T>::from_f(static_cast<float>(b * cs[j] + a * sn[j]));
      kp[j] = lo;
      kp[j + half] = hi;
      hp[j] = lo;
      hp[j + half] = hi;
    } else {
      kp[j + half] = hp[j + half];
    }
  }
  const long long sl = slot[t];
  if (sl < 0) return;  // rotate only
  if (sl >= num_slots) {
    if (threadIdx.x == 0 && status) atomicCAS(status, 0, ERR_BAD_INDEX);
    return;
  }
  __syncthreads();
  const int rb = kv4_row_bytes(d), cpr = d / 8;  // row bytes, 8-channel chunks per row
  const int heads = k1 - k0;
  for (int i = threadIdx.x; i < 2 * heads * cpr; i += blockDim.x) {
    const int kv = i / (heads * cpr), h = i / cpr % heads, chunk = i % cpr;
    const uint4 val = kv == 0
                          ? *reinterpret_cast<const uint4*>(krow + h * d + chunk * 8)
                          : *reinterpret_cast<const uint4*>(row + (hq + hkv + k0 + h) * static_cast<size_t>(d) + chunk * 8);
    uint8_t* dst = pages + (((sl / page * 2 + kv) * hkv + k0 + h) * page + sl % page) * static_cast<size_t>(rb);
    kv4_store8<T>(val, dst, chunk, d / 2);
  }
}

// The same for heads that are rotated as a whole (D = 64, 128, 256), which is what most models do. A thread takes one
// 16-byte item of 8 rotary pairs of q, two pairs of k (4 bytes each side) and one code word: at 32 / 8 heads of 128 that
// is one of each for all 256 threads, loaded before the angles are computed. k passes through shared memory between
// its rotation, whose 64-bit pairs want all threads, and its quantisation, where four neighbouring lanes own a group.
template <typename T, int D>
__global__ void __launch_bounds__(KV4_APPEND_THREADS)
kv4_append_whole_kernel(T* __restrict__ qkv, uint8_t* __restrict__ pages, const int* __restrict__ pos,
                        const int* __restrict__ slot, const float* __restrict__ inv_freq, int hq, int hkv, int page,
                        double attn_factor, long long num_slots, int* status) {
  constexpr int HALF = D / 2, JG = HALF / 8, CPR = D / 8, RB = kv4_row_bytes(D), STEP = KV4_APPEND_THREADS;
  __shared__ __align__(16) double sn[HALF], cs[HALF];
  __shared__ float snf[HALF], csf[HALF];
  extern __shared__ __align__(16) uint8_t smem[];
  T* krow = reinterpret_cast<T*>(smem);  // [kv heads of this part][D]
  const int t = blockIdx.x, parts = gridDim.y, part = blockIdx.y;
  const int k0 = hkv * part / parts, kn = hkv * (part + 1) / parts - k0;
  const int q0 = hq * part / parts, qn = hq * (part + 1) / parts - q0;
  const int nq = qn * JG, nk = kn * (HALF / 2), nw = kn * CPR;  // q items, k items, words of k (and of v)
  T* row = qkv + static_cast<size_t>(t) * (hq + 2 * hkv) * D;
  T* qrow = row + q0 * D;
  T* ksrc = row + (hq + k0) * D;
  const T* vsrc = row + (hq + hkv + k0) * D;
  auto q_at = [&](int i) { return reinterpret_cast<uint4*>(qrow + i / JG * D + i % JG * 8); };
  auto k_at = [&](int i) { return reinterpret_cast<uint32_t*>(ksrc + i / (HALF / 2) * D + i % (HALF / 2) * 2); };
  const int tid = threadIdx.x;
  uint4 qa, qb, v;
  uint32_t ka = 0, kb = 0;
  qa = qb = v = make_uint4(0, 0, 0, 0);
  if (tid < nq) {
    qa = q_at(tid)[0];
    qb = q_at(tid)[HALF / 8];
  }
  if (tid < nk) {
    ka = k_at(tid)[0];
    kb = k_at(tid)[HALF / 2];
  }
  if (tid >= nw && tid < 2 * nw) v = reinterpret_cast<const uint4*>(vsrc)[tid - nw];
  const long long sl = slot[t];
  const double p = static_cast<double>(pos[t]);
  for (int j = tid; j < HALF; j += STEP) {
    double s, c;
    kv4_sincos(p * static_cast<double>(inv_freq[j]), s, c);
    sn[j] = s * attn_factor;
    cs[j] = c * attn_factor;
    const int at = j % 8 * JG + j / 8;  // the JG items of a head read neighbouring words
    snf[at] = static_cast<float>(sn[j]);
    csf[at] = static_cast<float>(cs[j]);
  }
  __syncthreads();
  for (int i = tid; i < nk; i += STEP) {
    uint32_t* g = k_at(i);
    if (i != tid) {
      ka = g[0];
      kb = g[HALF / 2];
    }
    T* a = reinterpret_cast<T*>(&ka);
    T* b = reinterpret_cast<T*>(&kb);
    const int j0 = i % (HALF / 2) * 2;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const double u = static_cast<double>(Cvt<T>::to_f(a[j])), w = static_cast<double>(Cvt<T>::to_f(b[j]));
      a[j] = Cvt<T>::from_f(static_cast<float>(u * cs[j0 + j] - w * sn[j0 + j]));
      b[j] = Cvt<T>::from_f(static_cast<float>(w * cs[j0 + j] + u * sn[j0 + j]));
    }
    g[0] = ka;
    g[HALF / 2] = kb;
    uint32_t* sk = reinterpret_cast<uint32_t*>(krow + i / (HALF / 2) * D + j0);
    sk[0] = ka;
    sk[HALF / 2] = kb;
  }
  for (int i = tid; i < nq; i += STEP) {
    uint4* g = q_at(i);
    if (i != tid) {
      qa = g[0];
      qb = g[HALF / 8];
    }
    T* a = reinterpret_cast<T*>(&qa);
    T* b = reinterpret_cast<T*>(&qb);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float u = Cvt<T>::to_f(a[j]), w = Cvt<T>::to_f(b[j]), c = csf[j * JG + i % JG], s = snf[j * JG + i % JG];
      a[j] = Cvt<T>::from_f(u * c - w * s);
      b[j] = Cvt<T>::from_f(w * c + u * s);
    }
    g[0] = qa;
    g[HALF / 8] = qb;
  }
  if (sl < 0) return;  // rotate only
  if (sl >= num_slots) {
    if (tid == 0 && status) atomicCAS(status, 0, ERR_BAD_INDEX);
    return;
  }
  __syncthreads();
  uint8_t* dst = pages + ((sl / page * 2 * hkv + k0) * page + sl % page) * static_cast<size_t>(RB);
  for (int i = tid; i < 2 * nw; i += STEP) {
    const int kv = i >= nw, j = kv ? i - nw : i, h = j / CPR;
    const uint4 x = kv ? (i == tid ? v : reinterpret_cast<const uint4*>(vsrc)[j]) : reinterpret_cast<const uint4*>(krow)[j];
    kv4_store8<T>(x, dst + (static_cast<size_t>(kv * hkv) + h) * page * RB, j % CPR, D / 2);
  }
}

// ------------------------------------------------------------------ read back
// Values of the rows at slot[t]: k, v [T, hkv, d]. A thread expands one code word (8 channels, 16 bytes out) of
// N tokens, whose loads it issues together; which word that is costs its divisions once. Bound by the bytes: those
// written are 3.2 times those read. Negative slots read as zeros. 65536 scattered rows of 8 heads of 128 (153 MB read:
// 80-byte rows touch sectors of their neighbours; 268 MB written): N = 1 122 us, 2 100 us, 4 88 us, 8 96 us; with the page
// found by multiplication 4 85 us (4.1 TB/s of wanted bytes; divided: 88). 77 rows: 1 2.7 us, 4 3.9 us.
template <typename T, int N>
__global__ void __launch_bounds__(256)
kv4_read_kernel(const uint8_t* __restrict__ pages, const int* __restrict__ slot, T* __restrict__ k, T* __restrict__ v,
                int tokens, int hkv, int d, uint32_t page, uint32_t inv_page, long long num_slots, int* status) {
  const int cpr = d / 8;
  const int i = blockIdx.y * 256 + threadIdx.x;
  if (i >= 2 * hkv * cpr) return;
  const int kv = i / (hkv * cpr), h = i / cpr % hkv, chunk = i % cpr;
  const int t0 = blockIdx.x * N;
  const size_t rb = kv4_row_bytes(d);
  uint32_t w[N], meta[N];
#pragma unroll
  for (int x = 0; x < N; ++x) {
    w[x] = meta[x] = 0u;
    const int sl = t0 + x < tokens ? slot[t0 + x] : -1;
    if (sl >= num_slots) {
      if (status) atomicCAS(status, 0, ERR_BAD_INDEX);
    } else if (sl >= 0) {
      uint32_t pg = __umulhi(static_cast<uint32_t>(sl), inv_page), in = static_cast<uint32_t>(sl) - pg * page;
      if (in >= page) {
        ++pg;
        in -= page;
      }
      const uint8_t* row = pages + ((static_cast<size_t>(pg * 2 + kv) * hkv + h) * page + in) * rb;
      w[x] = reinterpret_cast<const uint32_t*>(row)[chunk];
      meta[x] = reinterpret_cast<const uint32_t*>(row + d / 2)[chunk >> 2];
    }
  }
  T* dst = (kv ? v : k) + (static_cast<size_t>(t0) * hkv + h) * d + chunk * 8;
#pragma unroll
  for (int x = 0; x < N; ++x) {
    if (t0 + x >= tokens) return;
    uint32_t out[4];
    Kv4Type<T>::expand4(w[x], __byte_perm(meta[x], meta[x], 0x3232), __byte_perm(meta[x], meta[x], 0x1010), out);
    *reinterpret_cast<uint4*>(dst + static_cast<size_t>(x) * hkv * d) = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

// ------------------------------------------------------------------ generic attention
// Any head size that is a multiple of 32 up to 256, any page size, any mask: one block per (query token, q head),
// a warp per cached position, lane = channel of each group. It serves the shapes without a tensor-core kernel
// (head sizes other than 64, 128 and 256, pages other than 16 tokens, calls without a plan).
struct Kv4SimtArgs {
  const void* q;
  const uint8_t* pages;
  void* out;
  float* lse;
  const int *q_seq, *q_kvlen, *q_kvstart;
  const unsigned long long* tree_mask;
  const int *page_indptr, *page_indices;
  int* status;
  long long q_stride, num_pages;
  int hq, hkv, d, page, sink;
  float sm_scale, softcap;
};

template <typename T>
__global__ void __launch_bounds__(128) kv4_attn_simt_kernel(const Kv4SimtArgs a) {
  const int t = blockIdx.x, h = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = a.d / 32;
  const int hk = h / (a.hq / a.hkv), b = a.q_seq[t];
  const int kvlen = a.q_kvlen[t];
  const int start = a.q_kvstart ? a.q_kvstart[t] : 0;
  const unsigned long long tm = a.tree_mask ? a.tree_mask[t] : 0ull;
  const int* pages = a.page_indices + a.page_indptr[b];
  const long long room = static_cast<long long>(a.page_indptr[b + 1] - a.page_indptr[b]) * a.page;
  long long total = static_cast<long long>(kvlen) + (tm ? 64 - __clzll(tm) : 0);
  if (total > room) {  // more positions than the sequence has pages for: never dereferenced
    if (threadIdx.x == 0 && a.status) atomicCAS(a.status, 0, ERR_BAD_INDEX);
    total = room;
  }
  const T* qp = reinterpret_cast<const T*>(a.q) + static_cast<size_t>(t) * a.q_stride + static_cast<size_t>(h) * a.d;
  float qv[8], acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    qv[i] = i < groups ? Cvt<T>::to_f(qp[lane + 32 * i]) : 0.f;
    acc[i] = 0.f;
  }
  const size_t rb = kv4_row_bytes(a.d);
  float m = -INFINITY, l = 0.f;
  for (int j = warp; j < total; j += 4) {
    const bool seen = j < kvlen ? (j < a.sink || j >= start) : ((tm >> (j - kvlen)) & 1ull) != 0;
    if (!seen) continue;
    const int pg = pages[j / a.page], off = j % a.page;
    if (pg < 0 || pg >= a.num_pages) {
      if (lane == 0 && a.status) atomicCAS(a.status, 0, ERR_BAD_INDEX);
      continue;
    }
    const uint8_t* kp = a.pages + ((static_cast<size_t>(pg) * 2 * a.hkv + hk) * a.page + off) * rb;
    const uint8_t* vp = kp + static_cast<size_t>(a.hkv) * a.page * rb;
    auto value = [&](const uint8_t* row, int i) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(row)[i * 4 + (lane >> 3)];
      const T* meta = reinterpret_cast<const T*>(row + a.d / 2) + 2 * i;
      return fmaf(Cvt<T>::to_f(meta[1]), static_cast<float>(kv4_code(w, lane & 7)), Cvt<T>::to_f(meta[0]));
    };
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < groups) s = fmaf(qv[i], value(kp, i), s);
    s = warp_sum(s) * a.sm_scale;
    if (a.softcap > 0.f) s = kv4_softcap(s, 2.f * 1.4426950408889634f / a.softcap, a.softcap);
    const float mn = fmaxf(m, s);
    const float corr = __expf(m - mn), pe = __expf(s - mn);
    l = l * corr + pe;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < groups) acc[i] = fmaf(pe, value(vp, i), acc[i] * corr);
    m = mn;
  }
  __shared__ float sm_m[4], sm_l[4], sm_acc[4][256];
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < groups) sm_acc[warp][lane + 32 * i] = acc[i];
  __syncthreads();
  const float M = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
  float L = 0.f, w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    w[k] = sm_m[k] == -INFINITY ? 0.f : __expf(sm_m[k] - M);
    L += sm_l[k] * w[k];
  }
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);  // an empty row is 0, NaN stays NaN
  T* op = reinterpret_cast<T*>(a.out) + (static_cast<size_t>(t) * a.hq + h) * a.d;
  for (int c = threadIdx.x; c < a.d; c += 128) {
    float o = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) o = fmaf(sm_acc[k][c], w[k], o);
    op[c] = Cvt<T>::from_f(o * inv);
  }
  if (a.lse && threadIdx.x == 0)
    a.lse[static_cast<size_t>(t) * a.hq + h] = L == 0.f ? -INFINITY : M + logf(L);
}

}  // namespace mlcb

using namespace mlcb;

// Return codes of the kv4 entry points: -1 shape, -2 alignment, -3 type, -4 out of grid range, > 0 a CUDA error.
MLCB_API int mlcb_kv4_append(void* qkv, void* pages, const int* pos, const int* slot, const float* inv_freq, int tokens,
                             int hq, int hkv, int d, int rot_dim, int page, double attn_factor, long long num_slots,
                             int dtype, int* status, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (hq < 0 || hkv <= 0 || d <= 0 || d % 32 || d > 256 || rot_dim < 0 || rot_dim % 2 || rot_dim > d || page <= 0) return -1;
  if ((reinterpret_cast<uintptr_t>(qkv) & 15) || (reinterpret_cast<uintptr_t>(pages) & 3)) return -2;
  if (dtype != 0 && dtype != 1) return -3;
  // fewer tokens than two blocks per SM: cut the heads so that the blocks still cover the GPU
  int parts = 1;
  while (parts < hkv && static_cast<long long>(tokens) * parts < 2LL * sm_count()) parts *= 2;
  if (parts > hkv) parts = hkv;
  // Shared memory of a block: the keys of its heads, and 64-bit sines, which the kernel for whole heads holds in static arrays
  // (with a 32-bit copy). Both count against the 48 KB that a launch gets without asking for more.
  const bool whole = rot_dim == d && (d == 64 || d == 128 || d == 256);
  const size_t fixed = static_cast<size_t>(whole ? 12 * d : 0), sines = whole ? 0 : static_cast<size_t>(rot_dim) * 8;
  auto bytes = [&] { return sines + static_cast<size_t>((hkv + parts - 1) / parts) * d * 2; };
  while (fixed + bytes() > 48 * 1024) parts *= 2;  // more kv heads than fit: ends at one head, under 4 KB
  const size_t smem = bytes();
  const dim3 grid(tokens, parts);
  auto run = [&](auto* rows) {
    using T = std::remove_pointer_t<decltype(rows)>;
    uint8_t* dst = static_cast<uint8_t*>(pages);
    if (whole) {
      auto kern = d == 64 ? kv4_append_whole_kernel<T, 64> : d == 128 ? kv4_append_whole_kernel<T, 128> : kv4_append_whole_kernel<T, 256>;
      kern<<<grid, KV4_APPEND_THREADS, smem, stream>>>(rows, dst, pos, slot, inv_freq, hq, hkv, page, attn_factor, num_slots, status);
    } else {
      kv4_append_kernel<T><<<grid, KV4_APPEND_THREADS, smem, stream>>>(rows, dst, pos, slot, inv_freq, hq, hkv, d, rot_dim, page,
                                                                       attn_factor, num_slots, status);
    }
  };
  if (dtype == 0) run(static_cast<__half*>(qkv));
  else run(static_cast<__nv_bfloat16*>(qkv));
  count_launch();
  return static_cast<int>(cudaGetLastError());
}

MLCB_API int mlcb_kv4_read(const void* pages, const int* slot, void* k, void* v, int tokens, int hkv, int d, int page,
                           long long num_slots, int dtype, int* status, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (hkv <= 0 || d <= 0 || d % 32 || d > 256 || page <= 0) return -1;
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) || (reinterpret_cast<uintptr_t>(pages) & 3)) return -2;
  if (dtype != 0 && dtype != 1) return -3;
  const int words = (2 * hkv * (d / 8) + 255) / 256;
  if (words > 65535) return -4;
  // four tokens per thread once that still leaves two blocks per SM
  const int n = static_cast<long long>(tokens) * words >= 8LL * sm_count() ? 4 : 1;
  const dim3 grid((tokens + n - 1) / n, words);
  // floor(slot / page) by multiplication with floor((2^32 - 1) / page): for slots below 2^31 short by at most one
  const uint32_t inv_page = 0xffffffffu / static_cast<uint32_t>(page);
  auto run = [&](auto* rows) {
    using T = std::remove_pointer_t<decltype(rows)>;
    auto kern = n == 4 ? kv4_read_kernel<T, 4> : kv4_read_kernel<T, 1>;
    kern<<<grid, 256, 0, stream>>>(static_cast<const uint8_t*>(pages), slot, rows, static_cast<T*>(v), tokens, hkv, d,
                                   static_cast<uint32_t>(page), inv_page, num_slots, status);
  };
  if (dtype == 0) run(static_cast<__half*>(k));
  else run(static_cast<__nv_bfloat16*>(k));
  count_launch();
  return static_cast<int>(cudaGetLastError());
}

MLCB_API int mlcb_kv4_attn_simt(const void* q, const void* pages, void* out, float* lse, const int* q_seq,
                                const int* q_kvlen, const int* q_kvstart, const unsigned long long* tree_mask,
                                const int* page_indptr, const int* page_indices, int tokens, long long q_stride, int hq,
                                int hkv, int d, int page, long long num_pages, int sink, float sm_scale, float softcap,
                                int dtype, int* status, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (hkv <= 0 || hq <= 0 || hq % hkv || d <= 0 || d % 32 || d > 256 || page <= 0) return -1;
  if (reinterpret_cast<uintptr_t>(pages) & 3) return -2;
  if (dtype != 0 && dtype != 1) return -3;
  if (hq > 65535) return -4;
  Kv4SimtArgs a{q,        static_cast<const uint8_t*>(pages), out, lse, q_seq, q_kvlen, q_kvstart, tree_mask, page_indptr,
                page_indices, status, q_stride, num_pages, hq, hkv, d, page, q_kvstart ? sink : 0, sm_scale, softcap};
  dim3 grid(tokens, hq);
  if (dtype == 0)
    kv4_attn_simt_kernel<__half><<<grid, 128, 0, stream>>>(a);
  else
    kv4_attn_simt_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(a);
  count_launch();
  return static_cast<int>(cudaGetLastError());
}
