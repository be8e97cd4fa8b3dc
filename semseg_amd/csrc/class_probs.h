// Class probabilities of logits: what class_logprobs.hip (log probabilities, entropy, alternatives) and distill.hip (distillation) share.
//
// A row is one pixel (or token) with C logits.  Rows are addressed as r = i * p + j, class c of row r at z[i * sn + j * sp + c * sc]
// (element strides): sc = 1 is the engine's pixel-major score buffer ("rows"), sp = 1 a model's [N, C, H, W] output ("planes").
//
// With m = max_c z_c, d_c = (z_c - m) / T, S = sum exp(d_c):
//   lse = m / T + log S      log p_c = d_c - log S      entropy = log S - (sum exp(d_c) d_c) / S
// The maximum is subtracted from the logits themselves, before the temperature: the difference of two close fp32 values is exact, a
// logsumexp rounded to fp32 and subtracted later is not (at |z| ~ 1e3 it would cost 6e-5 of every log probability).  All sums are fp32
// over fp32 terms (16-bit logits are widened exactly), losses are summed over rows in fp64; results are rounded to 16 bits only where a
// gradient is stored in the logits' type.
#pragma once
#include "common.h"
#include "../../include/semseg_hip.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int MAXK = SEMSEG_CLASS_TOP_MAX;

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ float load1(const _Float16* p) { return (float)*p; }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__bf16* p, float v) { *p = (__bf16)v; }
__device__ __forceinline__ void store1(_Float16* p, float v) { *p = (_Float16)v; }

// Order of the alternatives as unsigned integers: larger logit first, NaN above everything, -0 = +0.  Never 0.
__device__ __forceinline__ unsigned order_key(float z) {
  const unsigned u = __float_as_uint(z + 0.f);
  const unsigned k = u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
  return z != z ? 0xfffffffeu : k;
}
// ... with the class as the second criterion: the lowest one first
__device__ __forceinline__ unsigned long long pair_key(float z, int c) {
  return ((unsigned long long)order_key(z) << 32) | (unsigned)~c;
}

// ---- reductions over groups of G = 4, 8 or 64 neighbouring lanes: data-parallel moves inside a row of 16 lanes, swaps of rows beyond
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) { return (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true); }
constexpr int XOR1 = 0xB1, XOR2 = 0x4E, HALF_MIRROR = 0x141, MIRROR = 0x140;
template <int G, typename T, typename F>
__device__ __forceinline__ T group_reduce(T v, F f) {
  static_assert(sizeof(T) == 4, "");
  const auto bits = [](T x) { return __builtin_bit_cast(unsigned, x); };
  const auto val = [](unsigned x) { return __builtin_bit_cast(T, x); };
  v = f(v, val(dpp<XOR1>(bits(v))));
  v = f(v, val(dpp<XOR2>(bits(v))));
  if (G >= 8) v = f(v, val(dpp<HALF_MIRROR>(bits(v))));
  if (G == 64) {
    v = f(v, val(dpp<MIRROR>(bits(v))));
    // both operands v: the odd rows (the upper half) of the one and the even rows (the lower half) of the other change places
    const auto r = __builtin_amdgcn_permlane16_swap(bits(v), bits(v), false, false);
    v = f(val(r[0]), val(r[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(bits(v), bits(v), false, false);
    v = f(val(h[0]), val(h[1]));
  }
  return v;
}
template <int G> __device__ __forceinline__ float group_max(float v) { return group_reduce<G>(v, [](float a, float b) { return fmaxf(a, b); }); }
template <int G> __device__ __forceinline__ float group_sum(float v) { return group_reduce<G>(v, [](float a, float b) { return a + b; }); }
template <int G> __device__ __forceinline__ unsigned group_umax(unsigned v) { return group_reduce<G>(v, [](unsigned a, unsigned b) { return a > b ? a : b; }); }
template <int G> __device__ __forceinline__ unsigned group_umin(unsigned v) { return group_reduce<G>(v, [](unsigned a, unsigned b) { return a < b ? a : b; }); }
// by two reductions: the high words, then the low words of those that have the highest
template <int G>
__device__ __forceinline__ unsigned long long group_max64(unsigned long long v) {
  const unsigned hi = group_umax<G>((unsigned)(v >> 32));
  const unsigned lo = group_umax<G>((unsigned)(v >> 32) == hi ? (unsigned)v : 0u);
  return (unsigned long long)hi << 32 | lo;
}
__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float log2_(float v) { return __builtin_amdgcn_logf(v); }

// ---- 16 bytes of logits at an element's own alignment: rows of odd lengths start anywhere, and global loads and stores of this hardware
// need no more than that
template <typename E> constexpr int VEC = 16 / (int)sizeof(E);
template <typename E>
using Vec = E __attribute__((ext_vector_type(16 / sizeof(E))));
template <typename E>
struct __attribute__((packed, aligned(alignof(E)))) Raw { u32x4 v; };
template <typename E>
__device__ __forceinline__ void load_vec(const E* p, float (&x)[VEC<E>]) {
  const Vec<E> q = __builtin_bit_cast(Vec<E>, reinterpret_cast<const Raw<E>*>(p)->v);
#pragma unroll
  for (int e = 0; e < VEC<E>; ++e) x[e] = (float)q[e];
}
template <typename E>
__device__ __forceinline__ void store_vec(E* p, const float (&x)[VEC<E>]) {
  Vec<E> q;
#pragma unroll
  for (int e = 0; e < VEC<E>; ++e) q[e] = (E)x[e];
  reinterpret_cast<Raw<E>*>(p)->v = __builtin_bit_cast(u32x4, q);
}
// VEC classes of a row of C from class s on; what lies beyond the row is -inf and not read.  Returns the class of x[0]: the row's last
// chunk is loaded from C - VEC, its classes below s (another lane has them) made -inf too.  SHORT: C may be less than VEC.
template <bool SHORT = false, typename E>
__device__ __forceinline__ int load_chunk(const E* z, int s, int C, float (&x)[VEC<E>]) {
  constexpr int V = VEC<E>;
  if (!SHORT || C >= V) {
    const int b = min(s, C - V);
    load_vec(z + b, x);
    if (b != s) {
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = b + e >= s ? x[e] : -INFINITY;
    }
    return b;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) x[e] = s + e < C ? load1(z + s + e) : -INFINITY;
  return s;
}
// N chunks of a row, the i-th from class first + i * step on, into x[i]; returns their first classes in b.  All loads go out before the
// first value is looked at (a branch for the cut chunk behind each load would make the loads wait for each other), chunks in the same
// place for all lanes are masked only where the row can end in one of them.
template <int N, bool SHORT, typename E>
__device__ __forceinline__ void load_chunks(const E* z, int first, int step, int C, float (&x)[N][VEC<E>], int (&b)[N]) {
  constexpr int V = VEC<E>;
  if (SHORT && C < V) {
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = load_chunk<true>(z, first + i * step, C, x[i]);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    b[i] = min(first + i * step, C - V);
    load_vec(z + b[i], x[i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (__any(first + i * step + V > C)) {
#pragma unroll
      for (int e = 0; e < V; ++e) x[i][e] = b[i] + e >= first + i * step ? x[i][e] : -INFINITY;
    }
}
// One chunk as it lies in memory (for a gradient: what it holds below class s is never stored), and its values
template <bool SHORT, typename E>
__device__ __forceinline__ int load_raw(const E* z, int s, int C, Vec<E>& q) {
  constexpr int V = VEC<E>;
  if (SHORT && C < V) {
#pragma unroll
    for (int e = 0; e < V; ++e) q[e] = s + e < C ? z[s + e] : (E)0.f;
    return s;
  }
  const int b = min(s, C - V);
  q = __builtin_bit_cast(Vec<E>, reinterpret_cast<const Raw<E>*>(z + b)->v);
  return b;
}
template <typename E>
__device__ __forceinline__ void store_chunk(E* z, int s, int b, int C, const float (&x)[VEC<E>]) {
  if (s + VEC<E> <= C) {
    store_vec(z + s, x);
  } else {
#pragma unroll
    for (int e = 0; e < VEC<E>; ++e)
      if (b + e >= s && b + e < C) store1(z + b + e, x[e]);
  }
}

template <int G, typename E>
__device__ __forceinline__ void zero_row(E* dz, int l, int C) {
  float x[VEC<E>];
#pragma unroll
  for (int e = 0; e < VEC<E>; ++e) x[e] = 0.f;
  for (int c = l * VEC<E>; c < C; c += G * VEC<E>) store_chunk(dz, c, C < VEC<E> ? c : min(c, C - VEC<E>), C, x);
}

struct Logits {
  const void* z;
  long long R, p, sn, sp, sc;
  int C;
  float invT, scale2;      // 1 / T, log2(e) / T
  double inv_p;            // 1 / p
  __device__ __forceinline__ long long at(long long r) const;
};
// i * s0 + j * s1 of row r = i * p + j.  r < 2^40: the quotient by a multiplication in fp64 is off by one at most (an integer division
// of 64 bits is ~150 instructions, and kernels of a few microseconds are short).
__device__ __forceinline__ long long row_at(const Logits& a, long long r, long long s0, long long s1) {
  if (a.p == a.R) return r * s1;
  long long i = (long long)((double)r * a.inv_p), j = r - i * a.p;
  if (j < 0) { --i; j += a.p; }
  if (j >= a.p) { ++i; j -= a.p; }
  return i * s0 + j * s1;
}
__device__ __forceinline__ long long Logits::at(long long r) const { return row_at(*this, r, sn, sp); }

// s, u taken about `from` become sums about `to` >= from (u's terms carry a factor d); an empty sum may come from -inf
__device__ __forceinline__ void rescale(float& s, float& u, float from, float to, float scale2) {
  const float d = (from - to) * scale2, f = exp2_(d);
  u = (u + s * fmaxf(d, -300.f)) * f;
  s = s * f;
}

// ---- sums over thousands of classes.  Equal terms that are added to a large sum one by one round the same way every time (65536 classes of
// two values: 1.3e-4 of log S), and so does a sum that is moved to a new base with every small rise of the maximum.  So a group of 8 to 32
// terms is added up by itself, the groups with what the last addition rounded away (`lost`) taken along, and the base of running sums follows
// the maximum only once the sum is to be halved at least: older moves fade with what they moved.
__device__ __forceinline__ void add_group(float& s, float& lost, float g) {
  const float y = g - lost, t = s + y;
  lost = (t - s) - y;
  s = t;
}
// `base` -inf: nothing to move yet
__device__ __forceinline__ bool must_move(float top, float base, float scale2) { return (top - base) * scale2 >= 1.f; }
__device__ __forceinline__ float usable(float base) { return base == -INFINITY ? 0.f : base; }
// A sum about the row's maximum holds a term 1: where its last move has rounded it below that, no probability gets above 1.  (NaN stays.)
__device__ __forceinline__ float at_least_one(float s) { return s > 0.f && s < 1.f ? 1.f : s; }
__device__ __forceinline__ float not_positive(float u) { return u > 0.f ? 0.f : u; }

// Running sums of e^d (s) and of e^d d (u) of one lane; d in units of log 2
struct RowSums {
  float m = -INFINITY, base = -INFINITY, s = 0.f, u = 0.f, lost_s = 0.f, lost_u = 0.f;      // m: the maximum so far
  // the maximum has become `top`: the base to take d about
  __device__ __forceinline__ float follow(float top, float scale2) {
    m = top;
    const bool mv = must_move(top, base, scale2);
    if (__any(mv)) {
      const float to = mv ? top : base, d = (base - usable(to)) * scale2, f = exp2_(d);
      u = (u + s * fmaxf(d, -300.f)) * f;
      s *= f;
      lost_u = (lost_u + lost_s * fmaxf(d, -300.f)) * f;
      lost_s *= f;
      base = to;
    }
    return usable(base);
  }
  __device__ __forceinline__ void add(float gs, float gu) {
    add_group(s, lost_s, gs);
    add_group(u, lost_u, gu);
  }
  // about the maximum itself (or a larger one)
  __device__ __forceinline__ void settle(float to, float scale2) { rescale(s, u, base, usable(to), scale2); }
};

// ---- planes: PV neighbouring pixels to a lane, classes in a loop; every load of a wave is one contiguous piece of a class's plane.
// Where planes are written, or a tile is a single wave, neighbouring tiles go to the same XCD (xcd_remap), so that what runs there at a
// time walks through one piece of every plane (the distillation gradient of 4 x 150 x 473 x 473: 229 us, with tiles dealt out in turn 265).
// A lane's address is a wave-uniform plane and 32 bits of its own: no 64-bit addresses in vector registers.
template <typename T>
__device__ __forceinline__ T load_at(const void* plane, unsigned bytes) {
  struct __attribute__((packed, aligned(2))) W { T v; };
  return reinterpret_cast<const W*>(static_cast<const char*>(plane) + bytes)->v;
}
template <typename T>
__device__ __forceinline__ void store_at(void* plane, unsigned bytes, T v) {
  struct __attribute__((packed, aligned(2))) W { T v; };
  reinterpret_cast<W*>(static_cast<char*>(plane) + bytes)->v = v;
}
template <int BYTES> struct Word;
template <> struct Word<2> { using type = unsigned short; };
template <> struct Word<4> { using type = unsigned; };
template <> struct Word<8> { using type = u32x2; };
template <typename E, int PV>
__device__ __forceinline__ void load_px(const E* plane, unsigned bytes, E (&q)[PV]) {
  const auto w = load_at<typename Word<PV * sizeof(E)>::type>(plane, bytes);
  __builtin_memcpy(q, &w, sizeof(w));
}
template <typename E, int PV>
__device__ __forceinline__ void store_px(E* plane, unsigned bytes, const E (&q)[PV]) {
  typename Word<PV * sizeof(E)>::type w;
  __builtin_memcpy(&w, q, sizeof(w));
  store_at(plane, bytes, w);
}
// Pixels of a tile that starts at pixel t0: lane `pl` has PV pixels from `px` on, those from `p0` on are its own (an image's last lane is
// moved back so that it loads whole pieces); `base` is a pixel that no lane of the tile is before.
template <int PV>
struct Px {
  long long px, p0, base;
  __device__ __forceinline__ Px(long long t0, int pl, long long P) {
    p0 = t0 + pl * PV;
    px = p0 < P - PV ? p0 : P - PV;
    base = t0 < PV ? 0 : t0 - PV;
  }
  __device__ __forceinline__ bool own(int v) const { return px + v >= p0; }
  template <typename T>
  __device__ __forceinline__ unsigned bytes() const { return (unsigned)(px - base) * (unsigned)sizeof(T); }
  // the own values of `x` to p, p + step, ...: together where they lie side by side
  template <typename T>
  __device__ __forceinline__ void put(T* p, long long step, const T (&x)[PV]) const {
    if (step == 1 && own(0)) {
      store_px<T, PV>(p, 0, x);
    } else {
#pragma unroll
      for (int v = 0; v < PV; ++v)
        if (own(v)) p[v * step] = x[v];
    }
  }
};
// tile and image of a block
__device__ __forceinline__ void tile_of(unsigned bid, int tiles, unsigned& image, unsigned& tile) {
  image = __builtin_amdgcn_readfirstlane(bid / (unsigned)tiles);
  tile = __builtin_amdgcn_readfirstlane(bid - image * (unsigned)tiles);
}

// ---- host side
inline bool logits_ok(const void* z, int type, long long n, long long p, int C, float T) {
  return z && type >= 0 && type <= 2 && n > 0 && p > 0 && C > 0 && C <= (1 << 30) && p <= (1ll << 40) / n && T >= 1e-15f && T <= 1e15f;      // T^2 and 1 / T far from the ends of fp32
}
// rows: contiguous classes; planes: contiguous pixels, and fewer than 2^31 tiles of 64 pixels
inline bool layout_ok(int C, long long n, long long p, long long sp, long long sc) {
  return C == 1 || sc == 1 || (sp == 1 && p < (1ll << 31) && n < (1ll << 31) / ((p + 63) / 64));
}
inline Logits logits_of(const void* z, long long n, long long p, int C, long long sn, long long sp, long long sc, float T) {
  return Logits{z, n * p, p, sn, sp, sc, C, 1.f / T, LOG2E / T, 1.0 / (double)p};
}

// Slices of a row of more classes than ROW_CLASSES: none with 512 rows or more (two blocks a compute unit), else about 1024 blocks in
// all, a slice no shorter than 4096 classes.
constexpr int ROW_CLASSES = SEMSEG_ROW_CLASSES;      // held in registers up to here
struct Split { int nsplit, slice, join; };
inline Split split_rows(int type, long long R, int C) {
  const int v = type == SEMSEG_TYPE_F32 ? 4 : 8;
  if (C <= ROW_CLASSES) return Split{1, C, 1};
  long long n = R >= 512 ? 1 : 1024 / R;
  if (n > 64) n = 64;
  if (n > (C + 4095) / 4096) n = (C + 4095) / 4096;
  const int slice = (int)(((C + n - 1) / n + v - 1) / v * v);
  const int iters = (slice + 256 * v - 1) / (256 * v);
  return Split{(C + slice - 1) / slice, slice, (iters + 127) / 128};
}
inline int capped(long long blocks, int cap) { return (int)(blocks < cap ? blocks : cap); }

// a block to every segment of a row, rows in a loop beyond what a grid holds
inline dim3 seg_grid(long long R, int C, int seg) {
  const int segs = (C + seg - 1) / seg, most = (1 << 23) / segs;
  return dim3(segs, capped(R, most < 1 ? 1 : most > 65535 ? 65535 : most));
}

// launch(first image, images): groups of images whose grids stay below 2^32 lanes
template <typename F>
void by_images(const Logits& a, long long tiles, F launch) {
  const long long n = a.R / a.p, most = tiles >= (1ll << 23) ? 1 : (1ll << 23) / tiles;
  for (long long i = 0; i < n; i += most) launch(i, (int)(n - i < most ? n - i : most));
}

#define BY_TYPE(type, F, ...)                                  \
  do {                                                         \
    if (type == SEMSEG_TYPE_F32) F<float>(__VA_ARGS__);        \
    else if (type == SEMSEG_TYPE_BF16) F<__bf16>(__VA_ARGS__); \
    else F<_Float16>(__VA_ARGS__);                             \
  } while (0)

}  // namespace
