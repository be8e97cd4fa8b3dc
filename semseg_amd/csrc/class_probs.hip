// Class probabilities of logits: log probability of a given class, entropy and the k best classes of every row (forward, backward),
// and the distillation loss against a teacher's stored top logits (forward, backward).
//
// A row is one pixel (or token) with C logits.  Rows are addressed as r = i * p + j, class c of row r at z[i * sn + j * sp + c * sc]
// (element strides): sc = 1 is the engine's pixel-major score buffer ("rows"), sp = 1 a model's [N, C, H, W] output ("planes").
//
// With m = max_c z_c, d_c = (z_c - m) / T, S = sum exp(d_c):
//   lse = m / T + log S      log p_c = d_c - log S      entropy = log S - (sum exp(d_c) d_c) / S
// The maximum is subtracted from the logits themselves, before the temperature: the difference of two close fp32 values is exact, a
// logsumexp rounded to fp32 and subtracted later is not (at |z| ~ 1e3 it would cost 6e-5 of every log probability).  All sums are fp32
// over fp32 terms (16-bit logits are widened exactly); results are rounded to 16 bits only where a gradient is stored in the logits' type.
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

__device__ __forceinline__ float wave_max(float v) {
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ unsigned long long wave_max64(unsigned long long v) {
  for (int o = 32; o; o >>= 1) {
    const unsigned lo = __shfl_xor((unsigned)v, o), hi = __shfl_xor((unsigned)(v >> 32), o);
    const unsigned long long w = ((unsigned long long)hi << 32) | lo;
    v = w > v ? w : v;
  }
  return v;
}

// ---- reductions over groups of G = 8 or 64 neighbouring lanes: data-parallel moves inside a row of 16, a shuffle across rows
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
constexpr int XOR1 = 0xB1, XOR2 = 0x4E, HALF_MIRROR = 0x141, MIRROR = 0x140;
template <int G, typename T, typename F>
__device__ __forceinline__ T group_reduce(T v, F f) {
  v = f(v, dpp<XOR1>(v));
  v = f(v, dpp<XOR2>(v));
  v = f(v, dpp<HALF_MIRROR>(v));
  if (G == 64) {
    v = f(v, dpp<MIRROR>(v));
    v = f(v, __shfl_xor(v, 16));
    v = f(v, __shfl_xor(v, 32));
  }
  return v;
}
template <int G> __device__ __forceinline__ float group_max(float v) { return group_reduce<G>(v, [](float a, float b) { return fmaxf(a, b); }); }
template <int G> __device__ __forceinline__ float group_sum(float v) { return group_reduce<G>(v, [](float a, float b) { return a + b; }); }
template <int G> __device__ __forceinline__ unsigned group_umax(unsigned v) { return group_reduce<G>(v, [](unsigned a, unsigned b) { return a > b ? a : b; }); }
template <int G> __device__ __forceinline__ unsigned group_umin(unsigned v) { return group_reduce<G>(v, [](unsigned a, unsigned b) { return a < b ? a : b; }); }
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

// i * s0 + j * s1 of row r = i * p + j; 64-bit divisions (~150 instructions) are kept out of the usual cases
__device__ __forceinline__ long long row_at(long long r, long long p, long long R, long long s0, long long s1) {
  if (p == R) return r * s1;
  if (R <= 0x7fffffff) {
    const unsigned i = (unsigned)r / (unsigned)p;
    return i * s0 + ((unsigned)r - i * (unsigned)p) * s1;
  }
  return (r / p) * s0 + (r % p) * s1;
}

struct Logits {
  const void* z;
  long long R, p, sn, sp, sc;
  int C;
  float invT, scale2;      // 1 / T, log2(e) / T
  __device__ __forceinline__ long long at(long long r) const { return row_at(r, p, R, sn, sp); }
};

struct LogprobOut {
  const long long* label;
  long long ignore;
  float *logprob, *entropy, *lse, *stats;      // [R] each, stats [2][R]: m, log S
  int* top_ids;
  float* top_lp;
  int k;
  long long tn, tp, tk;
};

__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// s, u taken about `from` become sums about `to` >= from (u's terms carry a factor d); an empty sum may come from -inf
__device__ __forceinline__ void rescale(float& s, float& u, float from, float to, float scale2) {
  const float d = (from - to) * scale2, f = exp2_(d);
  u = (u + s * fmaxf(d, -300.f)) * f;
  s = s * f;
}

__device__ __forceinline__ void void_row(const LogprobOut& o, long long r, long long R) {
  if (o.logprob) o.logprob[r] = 0.f;
  if (o.entropy) o.entropy[r] = 0.f;
  if (o.lse) o.lse[r] = 0.f;
  if (o.stats) o.stats[r] = o.stats[R + r] = 0.f;
}
// s = sum exp2(d), u = sum exp2(d) d about base, ls = log s; s = 0: every logit is -inf
__device__ __forceinline__ void finish_row(const LogprobOut& o, long long r, const Logits& a, float base, float s, float u, float ls,
                                           bool is_class, float zy) {
  if (o.stats) { o.stats[r] = base; o.stats[a.R + r] = ls; }
  if (o.lse) o.lse[r] = base * a.invT + ls;
  if (o.entropy) o.entropy[r] = s == 0.f ? 0.f : ls - u / s * LN2;
  if (o.logprob) o.logprob[r] = !is_class ? NAN : s == 0.f ? -INFINITY : (zy - base) * a.invT - ls;
}

// One wave per row, lanes along the classes: any strides.
template <typename E>
__global__ __launch_bounds__(256) void logprobs_fwd_kernel(const Logits a, const LogprobOut o) {
  const int lane = threadIdx.x & 63;
  const long long waves = (long long)gridDim.x * 4;
  for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.R; r += waves) {
    const E* z = (const E*)a.z + a.at(r);
    const long long y = o.label ? o.label[r] : 0;
    const long long ot = row_at(r, a.p, a.R, o.tn, o.tp);
    if (o.label && y == o.ignore) {            // a void row is not read
      if (lane == 0) void_row(o, r, a.R);
      if (lane < o.k) {
        o.top_ids[ot + lane * o.tk] = -1;
        o.top_lp[ot + lane * o.tk] = -INFINITY;
      }
      continue;
    }
    float m = -INFINITY;
    for (int c = lane; c < a.C; c += 64) m = fmaxf(m, load1(z + c * a.sc));
    m = wave_max(m);
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f, u = 0.f;
    for (int c = lane; c < a.C; c += 64) {
      const float d = (load1(z + c * a.sc) - base) * a.scale2, e = exp2_(d);
      s += e;
      u += e * fmaxf(d, -300.f);               // exp2(-300) = 0 in fp32; 0 * -inf would be NaN
    }
    s = wave_sum(s);
    u = wave_sum(u);
    const float ls = log2_(s) * LN2;
    const bool is_class = y >= 0 && y < a.C;
    if (lane == 0) finish_row(o, r, a, base, s, u, ls, is_class, o.logprob && is_class ? load1(z + y * a.sc) : 0.f);
    unsigned long long prev = ~0ull;
    for (int j = 0; j < o.k; ++j) {
      unsigned long long best = 0;
      for (int c = lane; c < a.C; c += 64) {
        const unsigned long long key = pair_key(load1(z + c * a.sc), c);
        if (key < prev && key > best) best = key;
      }
      prev = wave_max64(best);
      if (lane == 0) {
        const int c = (int)~(unsigned)prev;
        o.top_ids[ot + j * o.tk] = c;
        o.top_lp[ot + j * o.tk] = s == 0.f ? -INFINITY : (load1(z + c * a.sc) - base) * a.invT - ls;
      }
    }
  }
}

// Rows of at most 2048 contiguous classes: G lanes (8 up to 256 classes, 64 beyond) hold a row in registers, NV chunks of 16 bytes each,
// so it is read once and its maximum, sums and alternatives are reductions over registers and a few data-parallel moves.
// An alternative is one round over the G lanes' order keys: the largest key, the lowest class that has it, that class taken out.
template <typename E, int G, int NV>
__global__ __launch_bounds__(256) void logprobs_rows_kernel(const Logits a, const LogprobOut o) {
  constexpr int V = VEC<E>;
  const int l = threadIdx.x % G;
  const long long step = (long long)gridDim.x * (256 / G);
  for (long long r = (long long)blockIdx.x * (256 / G) + threadIdx.x / G; r < a.R; r += step) {
    const long long y = o.label ? o.label[r] : 0;
    const long long ot = o.k ? row_at(r, a.p, a.R, o.tn, o.tp) : 0;
    if (o.label && y == o.ignore) {
      if (l == 0) void_row(o, r, a.R);
      for (int j = l; j < o.k; j += G) {
        o.top_ids[ot + j * o.tk] = -1;
        o.top_lp[ot + j * o.tk] = -INFINITY;
      }
      continue;
    }
    const E* z = (const E*)a.z + a.at(r);
    float x[NV][V];
    int b[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) b[i] = load_chunk<G == 8 && NV == 1>(z, (i * G + l) * V, a.C, x[i]);
    float zy = 0.f;
    const bool is_class = y >= 0 && y < a.C;
    if (l == 0 && o.logprob && is_class) zy = load1(z + y);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) m = fmaxf(m, x[i][e]);
    m = group_max<G>(m);
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = (x[i][e] - base) * a.scale2, w = exp2_(d);
        s += w;
        u += w * fmaxf(d, -300.f);               // exp2(-300) = 0 in fp32; 0 * -inf would be NaN
      }
    s = group_sum<G>(s);
    u = group_sum<G>(u);
    const float ls = log2_(s) * LN2;
    if (l == 0) finish_row(o, r, a, base, s, u, ls, is_class, zy);
    if (o.k == 0) continue;
    unsigned key[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = b[i] + e;
        key[i][e] = c >= (i * G + l) * V && c < a.C ? order_key(x[i][e]) : 0u;
      }
    for (int j = 0; j < o.k; ++j) {
      unsigned best = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) best = max(best, key[i][e]);
      best = group_umax<G>(best);
      unsigned c = 0xffffffffu;
#pragma unroll
      for (int i = NV - 1; i >= 0; --i)
#pragma unroll
        for (int e = V - 1; e >= 0; --e) c = key[i][e] == best ? (unsigned)(b[i] + e) : c;
      c = group_umin<G>(c);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) key[i][e] = (unsigned)(b[i] + e) == c ? 0u : key[i][e];
      if (l == (j & (G - 1))) {
        o.top_ids[ot + j * o.tk] = (int)c;
        o.top_lp[ot + j * o.tk] = s == 0.f ? -INFINITY : (key_value(best) - base) * a.invT - ls;
      }
    }
  }
}

// Rows of more classes: a block of 256 lanes streams a slice of a row (the whole row where there are rows enough), 16 bytes a lane and
// load, and keeps each lane's running maximum and sums, rescaled once per four loads.  The k best come out of the same pass: the 8 lanes
// that read one 128-byte line note its maximum in LDS (for rows beyond 4096 lines, that of `join` lines of theirs).  Afterwards
//   tau = the k-th largest of the 256 lanes' maxima over their lines' maxima (a bound: at least k logits are >= tau),
//   the lines whose maximum is >= tau are read again (about k of them), their logits >= tau collected and ranked by counting.
// With many equal logits the lists could run over: then (and where a NaN hides from the maxima) the k best are taken in k passes.
constexpr int LINES = 4096, CAND = 512, CLINES = 256;

struct Stream {
  long long r0;                       // first row of this launch
  int nsplit, slice, join;            // slices of a row, classes of one (a multiple of VEC), lines whose maximum is kept together
  float* part;                        // [R][nsplit][3]: maximum, sum, sum of e d (nsplit > 1)
  unsigned long long* keys;           // [R][nsplit][k] (nsplit > 1)
};

template <typename E>
__global__ __launch_bounds__(256) void logprobs_stream_kernel(const Logits a, const LogprobOut o, const Stream t) {
  constexpr int V = VEC<E>;
  __shared__ unsigned line[LINES];
  __shared__ unsigned long long cand[CAND];
  __shared__ int clist[CLINES];
  __shared__ float red[3][4];
  __shared__ unsigned long long red64[4];
  __shared__ unsigned tau_s;
  __shared__ int nlines, ncand;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, g8 = tid >> 3;
  const int sp = (int)(blockIdx.x % (unsigned)t.nsplit);
  const long long r = t.r0 + blockIdx.x / (unsigned)t.nsplit;
  const long long y = o.label ? o.label[r] : 0;
  const long long ot = o.k ? row_at(r, a.p, a.R, o.tn, o.tp) : 0;
  if (o.label && y == o.ignore) {      // with several slices the joining kernel writes the row
    if (t.nsplit == 1) {
      if (tid == 0) void_row(o, r, a.R);
      if (tid < o.k) {
        o.top_ids[ot + tid * o.tk] = -1;
        o.top_lp[ot + tid * o.tk] = -INFINITY;
      }
    }
    return;
  }
  const E* z = (const E*)a.z + a.at(r);
  const int c0 = sp * t.slice, c1 = min(a.C, c0 + t.slice);
  const int iters = (c1 - c0 + 256 * V - 1) / (256 * V);
  float m = -INFINITY, s = 0.f, u = 0.f, lm = -INFINITY;
  constexpr int UN = 4;
  for (int it = 0; it < iters; it += UN) {
    float x[UN][V], cm[UN];
    if (c0 + (it + UN) * 256 * V <= c1) {
#pragma unroll
      for (int n = 0; n < UN; ++n) load_vec(z + c0 + ((it + n) * 256 + tid) * V, x[n]);
    } else {
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        const int c = c0 + ((it + n) * 256 + tid) * V;
        if (c < c1) {
          load_chunk(z, c, a.C, x[n]);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) x[n][e] = -INFINITY;
        }
      }
    }
    float nm = m;
#pragma unroll
    for (int n = 0; n < UN; ++n) {
      cm[n] = x[n][0];
#pragma unroll
      for (int e = 1; e < V; ++e) cm[n] = fmaxf(cm[n], x[n][e]);
      nm = fmaxf(nm, cm[n]);
    }
    if (o.k) {
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        lm = fmaxf(lm, group_max<8>(cm[n]));
        const int q = it + n;
        if (q < iters && ((q + 1) % t.join == 0 || q + 1 == iters)) {
          if ((tid & 7) == 0) line[(q / t.join) * 32 + g8] = order_key(lm);
          lm = -INFINITY;
        }
      }
    }
    const float base = nm == -INFINITY ? 0.f : nm;
    rescale(s, u, m, base, a.scale2);
    m = nm;
#pragma unroll
    for (int n = 0; n < UN; ++n)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = (x[n][e] - base) * a.scale2, w = exp2_(d);
        s += w;
        u += w * fmaxf(d, -300.f);
      }
  }
  // join the lanes, then the waves
  const float wm = group_max<64>(m);
  rescale(s, u, m, wm == -INFINITY ? 0.f : wm, a.scale2);
  s = group_sum<64>(s);
  u = group_sum<64>(u);
  if (lane == 0) { red[0][wv] = wm; red[1][wv] = s; red[2][wv] = u; }
  if (tid == 0) nlines = ncand = 0;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float base = m == -INFINITY ? 0.f : m;
  s = u = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float sw = red[1][w], uw = red[2][w];
    rescale(sw, uw, red[0][w], base, a.scale2);
    s += sw;
    u += uw;
  }
  const float ls = log2_(s) * LN2;
  if (tid == 0) {
    if (t.nsplit > 1) {
      float* q = t.part + (r * t.nsplit + sp) * 3;
      q[0] = m;
      q[1] = s;
      q[2] = u;
    } else {
      const bool is_class = y >= 0 && y < a.C;
      finish_row(o, r, a, base, s, u, ls, is_class, o.logprob && is_class ? load1(z + y) : 0.f);
    }
  }
  if (o.k == 0) return;

  const int nl = ((iters + t.join - 1) / t.join) * 32;
  unsigned best = 0;
  for (int i = tid; i < nl; i += 256) best = max(best, line[i]);
  cand[tid] = best;
  __syncthreads();
  if (wv == 0) {                       // the k-th largest of the 256 maxima, bit by bit
    unsigned q[4], tau = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = (unsigned)cand[i * 64 + lane];
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned c = tau | (1u << bit);
      int n = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) n += __popcll(__ballot(q[i] >= c));
      if (n >= o.k) tau = c;
    }
    if (lane == 0) tau_s = tau > 1u ? tau : 1u;
  }
  __syncthreads();
  const unsigned tau = tau_s;
  for (int i = tid; i < nl; i += 256)
    if (line[i] >= tau) {
      const int n = atomicAdd(&nlines, 1);
      if (n < CLINES) clist[n] = i;
    }
  __syncthreads();
  bool slow = nlines > CLINES || !(s < INFINITY);
  if (!slow) {
    for (int i = g8; i < nlines; i += 32) {
      const int li = clist[i];
      for (int j = 0; j < t.join; ++j) {
        const int c = c0 + (((li / 32) * t.join + j) * 256 + (li % 32) * 8 + (tid & 7)) * V;
        if (c >= c1) continue;
        float x[V];
        const int b = load_chunk(z, c, a.C, x);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (b + e >= c && b + e < a.C && order_key(x[e]) >= tau) {
            const int n = atomicAdd(&ncand, 1);
            if (n < CAND) cand[n] = pair_key(x[e], b + e);
          }
      }
    }
  }
  __syncthreads();
  slow = slow || ncand > CAND;
  int n = ncand;
  if (slow) {
    unsigned long long prev = ~0ull;
    n = 0;
    for (int j = 0; j < o.k; ++j) {
      unsigned long long top = 0;
      for (int c = c0 + tid; c < c1; c += 256) {
        const unsigned long long key = pair_key(load1(z + c), c);
        if (key < prev && key > top) top = key;
      }
      top = wave_max64(top);
      __syncthreads();
      if (lane == 0) red64[wv] = top;
      __syncthreads();
      for (int w = 0; w < 4; ++w) top = red64[w] > top ? red64[w] : top;
      prev = top;
      if (top) n = j + 1;
      if (tid == 0) cand[j] = top;
    }
    __syncthreads();
  }
  for (int i = tid; i < n; i += 256) {
    const unsigned long long key = cand[i];
    int rank = i;
    if (!slow) {
      rank = 0;
      for (int j = 0; j < n; ++j) rank += cand[j] > key;
    }
    if (rank < o.k) {
      if (t.nsplit > 1) {
        t.keys[(r * t.nsplit + sp) * o.k + rank] = key;
      } else {
        o.top_ids[ot + rank * o.tk] = (int)~(unsigned)key;
        o.top_lp[ot + rank * o.tk] = s == 0.f ? -INFINITY : (key_value((unsigned)(key >> 32)) - base) * a.invT - ls;
      }
    }
  }
  if (t.nsplit > 1)                    // a short last slice
    for (int i = n + tid; i < o.k; i += 256) t.keys[(r * t.nsplit + sp) * o.k + i] = 0;
}

// One wave joins the slices of a row, a lane to a slice: sums by the joint maximum, alternatives by merging the slices' falling lists.
template <typename E>
__global__ __launch_bounds__(64) void logprobs_join_kernel(const Logits a, const LogprobOut o, const Stream t) {
  const int lane = threadIdx.x;
  const long long r = t.r0 + blockIdx.x;
  const long long y = o.label ? o.label[r] : 0;
  const long long ot = o.k ? row_at(r, a.p, a.R, o.tn, o.tp) : 0;
  if (o.label && y == o.ignore) {
    if (lane == 0) void_row(o, r, a.R);
    if (lane < o.k) {
      o.top_ids[ot + lane * o.tk] = -1;
      o.top_lp[ot + lane * o.tk] = -INFINITY;
    }
    return;
  }
  const bool on = lane < t.nsplit;
  const float* q = t.part + (r * t.nsplit + (on ? lane : 0)) * 3;
  const float m1 = on ? q[0] : -INFINITY;
  float s = on ? q[1] : 0.f, u = on ? q[2] : 0.f;
  const unsigned long long* keys = t.keys + (r * t.nsplit + (on ? lane : 0)) * o.k;
  unsigned long long head = on && o.k ? keys[0] : 0;
  const float m = group_max<64>(m1);
  const float base = m == -INFINITY ? 0.f : m;
  rescale(s, u, m1, base, a.scale2);
  s = group_sum<64>(s);
  u = group_sum<64>(u);
  const float ls = log2_(s) * LN2;
  if (lane == 0) {
    const bool is_class = y >= 0 && y < a.C;
    finish_row(o, r, a, base, s, u, ls, is_class, o.logprob && is_class ? load1((const E*)a.z + a.at(r) + y) : 0.f);
  }
  int at = 0;
  for (int j = 0; j < o.k; ++j) {
    const unsigned long long top = wave_max64(head);
    if (head == top) {
      ++at;
      head = on && at < o.k ? keys[at] : 0;
    }
    if (lane == 0) {
      o.top_ids[ot + j * o.tk] = (int)~(unsigned)top;
      o.top_lp[ot + j * o.tk] = s == 0.f ? -INFINITY : (key_value((unsigned)(top >> 32)) - base) * a.invT - ls;
    }
  }
}

// ---- planes: PV neighbouring pixels to a lane, classes in a loop; every load of a wave is one contiguous piece of a class's plane
template <typename E, int PV>
__device__ __forceinline__ void load_px(const E* p, E (&q)[PV]) {
  if constexpr (PV * sizeof(E) == 4) {
    struct __attribute__((packed, aligned(alignof(E)))) W { unsigned v; };
    const unsigned w = reinterpret_cast<const W*>(p)->v;
    __builtin_memcpy(q, &w, 4);
  } else if constexpr (PV * sizeof(E) == 8) {
    struct __attribute__((packed, aligned(alignof(E)))) W { u32x2 v; };
    const u32x2 w = reinterpret_cast<const W*>(p)->v;
    __builtin_memcpy(q, &w, 8);
  } else {
#pragma unroll
    for (int v = 0; v < PV; ++v) q[v] = p[v];
  }
}
template <typename E, int PV>
__device__ __forceinline__ void store_px(E* p, const E (&q)[PV]) {
  if constexpr (PV * sizeof(E) == 4) {
    struct __attribute__((packed, aligned(alignof(E)))) W { unsigned v; };
    unsigned w;
    __builtin_memcpy(&w, q, 4);
    reinterpret_cast<W*>(p)->v = w;
  } else if constexpr (PV * sizeof(E) == 8) {
    struct __attribute__((packed, aligned(alignof(E)))) W { u32x2 v; };
    u32x2 w;
    __builtin_memcpy(&w, q, 8);
    reinterpret_cast<W*>(p)->v = w;
  } else {
#pragma unroll
    for (int v = 0; v < PV; ++v) p[v] = q[v];
  }
}
// Pixels of a tile of lanes: lane `pl` of tile `t` has PV pixels from `px` on, those from `p0` on are its own (an image's last lane is
// moved back so that it loads whole pieces).
template <int PV>
struct Px {
  long long px, p0, P;
  __device__ __forceinline__ Px(long long first, long long P_) : px(first < P_ - PV ? first : P_ - PV), p0(first), P(P_) {}
  __device__ __forceinline__ bool own(int v) const { return px + v >= p0; }
};

// Falling lists of the K best: order keys (fp32) with their classes beside them, or, for 16-bit logits, key and class in one word.
// Classes come in rising order, so a key equal to one in the list goes behind it.  The median of (upper neighbour, entry, new key) is
// the entry's new key.
__device__ __forceinline__ unsigned med3u(unsigned a, unsigned b, unsigned c) { return max(min(a, b), min(max(a, b), c)); }
template <typename E, int K>
struct Best {
  unsigned key[K > 0 ? K : 1];
  int id[K > 0 ? K : 1];
  __device__ __forceinline__ Best() {
#pragma unroll
    for (int j = 0; j < K; ++j) { key[j] = 0; id[j] = 0; }
  }
  __device__ __forceinline__ void add_key(unsigned k, int c) {
#pragma unroll
    for (int j = K - 1; j > 0; --j) {
      id[j] = k > key[j - 1] ? id[j - 1] : k > key[j] ? c : id[j];
      key[j] = med3u(key[j - 1], key[j], k);
    }
    id[0] = k > key[0] ? c : id[0];
    key[0] = max(key[0], k);
  }
  __device__ __forceinline__ void add(E z, int c) { add_key(order_key((float)z), c); }
  __device__ __forceinline__ float value(int j) const { return key_value(key[j]); }
  __device__ __forceinline__ int cls(int j) const { return id[j]; }
};
template <typename E, int K>
struct Best16 {
  unsigned key[K > 0 ? K : 1];
  __device__ __forceinline__ Best16() {
#pragma unroll
    for (int j = 0; j < K; ++j) key[j] = 0;
  }
  __device__ __forceinline__ void add_key(unsigned k, int) {
#pragma unroll
    for (int j = K - 1; j > 0; --j) key[j] = med3u(key[j - 1], key[j], k);
    key[0] = max(key[0], k);
  }
  __device__ __forceinline__ void add(E z, int c) {
    constexpr unsigned INF16 = sizeof(E) == 2 && __is_same(E, __bf16) ? 0x7f80u : 0x7c00u;
    unsigned short h;
    __builtin_memcpy(&h, &z, 2);
    unsigned u = h == 0x8000u ? 0u : h;
    u = (u & 0x7fffu) > INF16 ? 0xffffu : u ^ (u & 0x8000u ? 0xffffu : 0x8000u);
    add_key(u << 16 | (0xffffu - (unsigned)c), c);
  }
  __device__ __forceinline__ float value(int j) const {
    const unsigned k = key[j] >> 16;
    const unsigned short h = (unsigned short)(k & 0x8000u ? k ^ 0x8000u : k ^ 0xffffu);
    E z;
    __builtin_memcpy(&z, &h, 2);
    return (float)z;
  }
  __device__ __forceinline__ int cls(int j) const { return 0xffff - (int)(key[j] & 0xffffu); }
};
template <typename E, int K> struct BestOf { using type = Best16<E, K>; };
template <int K> struct BestOf<float, K> { using type = Best<float, K>; };

constexpr int PLANE_K = 32, PLANE_CLASSES = 65536;

// SPLIT = 4: a block's four waves share 64 * PV pixels and take a quarter of the classes each (images too small to fill the device).
template <typename E, int PV, int K, int SPLIT>
__global__ __launch_bounds__(256) void logprobs_planes_kernel(const Logits a, const LogprobOut o, const long long i0, const int tiles) {
  using B = typename BestOf<E, K>::type;
  constexpr int LANES = 256 / SPLIT, UN = 8;
  __shared__ float red[SPLIT > 1 ? SPLIT - 1 : 1][3][PV][SPLIT > 1 ? 64 : 1];
  __shared__ unsigned lists[SPLIT > 1 ? SPLIT - 1 : 1][K > 0 ? K : 1][PV][SPLIT > 1 ? 64 : 1];
  __shared__ int ids[SPLIT > 1 && sizeof(B) > 4 * (K > 0 ? K : 1) ? SPLIT - 1 : 1][K > 0 ? K : 1][PV][SPLIT > 1 ? 64 : 1];
  const int wv = SPLIT > 1 ? threadIdx.x >> 6 : 0, pl = threadIdx.x & (LANES - 1);
  const long long i = i0 + blockIdx.x / (unsigned)tiles;
  const long long first = (long long)(blockIdx.x % (unsigned)tiles) * (LANES * PV) + pl * PV;
  const Px<PV> px(first, a.p);
  const E* z = (const E*)a.z + i * a.sn + px.px;
  const int per = (a.C + SPLIT - 1) / SPLIT, c0 = wv * per, c1 = min(a.C, c0 + per);
  float m[PV], s[PV], u[PV];
  B best[PV];
#pragma unroll
  for (int v = 0; v < PV; ++v) { m[v] = -INFINITY; s[v] = u[v] = 0.f; }
  for (int c = c0; c < c1; c += UN) {
    E q[UN][PV];
    float x[UN][PV];
#pragma unroll
    for (int n = 0; n < UN; ++n) load_px<E, PV>(z + min(c + n, c1 - 1) * a.sc, q[n]);
#pragma unroll
    for (int n = 0; n < UN; ++n)
#pragma unroll
      for (int v = 0; v < PV; ++v) x[n][v] = c + n < c1 ? (float)q[n][v] : -INFINITY;
#pragma unroll
    for (int v = 0; v < PV; ++v) {
      float nm = m[v];
#pragma unroll
      for (int n = 0; n < UN; ++n) nm = fmaxf(nm, x[n][v]);
      const float base = nm == -INFINITY ? 0.f : nm;
      rescale(s[v], u[v], m[v], base, a.scale2);
      m[v] = nm;
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        const float d = (x[n][v] - base) * a.scale2, w = exp2_(d);
        s[v] += w;
        u[v] += w * fmaxf(d, -300.f);
      }
    }
    if (K > 0) {
#pragma unroll
      for (int n = 0; n < UN; ++n)
        if (c + n < c1) {
#pragma unroll
          for (int v = 0; v < PV; ++v) best[v].add(q[n][v], c + n);
        }
    }
  }
  if constexpr (SPLIT > 1) {
    if (wv > 0) {
#pragma unroll
      for (int v = 0; v < PV; ++v) {
        red[wv - 1][0][v][pl] = m[v];
        red[wv - 1][1][v][pl] = s[v];
        red[wv - 1][2][v][pl] = u[v];
#pragma unroll
        for (int j = 0; j < K; ++j) {
          lists[wv - 1][j][v][pl] = best[v].key[j];
          if constexpr (sizeof(B) > 4 * (K > 0 ? K : 1)) ids[wv - 1][j][v][pl] = best[v].cls(j);
        }
      }
    }
    __syncthreads();
    if (wv > 0) return;
    for (int w = 0; w < SPLIT - 1; ++w) {
#pragma unroll
      for (int v = 0; v < PV; ++v) {
        const float om = red[w][0][v][pl], nm = fmaxf(m[v], om), base = nm == -INFINITY ? 0.f : nm;
        float os = red[w][1][v][pl], ou = red[w][2][v][pl];
        rescale(s[v], u[v], m[v], base, a.scale2);
        rescale(os, ou, om, base, a.scale2);
        s[v] += os;
        u[v] += ou;
        m[v] = nm;
        if (K > 0) {
          for (int j = 0; j < K; ++j) {        // the other waves' classes are higher: equal keys stay behind
            const unsigned k = lists[w][j][v][pl];
            int id = 0;
            if constexpr (sizeof(B) > 4 * (K > 0 ? K : 1)) id = ids[w][j][v][pl];
            best[v].add_key(k, id);
          }
        }
      }
    }
  }
  if (first >= a.p) return;
#pragma unroll
  for (int v = 0; v < PV; ++v) {
    if (!px.own(v)) continue;
    const long long r = i * a.p + px.px + v;
    const long long y = o.label ? o.label[r] : 0;
    const bool empty = o.label && y == o.ignore, is_class = y >= 0 && y < a.C;
    const float base = m[v] == -INFINITY ? 0.f : m[v], ls = log2_(s[v]) * LN2;
    if (empty) void_row(o, r, a.R);
    else finish_row(o, r, a, base, s[v], u[v], ls, is_class, o.logprob && is_class ? load1(z + y * a.sc + v) : 0.f);
    const long long ot = i * o.tn + (px.px + v) * o.tp;
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (j < o.k) {
        o.top_ids[ot + j * o.tk] = empty ? -1 : best[v].cls(j);
        o.top_lp[ot + j * o.tk] = empty || s[v] == 0.f ? -INFINITY : (best[v].value(j) - base) * a.invT - ls;
      }
  }
}

struct LogprobGrad {
  const long long* label;
  long long ignore;
  const float *stats, *entropy, *g_logprob, *g_entropy, *g_lse;
  void* dz;
  long long dn, dp, dc;
  int accumulate;
};

// dz_c = p_c (A + B log p_c) + [c = y] G  with  G = g_logprob / T,  B = -g_entropy / T,  A = (g_lse - g_logprob - g_entropy H) / T
struct RowGrad {
  float m, ls, A, B, G;
  long long y;
  bool dead;                 // void, or nothing but -inf: no gradient
  __device__ __forceinline__ RowGrad(const Logits& a, const LogprobGrad& g, long long r) {
    y = g.label ? g.label[r] : -1;
    m = g.stats[r];
    ls = g.stats[a.R + r];
    dead = (g.label && y == g.ignore) || ls == -INFINITY;
    G = g.g_logprob && y >= 0 && y < a.C ? g.g_logprob[r] * a.invT : 0.f;
    B = g.g_entropy ? -g.g_entropy[r] * a.invT : 0.f;
    A = (g.g_lse ? g.g_lse[r] * a.invT : 0.f) - G + (g.g_entropy ? B * g.entropy[r] : 0.f);
  }
  __device__ __forceinline__ float operator()(const Logits& a, float z, int c) const {
    const float lp = (z - m) * a.invT - ls;
    float v = exp2_(lp * LOG2E) * (A + B * fmaxf(lp, -200.f));      // exp(-200) = 0 in fp32; 0 * -inf would be NaN
    if (c == y) v += G;
    return dead ? 0.f : v;
  }
};

// Contiguous classes: G lanes to a row (8, 64) or a block to a segment of SEG chunks a lane; one read, one write, no reductions.
template <typename E, int G>
__global__ __launch_bounds__(256) void logprobs_bwd_rows_kernel(const Logits a, const LogprobGrad g, const int segs) {
  constexpr int V = VEC<E>, SEG = 4;
  const int l = threadIdx.x % G;
  const long long step = (long long)gridDim.x * (256 / G), items = a.R * segs;
  for (long long it = (long long)blockIdx.x * (256 / G) + threadIdx.x / G; it < items; it += step) {
    long long r = it;
    int seg = 0;
    if (segs > 1) {
      r = items <= 0x7fffffff ? (unsigned)it / (unsigned)segs : it / segs;
      seg = (int)(it - r * segs);
    }
    const RowGrad f(a, g, r);
    const E* z = (const E*)a.z + a.at(r);
    E* dz = (E*)g.dz + row_at(r, a.p, a.R, g.dn, g.dp);
    for (int q = 0; q < (G == 256 ? SEG : (a.C + G * V - 1) / (G * V)); ++q) {
      const int c = (G == 256 ? seg * (SEG * G * V) : 0) + (q * G + l) * V;
      if (c >= a.C) break;
      float x[V], old[V];
      const int b = load_chunk<G == 8>(z, c, a.C, x);
      if (g.accumulate) load_chunk<G == 8>((const E*)dz, c, a.C, old);
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = f(a, x[e], b + e) + (g.accumulate ? old[e] : 0.f);
      store_chunk(dz, c, b, a.C, x);
    }
  }
}

// Planes: PV pixels and a slice of the classes to a lane.
template <typename E, int PV>
__global__ __launch_bounds__(256) void logprobs_bwd_planes_kernel(const Logits a, const LogprobGrad g, const long long i0, const int tiles,
                                                                  const int slice) {
  constexpr int UN = 4;
  const long long i = i0 + blockIdx.x / (unsigned)tiles;
  const long long first = (long long)(blockIdx.x % (unsigned)tiles) * (256 * PV) + threadIdx.x * PV;
  if (first >= a.p) return;
  const Px<PV> px(first, a.p);
  const E* z = (const E*)a.z + i * a.sn + px.px;
  E* dz = (E*)g.dz + i * g.dn + px.px;
  const RowGrad f0(a, g, i * a.p + px.px), f1(a, g, i * a.p + px.px + PV - 1);
  const int c0 = blockIdx.y * slice, c1 = min(a.C, c0 + slice);
  for (int c = c0; c < c1; c += UN) {
    E q[UN][PV], old[UN][PV];
#pragma unroll
    for (int n = 0; n < UN; ++n) {
      load_px<E, PV>(z + min(c + n, c1 - 1) * a.sc, q[n]);
      if (g.accumulate) load_px<E, PV>(dz + min(c + n, c1 - 1) * g.dc, old[n]);
    }
#pragma unroll
    for (int n = 0; n < UN; ++n) {
      if (c + n >= c1) break;
#pragma unroll
      for (int v = 0; v < PV; ++v) q[n][v] = (E)((v ? f1 : f0)(a, (float)q[n][v], c + n) + (g.accumulate ? (float)old[n][v] : 0.f));
      if (px.own(0)) {
        store_px<E, PV>(dz + (c + n) * g.dc, q[n]);
      } else {
#pragma unroll
        for (int v = 1; v < PV; ++v)
          if (px.own(v)) store1(dz + (c + n) * g.dc + v, (float)q[n][v]);
      }
    }
  }
}

struct Teacher {
  const void* ids;
  const void* top;
  int ids64, top_type, k, tail;
  long long in, ip, ik, vn, vp, vk;
  const float* weight;
  // entry j of the row whose entries start at io / vo
  __device__ __forceinline__ long long id(long long io, int j) const {
    const long long o = io + j * ik;
    return ids64 ? ((const long long*)ids)[o] : ((const int*)ids)[o];
  }
  __device__ __forceinline__ float value(long long vo, int j) const {
    const long long o = vo + j * vk;
    return top_type == SEMSEG_TYPE_F32 ? ((const float*)top)[o]
         : top_type == SEMSEG_TYPE_BF16 ? (float)((const __bf16*)top)[o] : (float)((const _Float16*)top)[o];
  }
};

// The teacher's distribution of one row over TG lanes, entry j = i * TG + lane in element i of a lane (NE of them): class (-1 where the
// entry is absent), q, log q.
template <int TG, int NE>
struct RowTeacher {
  int id[NE];
  float q[NE], lq[NE], qsum, qrest;
  bool any, bad;             // any entry present; an id that is no class
  __device__ __forceinline__ RowTeacher(const Teacher& t, const Logits& a, long long r, int l) {
    const long long io = row_at(r, a.p, a.R, t.in, t.ip), vo = row_at(r, a.p, a.R, t.vn, t.vp);
    unsigned flags = 0;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int j = i * TG + l;
      id[i] = -1;
      lq[i] = -INFINITY;
      if (j < t.k) {
        const long long c = t.id(io, j);
        if (c >= a.C) flags |= 2u;
        if (c >= 0 && c < a.C) {
          flags |= 1u;
          id[i] = (int)c;
          lq[i] = t.value(vo, j);
          m = fmaxf(m, lq[i]);
        }
      }
    }
    flags = group_reduce<TG>(flags, [](unsigned x, unsigned y) { return x | y; });
    any = flags & 1u;
    bad = flags & 2u;
    float s = 0.f;
    if (t.tail) {
#pragma unroll
      for (int i = 0; i < NE; ++i) s += q[i] = exp2_(lq[i] * LOG2E);
      qsum = group_sum<TG>(s);
      qrest = fmaxf(1.f - qsum, 0.f);
    } else {
      m = group_max<TG>(m);
      if (m == -INFINITY) m = 0.f;
#pragma unroll
      for (int i = 0; i < NE; ++i) s += q[i] = exp2_((lq[i] - m) * a.scale2);
      s = group_sum<TG>(s);
      const float ls = log2_(s) * LN2, inv = s == 0.f ? 0.f : 1.f / s;
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        lq[i] = (lq[i] - m) * a.invT - ls;
        q[i] *= inv;
      }
      qsum = s == 0.f ? 0.f : 1.f;
      qrest = 0.f;
    }
  }
  // sum of q over all entries of element i's class; what the other lanes hold comes by shuffles
  __device__ __forceinline__ float of_class(int i, int k, int c) const {
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < NE; ++n)
      if (n * TG < k)
        for (int src = 0; src < TG; ++src) {
          const int o = __shfl(id[n], src, TG);
          const float v = __shfl(q[n], src, TG);
          sum += o == c ? v : 0.f;
          if (n * TG + src + 1 >= k) break;
        }
    return sum;
  }
};

struct DistillOut {
  float *rows, *stats;       // [R] loss per row (or null), stats [3][R]: m, log S, log p_rest (+inf: no class outside the entries)
  double* part;              // [2][blocks]: weighted loss, weights (or null)
  float T2;
};
struct DistillGrad {
  const float* stats;
  const double* acc;         // acc[1]: sum of weights (mean), null: `den` is
  double den;
  const float* g;            // one gradient (or one per row), null: 1
  float gmul, T;
  int mean, per_row, accumulate;
  void* dz;
  long long dn, dp, dc;
  __device__ __forceinline__ float coef(long long r, float w) const {
    const float c = gmul * T * w * (g ? g[per_row ? r : 0] : 1.f);
    if (!mean) return c;
    const double d = acc ? acc[1] : den;
    return d == 0.0 ? 0.f : (float)((double)c / d);
  }
};

// A block's partial sums, added over its lanes in a fixed order
template <int THREADS>
__device__ __forceinline__ void block_part(double* part, double loss, double wsum) {
  for (int o = 32; o; o >>= 1) { loss += shfl_xor_f64(loss, o); wsum += shfl_xor_f64(wsum, o); }
  __shared__ double sl[THREADS / 64], sw[THREADS / 64];
  if ((threadIdx.x & 63) == 0) { sl[threadIdx.x >> 6] = loss; sw[threadIdx.x >> 6] = wsum; }
  __syncthreads();
  if (threadIdx.x == 0 && part) {
    loss = wsum = 0.0;
    for (int i = 0; i < THREADS / 64; ++i) { loss += sl[i]; wsum += sw[i]; }
    part[blockIdx.x] = loss;
    part[gridDim.x + blockIdx.x] = wsum;
  }
}
__global__ __launch_bounds__(256) void weight_sum_kernel(const float* w, long long R, double* part) {
  double s = 0.0;
  for (long long r = (long long)blockIdx.x * 256 + threadIdx.x; r < R; r += (long long)gridDim.x * 256) s += (double)w[r];
  block_part<256>(part, 0.0, s);
}
// acc = {sum of weighted losses, sum of weights} from the blocks' partials, added in a fixed order; loss = T^2 acc0 [/ acc1].
// loss null: the weights alone.
__global__ __launch_bounds__(1024) void distill_finish_kernel(const double* part, int blocks, double* acc, float* loss, float T2, int mean) {
  double l = 0.0, w = 0.0;
  for (int i = threadIdx.x; i < blocks; i += 1024) { l += part[i]; w += part[blocks + i]; }
  for (int o = 32; o; o >>= 1) { l += shfl_xor_f64(l, o); w += shfl_xor_f64(w, o); }
  __shared__ double sl[16], sw[16];
  if ((threadIdx.x & 63) == 0) { sl[threadIdx.x >> 6] = l; sw[threadIdx.x >> 6] = w; }
  __syncthreads();
  if (threadIdx.x == 0) {
    l = w = 0.0;
    for (int i = 0; i < 16; ++i) { l += sl[i]; w += sw[i]; }
    acc[1] = w;
    if (!loss) return;
    acc[0] = l;
    loss[0] = (float)((double)T2 * (mean ? l / w : l));
  }
}

// dz_c = coef (p_c Q - sum_{j: id_j = c} q_j) for the teacher's classes, coef p_c Q for the others; with a tail Q counts it, and the
// others are coef exp(log p_c - log p_rest) (Q p_rest - q_rest): one exponential, and no overflow where p_rest is tiny.
//
// The teacher's classes are few: a row is first written as if there were none, then the lanes that hold entries write theirs (from the
// logits that they gather), behind the first stores in the same wave (or behind a barrier of the block).

// Rows of at most 2048 contiguous classes: G lanes hold a row in registers.  GRAD: loss and gradient from one read of the logits.
template <typename E, int G, int NV, int NE, bool GRAD>
__global__ __launch_bounds__(256) void distill_rows_kernel(const Logits a, const Teacher t, const DistillOut o, const DistillGrad g) {
  constexpr int V = VEC<E>;
  constexpr bool SHORT = G == 8 && NV == 1;
  const int l = threadIdx.x % G;
  const long long step = (long long)gridDim.x * (256 / G);
  double loss = 0.0, wsum = 0.0;
  for (long long r = (long long)blockIdx.x * (256 / G) + threadIdx.x / G; r < a.R; r += step) {
    const float w = t.weight ? t.weight[r] : 1.f;
    E* dz = GRAD ? (E*)g.dz + row_at(r, a.p, a.R, g.dn, g.dp) : nullptr;
    bool dead = w == 0.f;
    if (!dead) {
      const E* z = (const E*)a.z + a.at(r);
      float x[NV][V];
      int b[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) b[i] = load_chunk<SHORT>(z, (i * G + l) * V, a.C, x[i]);
      const RowTeacher<G, NE> q(t, a, r, l);
      float zj[NE];
#pragma unroll
      for (int i = 0; i < NE; ++i) zj[i] = q.id[i] >= 0 ? load1(z + q.id[i]) : -INFINITY;
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) m = fmaxf(m, x[i][e]);
      m = group_max<G>(m);
      const float base = m == -INFINITY ? 0.f : m;
      float s = 0.f, st = 0.f;
      unsigned in = 0;             // of the lane's NV * V logits: those of the teacher's classes
      if (t.tail) {
#pragma unroll
        for (int n = 0; n < NE; ++n)
          if (n * G < t.k)
            for (int src = 0; src < G && n * G + src < t.k; ++src) {
              const int c = __shfl(q.id[n], src, G);
              if (c >= 0 && (c / V) % G == l) {
                const int ch = c / V, first = SHORT && a.C < V ? ch * V : min(ch * V, a.C - V);
                in |= 1u << (ch / G * V + c - first);
              }
            }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float p = exp2_((x[i][e] - base) * a.scale2);
          s += p;
          if (t.tail) st += in >> (i * V + e) & 1u ? 0.f : p;
        }
      s = group_sum<G>(s);
      const float ls = log2_(s) * LN2;
      float lpt = 0.f, rbase = base, rsum = s;
      bool rest = false;
      if (t.tail) {
        st = group_sum<G>(st);
        rest = true;
        if (st < 1e-20f) {         // the rest is far below the row's maximum: about its own
          float mt = -INFINITY;
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) mt = fmaxf(mt, in >> (i * V + e) & 1u ? -INFINITY : x[i][e]);
          mt = group_max<G>(mt);
          rest = mt != -INFINITY;
          rbase = rest ? mt : 0.f;
          st = 0.f;
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) st += in >> (i * V + e) & 1u ? 0.f : exp2_((x[i][e] - rbase) * a.scale2);
          st = group_sum<G>(st);
        }
        if (rest) {
          lpt = (rbase - base) * a.invT + log2_(st) * LN2 - ls;
          rsum = st;
        } else {
          rbase = base;
        }
      }
      float kl = 0.f;
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        const float lp = s == 0.f ? -INFINITY : (zj[i] - base) * a.invT - ls;
        kl += q.q[i] == 0.f ? 0.f : q.q[i] * (q.lq[i] - lp);
        zj[i] = lp;
      }
      kl = group_sum<G>(kl);
      if (rest && q.qrest > 0.f) kl += q.qrest * (log2_(q.qrest) * LN2 - lpt);
      if (!q.any) kl = 0.f;
      if (q.bad) kl = NAN;
      if (l == 0) {
        if (!GRAD) {
          o.stats[r] = base;
          o.stats[a.R + r] = ls;
          o.stats[2 * a.R + r] = t.tail && !rest ? INFINITY : lpt;
        }
        if (o.rows) o.rows[r] = o.T2 * w * kl;
        loss += (double)w * (double)kl;
        wsum += (double)w;
      }
      if (GRAD) {
        dead = q.bad || !q.any || s == 0.f;
        if (!dead) {
          const float coef = g.coef(r, w), Q = rest ? q.qsum + q.qrest : q.qsum;
          const float f = coef * (rest ? Q * exp2_(lpt * LOG2E) - q.qrest : Q) / rsum;
          float fix[NE];
#pragma unroll
          for (int i = 0; i < NE; ++i) {
            fix[i] = 0.f;
            if (i * G < t.k) {
              fix[i] = coef * (Q * exp2_(zj[i] * LOG2E) - q.of_class(i, t.k, q.id[i]));
              if (g.accumulate && q.id[i] >= 0) fix[i] += load1(dz + q.id[i]);
            }
          }
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int c = (i * G + l) * V;
            if (c < a.C) {
              float old[V];
              if (g.accumulate) load_chunk<SHORT>((const E*)dz, c, a.C, old);
#pragma unroll
              for (int e = 0; e < V; ++e) x[i][e] = f * exp2_((x[i][e] - rbase) * a.scale2) + (g.accumulate ? old[e] : 0.f);
              store_chunk(dz, c, b[i], a.C, x[i]);
            }
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int i = 0; i < NE; ++i)
            if (q.id[i] >= 0) store1(dz + q.id[i], fix[i]);
        }
      }
    } else if (l == 0) {
      if (!GRAD) o.stats[r] = o.stats[a.R + r] = o.stats[2 * a.R + r] = 0.f;
      if (o.rows) o.rows[r] = 0.f;
    }
    if (GRAD && dead && !g.accumulate) zero_row<G>(dz, l, a.C);
  }
  block_part<256>(o.part, loss, wsum);
}

// Longer rows: every block streams a slice and leaves its maximum and sum (with a tail: of the classes outside the entries, found by a
// bitmap of the 16-byte chunks that hold one) ...
constexpr int MAP_WORDS = 2048;
struct DStream {
  long long r0;
  int nsplit, slice;
  float* part;               // [R][nsplit][2]
};
template <typename E>
__global__ __launch_bounds__(256) void distill_stream_kernel(const Logits a, const Teacher t, const DStream d) {
  constexpr int V = VEC<E>, UN = 4;
  __shared__ unsigned map[MAP_WORDS];
  __shared__ int ids[MAXK];
  __shared__ float red[2][4];
  const int tid = threadIdx.x;
  const int sp = (int)(blockIdx.x % (unsigned)d.nsplit);
  const long long r = d.r0 + blockIdx.x / (unsigned)d.nsplit;
  if (t.weight && t.weight[r] == 0.f) return;
  const E* z = (const E*)a.z + a.at(r);
  if (t.tail) {
    const long long io = row_at(r, a.p, a.R, t.in, t.ip);
    for (int j = tid; j < t.k; j += 256) {
      const long long c = t.id(io, j);
      ids[j] = c >= 0 && c < a.C ? (int)c : -1;
    }
  }
  const int first = sp * d.slice, last = min(a.C, first + d.slice);
  float m = -INFINITY, s = 0.f, unused = 0.f;
  for (int c0 = first; c0 < last; c0 += MAP_WORDS * 32 * V) {      // one turn up to 262144 classes
    const int c1 = min(last, c0 + MAP_WORDS * 32 * V);
    const int iters = (c1 - c0 + 256 * V - 1) / (256 * V);
    if (t.tail) {
      __syncthreads();
      for (int i = tid; i < min(MAP_WORDS, iters * 8); i += 256) map[i] = 0;
      __syncthreads();
      for (int j = tid; j < t.k; j += 256)
        if (ids[j] >= c0 && ids[j] < c1) atomicOr(&map[(ids[j] - c0) / V >> 5], 1u << ((ids[j] - c0) / V & 31));
      __syncthreads();
    }
    for (int it = 0; it < iters; it += UN) {
      float x[UN][V];
      if (c0 + (it + UN) * 256 * V <= c1) {
#pragma unroll
        for (int n = 0; n < UN; ++n) load_vec(z + c0 + ((it + n) * 256 + tid) * V, x[n]);
      } else {
#pragma unroll
        for (int n = 0; n < UN; ++n) {
          const int c = c0 + ((it + n) * 256 + tid) * V;
          if (c < c1) {
            load_chunk(z, c, a.C, x[n]);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[n][e] = -INFINITY;
          }
        }
      }
      if (t.tail) {
#pragma unroll
        for (int n = 0; n < UN; ++n) {
          const int ch = (it + n) * 256 + tid, c = c0 + ch * V;
          if (c < c1 && (map[ch >> 5] >> (ch & 31) & 1u)) {
            const int b = min(c, a.C - V);
            for (int j = 0; j < t.k; ++j)
#pragma unroll
              for (int e = 0; e < V; ++e) x[n][e] = ids[j] == b + e ? -INFINITY : x[n][e];
          }
        }
      }
      float nm = m;
#pragma unroll
      for (int n = 0; n < UN; ++n)
#pragma unroll
        for (int e = 0; e < V; ++e) nm = fmaxf(nm, x[n][e]);
      const float base = nm == -INFINITY ? 0.f : nm;
      s *= exp2_((m - base) * a.scale2);
      m = nm;
#pragma unroll
      for (int n = 0; n < UN; ++n)
#pragma unroll
        for (int e = 0; e < V; ++e) s += exp2_((x[n][e] - base) * a.scale2);
    }
  }
  const float wm = group_max<64>(m);
  rescale(s, unused, m, wm == -INFINITY ? 0.f : wm, a.scale2);
  s = group_sum<64>(s);
  if ((tid & 63) == 0) { red[0][tid >> 6] = wm; red[1][tid >> 6] = s; }
  __syncthreads();
  if (tid == 0) {
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float base = m == -INFINITY ? 0.f : m;
    s = 0.f;
    for (int w = 0; w < 4; ++w) s += red[1][w] * exp2_((red[0][w] - base) * a.scale2);
    float* q = d.part + (r * d.nsplit + sp) * 2;
    q[0] = m;
    q[1] = s;
  }
}
// ... and one wave a row joins them, adds the entries' logits and takes the loss.
template <typename E>
__global__ __launch_bounds__(256) void distill_join_kernel(const Logits a, const Teacher t, const DistillOut o, const DStream d) {
  const int lane = threadIdx.x & 63;
  double loss = 0.0, wsum = 0.0;
  for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.R; r += (long long)gridDim.x * 4) {
    const float w = t.weight ? t.weight[r] : 1.f;
    if (w == 0.f) {
      if (lane == 0) {
        o.stats[r] = o.stats[a.R + r] = o.stats[2 * a.R + r] = 0.f;
        if (o.rows) o.rows[r] = 0.f;
      }
      continue;
    }
    const E* z = (const E*)a.z + a.at(r);
    const RowTeacher<64, 1> q(t, a, r, lane);
    const float zj = q.id[0] >= 0 ? load1(z + q.id[0]) : -INFINITY;
    const float* part = d.part + (r * d.nsplit + (lane < d.nsplit ? lane : 0)) * 2;
    const float m1 = lane < d.nsplit ? part[0] : -INFINITY;
    float s = lane < d.nsplit ? part[1] : 0.f, st = 0.f;
    const float mt = group_max<64>(m1);
    float m = mt;
    bool once = q.id[0] >= 0;                  // an entry's class counts once
    if (t.tail) {
      m = fmaxf(mt, group_max<64>(zj));
      for (int j = 0; j < t.k; ++j) once = once && !(__shfl(q.id[0], j) == q.id[0] && j < lane);
      const float tb = mt == -INFINITY ? 0.f : mt;
      st = group_sum<64>(s * exp2_((m1 - tb) * a.scale2));
    }
    const float base = m == -INFINITY ? 0.f : m;
    s *= exp2_((m1 - base) * a.scale2);
    if (t.tail && once) s += exp2_((zj - base) * a.scale2);
    s = group_sum<64>(s);
    const float ls = log2_(s) * LN2;
    const float lp = s == 0.f ? -INFINITY : (zj - base) * a.invT - ls;
    float kl = group_sum<64>(q.q[0] == 0.f ? 0.f : q.q[0] * (q.lq[0] - lp));
    float lpt = 0.f;
    const bool rest = t.tail && mt != -INFINITY;
    if (rest) {
      lpt = (mt - base) * a.invT + log2_(st) * LN2 - ls;
      if (q.qrest > 0.f) kl += q.qrest * (log2_(q.qrest) * LN2 - lpt);
    }
    if (!q.any) kl = 0.f;
    if (q.bad) kl = NAN;
    if (lane == 0) {
      o.stats[r] = base;
      o.stats[a.R + r] = ls;
      o.stats[2 * a.R + r] = t.tail && !rest ? INFINITY : lpt;
      if (o.rows) o.rows[r] = o.T2 * w * kl;
      loss += (double)w * (double)kl;
      wsum += (double)w;
    }
  }
  block_part<256>(o.part, loss, wsum);
}

// The gradient from the forward call's statistics: G lanes to a row (8, 64), or a block to a segment of SEG chunks a lane.
template <typename E, int G>
__global__ __launch_bounds__(256) void distill_bwd_rows_kernel(const Logits a, const Teacher t, const DistillGrad g, const int segs) {
  constexpr int V = VEC<E>, SEG = 4, TG = G < 64 ? G : 64, NE = MAXK / TG;
  const int l = threadIdx.x % G;
  const long long step = (long long)gridDim.x * (256 / G), items = a.R * segs;
  for (long long it = (long long)blockIdx.x * (256 / G) + threadIdx.x / G; it < items; it += step) {
    long long r = it;
    int seg = 0;
    if (segs > 1) {
      r = items <= 0x7fffffff ? (unsigned)it / (unsigned)segs : it / segs;
      seg = (int)(it - r * segs);
    }
    const float w = t.weight ? t.weight[r] : 1.f, base = g.stats[r], ls = g.stats[a.R + r], lpt = g.stats[2 * a.R + r];
    E* dz = (E*)g.dz + row_at(r, a.p, a.R, g.dn, g.dp);
    const int c0 = G == 256 ? seg * (SEG * G * V) : 0, c1 = G == 256 ? min(a.C, c0 + SEG * G * V) : a.C;
    const RowTeacher<TG, NE> q(t, a, r, threadIdx.x % TG);
    const bool dead = w == 0.f || q.bad || !q.any || ls == -INFINITY;
    const E* z = (const E*)a.z + a.at(r);
    const bool rest = t.tail && lpt != INFINITY;
    const float coef = g.coef(r, w), Q = rest ? q.qsum + q.qrest : q.qsum;
    const float off = rest ? ls + lpt : ls, f = coef * (rest ? Q * exp2_(lpt * LOG2E) - q.qrest : Q);
    float fix[NE];
    bool mine[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      fix[i] = 0.f;
      mine[i] = !dead && q.id[i] >= c0 && q.id[i] < c1 && (G < 256 || threadIdx.x < 64);
      if (i * TG < t.k && __any(mine[i])) {      // most segments of a long row hold no entry
        const float sum = q.of_class(i, t.k, q.id[i]);
        if (mine[i]) {
          fix[i] = coef * (Q * exp2_(((load1(z + q.id[i]) - base) * a.invT - ls) * LOG2E) - sum);
          if (g.accumulate) fix[i] += load1(dz + q.id[i]);
        }
      }
    }
    if (G == 256) __syncthreads();       // with accumulate: the entries' old values are read before the row is written
    for (int c = c0 + l * V; c < c1; c += G * V) {
      float x[V], old[V];
      int b = c;
      if (dead) {
        if (g.accumulate) break;
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = 0.f;
        if (c + V > a.C) b = G == 8 && a.C < V ? c : a.C - V;
      } else {
        b = load_chunk<G == 8>(z, c, a.C, x);
        if (g.accumulate) load_chunk<G == 8>((const E*)dz, c, a.C, old);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = f * exp2_(((x[e] - base) * a.invT - off) * LOG2E) + (g.accumulate ? old[e] : 0.f);
      }
      store_chunk(dz, c, b, a.C, x);
    }
    if (G == 256) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (mine[i]) store1(dz + q.id[i], fix[i]);
  }
}

// ---- planes.  A lane needs q at the teacher's classes of its own PV pixels while it walks through all classes: CH classes at a time, q is
// scattered into the lane's own columns of a small LDS tile (no other lane touches them: no barrier, no conflict, the same class twice adds
// up in order), which costs an LDS write and read per logit instead of k comparisons.  A class of the teacher is marked by the sign.
constexpr int CH = 16;
__device__ __forceinline__ float tile_q(float v) { return __uint_as_float(__float_as_uint(v) & 0x7fffffffu); }
__device__ __forceinline__ bool tile_in(float v) { return __float_as_uint(v) >> 31; }

// The teacher of one pixel, its entries in a loop; the first KR of them stay in registers (0: they are read again, k > 8).
template <int KR>
struct PixTeacher {
  float m, ls, qsum, qrest, qlogq;
  bool any, bad, none;
  int id_[KR > 0 ? KR : 1];
  float q_[KR > 0 ? KR : 1];
  __device__ __forceinline__ float logq(const Teacher& t, const Logits& a, float v) const { return t.tail ? v : (v - m) * a.invT - ls; }
  __device__ __forceinline__ void init(const Teacher& t, const Logits& a, long long io, long long vo) {
    m = -INFINITY;
    any = bad = false;
    for (int j = 0; j < t.k; ++j) {
      const long long c = t.id(io, j);
      bad |= c >= a.C;
      if (c >= 0 && c < a.C) {
        any = true;
        m = fmaxf(m, t.value(vo, j));
      }
    }
    if (m == -INFINITY) m = 0.f;
    ls = 0.f;
    none = false;
    if (!t.tail) {
      float s = 0.f;
      for (int j = 0; j < t.k; ++j) {
        const long long c = t.id(io, j);
        if (c >= 0 && c < a.C) s += exp2_((t.value(vo, j) - m) * a.scale2);
      }
      none = s == 0.f;
      ls = none ? 0.f : log2_(s) * LN2;
    }
    qsum = qlogq = 0.f;
    if (KR > 0) {
#pragma unroll
      for (int j = 0; j < KR; ++j) {
        id_[j] = -1;
        q_[j] = 0.f;
        if (j < t.k) entry(t, a, io, vo, j, id_[j], q_[j]);
      }
    } else {
      for (int j = 0; j < t.k; ++j) entry(t, a, io, vo, j, id_[0], q_[0]);
    }
    qrest = t.tail ? fmaxf(1.f - qsum, 0.f) : 0.f;
    if (!t.tail) qsum = none ? 0.f : 1.f;
  }
  __device__ __forceinline__ void entry(const Teacher& t, const Logits& a, long long io, long long vo, int j, int& id, float& q) {
    const long long c = t.id(io, j);
    id = c < 0 || c >= a.C ? -1 : (int)c;
    q = 0.f;
    if (id >= 0) {
      const float lq = logq(t, a, t.value(vo, j));
      q = exp2_(lq * LOG2E);
      qlogq += q == 0.f ? 0.f : q * lq;
    }
    qsum += q;
  }
  // q of classes [c0, c0 + CH) into column `col` of the tile
  template <int COLS>
  __device__ __forceinline__ void scatter(const Teacher& t, const Logits& a, long long io, long long vo, int c0, float (*tile)[COLS],
                                          int col) const {
    if (KR > 0) {
#pragma unroll
      for (int j = 0; j < KR; ++j)
        if ((unsigned)(id_[j] - c0) < (unsigned)CH) {
          float* p = &tile[id_[j] - c0][col];
          *p = -(tile_q(*p) + q_[j]);
        }
    } else {
      for (int j = 0; j < t.k; ++j) {
        const long long c = t.id(io, j);
        if (c >= c0 && c < c0 + CH && c < a.C) {
          float* p = &tile[c - c0][col];
          *p = -(tile_q(*p) + exp2_(logq(t, a, t.value(vo, j)) * LOG2E));
        }
      }
    }
  }
};

// Loss: S about the running maximum, the mass outside the entries about the same one, sum of q d as it goes.  A wave has 64 * PV pixels;
// with SPLIT = 4 four waves share them and take a quarter of the classes each.
template <typename E, int PV, int KR, int SPLIT>
__global__ __launch_bounds__(64 * SPLIT) void distill_planes_kernel(const Logits a, const Teacher t, const DistillOut o, const int tiles,
                                                                    const long long all) {
  constexpr int COLS = 64 * PV, UN = 8;
  __shared__ float tiles_s[SPLIT][CH][COLS];
  __shared__ float red[SPLIT > 1 ? SPLIT - 1 : 1][5][SPLIT > 1 ? COLS : 1];
  const int wv = SPLIT > 1 ? threadIdx.x >> 6 : 0, lane = threadIdx.x & 63;
  float(*tile)[COLS] = tiles_s[wv];
  const int per = SPLIT > 1 ? ((a.C + SPLIT - 1) / SPLIT + CH - 1) / CH * CH : a.C;
  const int c_lo = wv * per, c_hi = min(a.C, c_lo + per);
  double loss = 0.0, wsum = 0.0;
  for (long long it = blockIdx.x; it < all; it += gridDim.x) {
    const long long i = all <= 0x7fffffff ? (unsigned)it / (unsigned)tiles : it / tiles, first = (it - i * tiles) * COLS + lane * PV;
    const Px<PV> px(first, a.p);
    const E* z = (const E*)a.z + i * a.sn + px.px;
    const long long r0 = i * a.p + px.px, io = i * t.in + px.px * t.ip, vo = i * t.vn + px.px * t.vp;
    float m[PV], base[PV], s[PV], st[PV], dot[PV], qacc[PV];
    PixTeacher<KR> q[PV];
#pragma unroll
    for (int v = 0; v < PV; ++v) {
      q[v].init(t, a, io + v * t.ip, vo + v * t.vp);
      m[v] = -INFINITY;
      base[v] = s[v] = st[v] = dot[v] = qacc[v] = 0.f;
    }
    for (int c0 = c_lo; c0 < c_hi; c0 += CH) {
#pragma unroll
      for (int n = 0; n < CH; ++n)
#pragma unroll
        for (int v = 0; v < PV; ++v) tile[n][lane * PV + v] = 0.f;
#pragma unroll
      for (int v = 0; v < PV; ++v) q[v].scatter(t, a, io + v * t.ip, vo + v * t.vp, c0, tile, lane * PV + v);
      for (int h = 0; h < CH && c0 + h < c_hi; h += UN) {
        E x[UN][PV];
#pragma unroll
        for (int n = 0; n < UN; ++n) load_px<E, PV>(z + min(c0 + h + n, c_hi - 1) * a.sc, x[n]);
#pragma unroll
        for (int v = 0; v < PV; ++v) {
          float y[UN], nm = m[v];
#pragma unroll
          for (int n = 0; n < UN; ++n) {
            y[n] = c0 + h + n < c_hi ? (float)x[n][v] : -INFINITY;
            nm = fmaxf(nm, y[n]);
          }
          const float nb = nm == -INFINITY ? 0.f : nm, f = exp2_((m[v] - nb) * a.scale2);
          s[v] *= f;
          st[v] *= f;
          dot[v] += qacc[v] == 0.f ? 0.f : qacc[v] * (base[v] - nb);
          m[v] = nm;
          base[v] = nb;
#pragma unroll
          for (int n = 0; n < UN; ++n) {
            const float d = y[n] - nb, p = exp2_(d * a.scale2), tv = tile[h + n][lane * PV + v], qc = tile_q(tv);
            s[v] += p;
            if (t.tail) st[v] += tile_in(tv) ? 0.f : p;
            dot[v] += qc == 0.f ? 0.f : qc * d;
            qacc[v] += qc;
          }
        }
      }
    }
    if constexpr (SPLIT > 1) {
      __syncthreads();                 // the tile before this one has been joined
      if (wv > 0) {
#pragma unroll
        for (int v = 0; v < PV; ++v) {
          float* p = &red[wv - 1][0][lane * PV + v];
          p[0] = m[v];
          p[COLS] = s[v];
          p[2 * COLS] = st[v];
          p[3 * COLS] = dot[v];
          p[4 * COLS] = qacc[v];
        }
      }
      __syncthreads();
      if (wv > 0) continue;
      for (int w = 0; w < SPLIT - 1; ++w) {
#pragma unroll
        for (int v = 0; v < PV; ++v) {
          const float* p = &red[w][0][lane * PV + v];
          const float om = p[0], ob = om == -INFINITY ? 0.f : om, oq = p[4 * COLS];
          const float nm = fmaxf(m[v], om), nb = nm == -INFINITY ? 0.f : nm;
          const float f = exp2_((m[v] - nb) * a.scale2), of = exp2_((om - nb) * a.scale2);
          s[v] = s[v] * f + p[COLS] * of;
          st[v] = st[v] * f + p[2 * COLS] * of;
          dot[v] += p[3 * COLS] + (qacc[v] == 0.f ? 0.f : qacc[v] * (base[v] - nb)) + (oq == 0.f ? 0.f : oq * (ob - nb));
          qacc[v] += oq;
          m[v] = nm;
          base[v] = nb;
        }
      }
    }
    if (first >= a.p) continue;
#pragma unroll
    for (int v = 0; v < PV; ++v) {
      if (!px.own(v)) continue;
      const long long r = r0 + v;
      const float w = t.weight ? t.weight[r] : 1.f;
      const float ls = log2_(s[v]) * LN2;
      float lpt = 0.f, kl = s[v] == 0.f ? (q[v].qsum > 0.f ? INFINITY : 0.f) : q[v].qlogq - (dot[v] * a.invT - q[v].qsum * ls);
      bool rest = t.tail;
      if (t.tail) {
        lpt = log2_(st[v]) * LN2 - ls;
        if (st[v] < 1e-20f) {          // the rest is far below the row's maximum: once more, about its own
          float mt = -INFINITY, sum = 0.f;
          for (int c = 0; c < a.C; ++c) {
            const float y = load1(z + c * a.sc + v);
            bool in = false;
            for (int j = 0; j < t.k; ++j) in |= t.id(io + v * t.ip, j) == c;
            if (in || y == -INFINITY) continue;
            const float nm = fmaxf(mt, y);
            sum = sum * exp2_((mt - nm) * a.scale2) + exp2_((y - nm) * a.scale2);
            mt = nm;
          }
          rest = mt != -INFINITY;
          lpt = rest ? (mt - base[v]) * a.invT + log2_(sum) * LN2 - ls : 0.f;
        }
        if (rest && q[v].qrest > 0.f) kl += q[v].qrest * (log2_(q[v].qrest) * LN2 - lpt);
      }
      if (!q[v].any) kl = 0.f;
      if (q[v].bad) kl = NAN;
      const bool on = w != 0.f;        // a masked row's logits have been read, but nothing of them goes on
      o.stats[r] = on ? base[v] : 0.f;
      o.stats[a.R + r] = on ? ls : 0.f;
      o.stats[2 * a.R + r] = !on ? 0.f : t.tail && !rest ? INFINITY : lpt;
      if (o.rows) o.rows[r] = on ? o.T2 * w * kl : 0.f;
      if (on) {
        loss += (double)w * (double)kl;
        wsum += (double)w;
      }
    }
  }
  block_part<64 * SPLIT>(o.part, loss, wsum);
}

template <typename E, int PV, int KR>
__global__ __launch_bounds__(64) void distill_bwd_planes_kernel(const Logits a, const Teacher t, const DistillGrad g, const long long i0,
                                                                const int tiles, const int slice) {
  constexpr int COLS = 64 * PV, UN = 8;
  __shared__ float tile[CH][COLS];
  const int lane = threadIdx.x;
  const long long i = i0 + blockIdx.x / (unsigned)tiles, first = (long long)(blockIdx.x % (unsigned)tiles) * COLS + lane * PV;
  if (first >= a.p) return;
  const Px<PV> px(first, a.p);
  const E* z = (const E*)a.z + i * a.sn + px.px;
  E* dz = (E*)g.dz + i * g.dn + px.px;
  const long long r0 = i * a.p + px.px, io = i * t.in + px.px * t.ip, vo = i * t.vn + px.px * t.vp;
  PixTeacher<KR> q[PV];
  float base[PV], ls[PV], off[PV], cq[PV], f[PV], coef[PV];
  bool dead[PV];
#pragma unroll
  for (int v = 0; v < PV; ++v) {
    q[v].init(t, a, io + v * t.ip, vo + v * t.vp);
    const float w = t.weight ? t.weight[r0 + v] : 1.f;
    base[v] = g.stats[r0 + v];
    ls[v] = g.stats[a.R + r0 + v];
    const float lpt = g.stats[2 * a.R + r0 + v];
    const bool rest = t.tail && lpt != INFINITY;
    const float Q = rest ? q[v].qsum + q[v].qrest : q[v].qsum;
    dead[v] = w == 0.f || q[v].bad || !q[v].any || ls[v] == -INFINITY;
    coef[v] = g.coef(r0 + v, w);
    cq[v] = coef[v] * Q;
    off[v] = rest ? ls[v] + lpt : ls[v];
    f[v] = coef[v] * (rest ? Q * exp2_(lpt * LOG2E) - q[v].qrest : Q);
  }
  const int c_lo = blockIdx.y * slice, c_hi = min(a.C, c_lo + slice);
  for (int c0 = c_lo; c0 < c_hi; c0 += CH) {
#pragma unroll
    for (int n = 0; n < CH; ++n)
#pragma unroll
      for (int v = 0; v < PV; ++v) tile[n][lane * PV + v] = 0.f;
#pragma unroll
    for (int v = 0; v < PV; ++v) q[v].scatter(t, a, io + v * t.ip, vo + v * t.vp, c0, tile, lane * PV + v);
    for (int h = 0; h < CH && c0 + h < c_hi; h += UN) {
      E x[UN][PV], old[UN][PV];
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        load_px<E, PV>(z + min(c0 + h + n, c_hi - 1) * a.sc, x[n]);
        if (g.accumulate) load_px<E, PV>(dz + min(c0 + h + n, c_hi - 1) * g.dc, old[n]);
      }
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        if (c0 + h + n >= c_hi) break;
#pragma unroll
        for (int v = 0; v < PV; ++v) {
          const float tv = tile[h + n][lane * PV + v], d = ((float)x[n][v] - base[v]) * a.invT;
          const bool in = tile_in(tv);
          float y = (in ? cq[v] : f[v]) * exp2_((d - (in ? ls[v] : off[v])) * LOG2E) - coef[v] * tile_q(tv);
          if (dead[v]) y = 0.f;
          x[n][v] = (E)(y + (g.accumulate ? (float)old[n][v] : 0.f));
        }
        if (px.own(0)) {
          store_px<E, PV>(dz + (c0 + h + n) * g.dc, x[n]);
        } else {
#pragma unroll
          for (int v = 1; v < PV; ++v)
            if (px.own(v)) store1(dz + (c0 + h + n) * g.dc + v, (float)x[n][v]);
        }
      }
    }
  }
}

int row_blocks(long long R) {
  const long long b = (R + 3) / 4;
  return (int)(b < 8192 ? b : 8192);
}

bool logits_ok(const void* z, int type, long long n, long long p, int C, float T) {
  return z && type >= 0 && type <= 2 && n > 0 && p > 0 && C > 0 && C <= (1 << 30) && p <= (1ll << 40) / n && T > 0.f && T <= 3e38f;
}
// rows: contiguous classes; planes: contiguous pixels (of fewer than 2^31 to an image)
bool layout_ok(int C, long long p, long long sp, long long sc) { return C == 1 || sc == 1 || (sp == 1 && p < (1ll << 31)); }
bool teacher_ok(const void* ids, int ids64, const void* top, int top_type, int k) {
  return ids && top && (ids64 == 0 || ids64 == 1) && top_type >= 0 && top_type <= 2 && k >= 1 && k <= MAXK;
}

Logits logits_of(const void* z, long long n, long long p, int C, long long sn, long long sp, long long sc, float T) {
  return Logits{z, n * p, p, sn, sp, sc, C, 1.f / T, LOG2E / T};
}

// Slices of a row of more classes than ROW_CLASSES: none with 512 rows or more (two blocks a compute unit), else about 1024 blocks in
// all, a slice no shorter than 4096 classes.
constexpr int ROW_CLASSES = 2048;
struct Split { int nsplit, slice, join; };
Split split_rows(int type, long long R, int C) {
  const int v = type == SEMSEG_TYPE_F32 ? 4 : 8;
  if (C <= ROW_CLASSES) return Split{1, C, 1};
  long long n = R >= 512 ? 1 : 1024 / R;
  if (n > 64) n = 64;
  if (n > (C + 4095) / 4096) n = (C + 4095) / 4096;
  const int slice = (int)(((C + n - 1) / n + v - 1) / v * v);
  const int iters = (slice + 256 * v - 1) / (256 * v);
  return Split{(C + slice - 1) / slice, slice, (iters + 127) / 128};
}
int capped(long long blocks, int cap) { return (int)(blocks < cap ? blocks : cap); }

// launch(first image, images): groups of images whose grids stay below 2^32 lanes
template <typename F>
void by_images(const Logits& a, long long tiles, F launch) {
  const long long n = a.R / a.p, most = tiles >= (1ll << 23) ? 1 : (1ll << 23) / tiles;
  for (long long i = 0; i < n; i += most) launch(i, (int)(n - i < most ? n - i : most));
}

template <typename E, int PV, int K>
void logprobs_planes_k(const Logits& a, const LogprobOut& o, hipStream_t stream) {
  // a wave to every class quarter where whole images to a lane give less than four blocks a compute unit
  const long long whole = (a.p + 256 * PV - 1) / (256 * PV), quarter = (a.p + 64 * PV - 1) / (64 * PV);
  if (a.R / a.p * whole >= 1024 || a.C < 16)
    by_images(a, whole, [&](long long i0, int n) { logprobs_planes_kernel<E, PV, K, 1><<<n * (int)whole, 256, 0, stream>>>(a, o, i0, (int)whole); });
  else
    by_images(a, quarter, [&](long long i0, int n) { logprobs_planes_kernel<E, PV, K, 4><<<n * (int)quarter, 256, 0, stream>>>(a, o, i0, (int)quarter); });
}
template <typename E>
void logprobs_planes(const Logits& a, const LogprobOut& o, hipStream_t stream) {
  constexpr int PV = sizeof(E) == 2 ? 2 : 1;      // two 16-bit pixels to a lane while their lists leave registers for it
  if (PV == 2 && a.p == 1) {
    if (o.k <= 16) logprobs_planes_k<E, 1, 16>(a, o, stream);
    else logprobs_planes_k<E, 1, 32>(a, o, stream);
  } else if (o.k == 0) logprobs_planes_k<E, PV, 0>(a, o, stream);
  else if (o.k == 1) logprobs_planes_k<E, PV, 1>(a, o, stream);
  else if (o.k == 2) logprobs_planes_k<E, PV, 2>(a, o, stream);
  else if (o.k == 3) logprobs_planes_k<E, PV, 3>(a, o, stream);
  else if (o.k == 4) logprobs_planes_k<E, PV, 4>(a, o, stream);
  else if (o.k <= 8) logprobs_planes_k<E, PV, 8>(a, o, stream);
  else if (o.k <= 16) logprobs_planes_k<E, 1, 16>(a, o, stream);
  else logprobs_planes_k<E, 1, 32>(a, o, stream);
}

template <typename E>
void logprobs_bwd(const Logits& a, const LogprobGrad& g, hipStream_t stream) {
  if (a.C > 1 && a.sc != 1) {
    constexpr int PV = sizeof(E) == 2 ? 2 : 1;
    const int pv = a.p > 1 ? PV : 1;
    const long long tiles = (a.p + 256 * pv - 1) / (256 * pv);
    // slices of the classes until there are about eight blocks a compute unit, none shorter than 16 classes
    const long long blocks = a.R / a.p * tiles;
    int slices = blocks >= 2048 ? 1 : (int)(2048 / blocks);
    if (slices > (a.C + 15) / 16) slices = (a.C + 15) / 16;
    const int slice = (a.C + slices - 1) / slices;
    by_images(a, tiles * slices, [&](long long i0, int n) {
      const dim3 grid(n * (unsigned)tiles, (a.C + slice - 1) / slice);
      if (pv == PV) logprobs_bwd_planes_kernel<E, PV><<<grid, 256, 0, stream>>>(a, g, i0, (int)tiles, slice);
      else logprobs_bwd_planes_kernel<E, 1><<<grid, 256, 0, stream>>>(a, g, i0, (int)tiles, slice);
    });
    return;
  }
  if (a.C <= 256) logprobs_bwd_rows_kernel<E, 8><<<capped((a.R + 31) / 32, 16384), 256, 0, stream>>>(a, g, 1);
  else if (a.C <= 4 * 64 * VEC<E>) logprobs_bwd_rows_kernel<E, 64><<<capped((a.R + 3) / 4, 16384), 256, 0, stream>>>(a, g, 1);
  else {
    const int segs = (a.C + 4 * 256 * VEC<E> - 1) / (4 * 256 * VEC<E>);
    logprobs_bwd_rows_kernel<E, 256><<<capped(a.R * segs, 1 << 20), 256, 0, stream>>>(a, g, segs);
  }
}

template <typename E>
void logprobs_fwd(const Logits& a, const LogprobOut& o, int type, void* scratch, hipStream_t stream) {
  if (a.C > 1 && a.sc != 1) {
    if (o.k > PLANE_K || a.C > PLANE_CLASSES) {
      logprobs_fwd_kernel<E><<<row_blocks(a.R), 256, 0, stream>>>(a, o);
    } else {
      logprobs_planes<E>(a, o, stream);
    }
    return;
  }
  if (a.C <= ROW_CLASSES) {
    const int chunks = (a.C + VEC<E> - 1) / VEC<E>;
#define ROWS(G, NV) logprobs_rows_kernel<E, G, NV><<<capped((a.R + 256 / G - 1) / (256 / G), 16384), 256, 0, stream>>>(a, o)
    if (chunks <= 8) ROWS(8, 1);
    else if (chunks <= 16) ROWS(8, 2);
    else if (chunks <= 24) ROWS(8, 3);
    else if (chunks <= 32) ROWS(8, 4);
    else if (VEC<E> == 4 && chunks <= 40) ROWS(8, VEC<E> == 4 ? 5 : 1);
    else if (VEC<E> == 4 && chunks <= 64) ROWS(8, VEC<E> == 4 ? 8 : 1);
    else if (chunks <= 64) ROWS(64, 1);
    else if (chunks <= 128) ROWS(64, 2);
    else if (chunks <= 256) ROWS(64, 4);
    else ROWS(64, VEC<E> == 4 ? 8 : 1);
#undef ROWS
    return;
  }
  const Split s = split_rows(type, a.R, a.C);
  Stream t{0, s.nsplit, s.slice, s.join, (float*)scratch, nullptr};
  // the keys first in the scratch: they need 8-byte alignment
  t.keys = (unsigned long long*)scratch;
  t.part = (float*)(t.keys + a.R * s.nsplit * o.k);
  const long long most = (1ll << 23) / s.nsplit;       // a grid holds less than 2^32 lanes
  for (t.r0 = 0; t.r0 < a.R; t.r0 += most) {
    const int rows = (int)(a.R - t.r0 < most ? a.R - t.r0 : most);
    logprobs_stream_kernel<E><<<rows * s.nsplit, 256, 0, stream>>>(a, o, t);
    if (s.nsplit > 1) logprobs_join_kernel<E><<<rows, 64, 0, stream>>>(a, o, t);
  }
}

// Blocks of the loss kernels: one partial sum each
constexpr int PARTS = 4096;
template <typename E>
int distill_blocks(const Logits& a, long long* all, int* split) {
  if (a.C > 1 && a.sc != 1) {
    const int pv = sizeof(E) == 2 && a.p > 1 ? 2 : 1;
    *all = a.R / a.p * ((a.p + 64 * pv - 1) / (64 * pv));
    *split = *all < 2048 && a.C >= 64 ? 4 : 1;      // too few waves for the device: a quarter of the classes each
    return capped(*all, PARTS);
  }
  *all = a.R;
  *split = 1;
  return capped((a.R + (a.C <= 256 ? 31 : 3)) / (a.C <= 256 ? 32 : 4), PARTS);
}

template <typename E, bool GRAD>
void distill_rows(const Logits& a, const Teacher& t, const DistillOut& o, const DistillGrad& g, int blocks, hipStream_t stream) {
  const int chunks = (a.C + VEC<E> - 1) / VEC<E>;
#define DROWS(G, NV, NE) distill_rows_kernel<E, G, NV, NE, GRAD><<<blocks, 256, 0, stream>>>(a, t, o, g)
#define DROWS8(NV) do { if (t.k <= 8) DROWS(8, NV, 1); else DROWS(8, NV, 8); } while (0)
  if (chunks <= 8) DROWS8(1);
  else if (chunks <= 16) DROWS8(2);
  else if (chunks <= 32 && VEC<E> == 8) DROWS8(4);
  else if (chunks <= 24) DROWS8(3);
  else if (chunks <= 40 && VEC<E> == 4) DROWS8(VEC<E> == 4 ? 5 : 1);
  else if (chunks <= 64 && VEC<E> == 4) DROWS8(VEC<E> == 4 ? 8 : 1);
  else if (chunks <= 64) DROWS(64, 1, 1);
  else if (chunks <= 128) DROWS(64, 2, 1);
  else if (chunks <= 256) DROWS(64, 4, 1);
  else DROWS(64, VEC<E> == 4 ? 8 : 1, 1);
#undef DROWS8
#undef DROWS
}

// Loss and statistics; partial sums to o.part
template <typename E>
void distill_fwd(const Logits& a, const Teacher& t, const DistillOut& o, int type, float* scratch, hipStream_t stream) {
  long long all;
  int split;
  const int blocks = distill_blocks<E>(a, &all, &split);
  if (a.C > 1 && a.sc != 1) {
    constexpr int PV = sizeof(E) == 2 ? 2 : 1;
    const int pv = a.p > 1 ? PV : 1, tiles = (int)((a.p + 64 * pv - 1) / (64 * pv));
#define DPLANES(PV_, KR, SP) distill_planes_kernel<E, PV_, KR, SP><<<blocks, 64 * SP, 0, stream>>>(a, t, o, tiles, all)
    if (PV == 2 && pv == 1) DPLANES(1, 0, 4);
    else if (split == 1 && t.k <= 4) DPLANES(PV, 4, 1);
    else if (split == 1 && t.k <= 8) DPLANES(PV, 8, 1);
    else if (split == 1) DPLANES(PV, 0, 1);
    else if (t.k <= 4) DPLANES(PV, 4, 4);
    else if (t.k <= 8) DPLANES(PV, 8, 4);
    else DPLANES(PV, 0, 4);
#undef DPLANES
    return;
  }
  if (a.C <= ROW_CLASSES) {
    distill_rows<E, false>(a, t, o, DistillGrad{}, blocks, stream);
    return;
  }
  const Split s = split_rows(type, a.R, a.C);
  DStream d{0, s.nsplit, s.slice, scratch};
  const long long most = (1ll << 23) / s.nsplit;
  for (d.r0 = 0; d.r0 < a.R; d.r0 += most)
    distill_stream_kernel<E><<<(int)(a.R - d.r0 < most ? a.R - d.r0 : most) * s.nsplit, 256, 0, stream>>>(a, t, d);
  distill_join_kernel<E><<<blocks, 256, 0, stream>>>(a, t, o, d);
}

template <typename E>
void distill_bwd(const Logits& a, const Teacher& t, const DistillGrad& g, hipStream_t stream) {
  if (a.C > 1 && a.sc != 1) {
    constexpr int PV = sizeof(E) == 2 ? 2 : 1;
    const int pv = a.p > 1 ? PV : 1;
    const long long tiles = (a.p + 64 * pv - 1) / (64 * pv), blocks = a.R / a.p * tiles;
    // slices of the classes until there are about 16 waves a compute unit
    const int tc = (a.C + CH - 1) / CH, slices = blocks >= 4096 ? 1 : (int)(4096 / blocks < tc ? 4096 / blocks : tc);
    const int slice = (tc + slices - 1) / slices * CH;
    by_images(a, tiles * slices, [&](long long i0, int n) {
      const dim3 grid(n * (unsigned)tiles, (a.C + slice - 1) / slice);
      if (pv != PV) distill_bwd_planes_kernel<E, 1, 0><<<grid, 64, 0, stream>>>(a, t, g, i0, (int)tiles, slice);
      else if (t.k <= 4) distill_bwd_planes_kernel<E, PV, 4><<<grid, 64, 0, stream>>>(a, t, g, i0, (int)tiles, slice);
      else if (t.k <= 8) distill_bwd_planes_kernel<E, PV, 8><<<grid, 64, 0, stream>>>(a, t, g, i0, (int)tiles, slice);
      else distill_bwd_planes_kernel<E, PV, 0><<<grid, 64, 0, stream>>>(a, t, g, i0, (int)tiles, slice);
    });
    return;
  }
  if (a.C <= 256) distill_bwd_rows_kernel<E, 8><<<capped((a.R + 31) / 32, 16384), 256, 0, stream>>>(a, t, g, 1);
  else if (a.C <= 4 * 64 * VEC<E>) distill_bwd_rows_kernel<E, 64><<<capped((a.R + 3) / 4, 16384), 256, 0, stream>>>(a, t, g, 1);
  else {
    const int segs = (a.C + 4 * 256 * VEC<E> - 1) / (4 * 256 * VEC<E>);
    distill_bwd_rows_kernel<E, 256><<<capped(a.R * segs, 1 << 20), 256, 0, stream>>>(a, t, g, segs);
  }
}

#define BY_TYPE(type, F, ...)                                  \
  do {                                                         \
    if (type == SEMSEG_TYPE_F32) F<float>(__VA_ARGS__);        \
    else if (type == SEMSEG_TYPE_BF16) F<__bf16>(__VA_ARGS__); \
    else F<_Float16>(__VA_ARGS__);                             \
  } while (0)

// Scratch of a distillation call: partial sums, then the slices' maxima and sums of long rows
size_t distill_need(int type, long long R, int C, long long sc) {
  size_t need = (size_t)PARTS * 2 * sizeof(double);
  if ((C == 1 || sc == 1) && C > ROW_CLASSES) need += (size_t)R * split_rows(type, R, C).nsplit * 2 * sizeof(float);
  return need;
}
float* distill_slices(void* scratch) { return (float*)((double*)scratch + 2 * PARTS); }

}  // namespace

extern "C" {

size_t semseg_class_logprobs_scratch_bytes(int type, long long n, long long p, int C, long long sc, int k) {
  if (n <= 0 || p <= 0 || C <= 0 || k < 0 || (sc != 1 && C > 1)) return 0;
  const Split s = split_rows(type, n * p, C);
  return s.nsplit < 2 ? 0 : (size_t)(n * p) * s.nsplit * (3 * sizeof(float) + k * sizeof(unsigned long long));
}

int semseg_class_logprobs_fwd(const void* z, int type, long long n, long long p, int C, long long sn, long long sp, long long sc,
                              const long long* label, long long ignore_index, float T, int k, float* logprob, float* entropy,
                              float* lse, float* stats, int* top_ids, float* top_logprobs, long long tn, long long tp, long long tk,
                              void* scratch, size_t scratch_bytes, hipStream_t stream) {
  if (!logits_ok(z, type, n, p, C, T) || k < 0 || k > MAXK || k > C || (k && (!top_ids || !top_logprobs)) || (logprob && !label))
    return SEMSEG_EINVAL;
  if (!layout_ok(C, p, sp, sc)) return SEMSEG_EINVAL;
  const size_t need = semseg_class_logprobs_scratch_bytes(type, n, p, C, sc, k);
  if (need && (!scratch || scratch_bytes < need)) return SEMSEG_EINVAL;
  const Logits a = logits_of(z, n, p, C, sn, sp, sc, T);
  const LogprobOut o{label, ignore_index, logprob, entropy, lse, stats, top_ids, top_logprobs, k, tn, tp, tk};
  BY_TYPE(type, logprobs_fwd, a, o, type, scratch, stream);
  return semseg_launch_status();
}

int semseg_class_logprobs_bwd(const void* z, int type, long long n, long long p, int C, long long sn, long long sp, long long sc,
                              const long long* label, long long ignore_index, float T, const float* stats, const float* entropy,
                              const float* g_logprob, const float* g_entropy, const float* g_lse, void* dz, long long dn,
                              long long dp, long long dc, int accumulate, hipStream_t stream) {
  if (!logits_ok(z, type, n, p, C, T) || !stats || !dz || (g_entropy && !entropy) || (g_logprob && !label)) return SEMSEG_EINVAL;
  // the gradient is in the logits' form
  if (!layout_ok(C, p, sp, sc) || !(C == 1 || (sc == 1 ? dc == 1 : dp == 1))) return SEMSEG_EINVAL;
  const Logits a = logits_of(z, n, p, C, sn, sp, sc, T);
  const LogprobGrad g{label, ignore_index, stats, entropy, g_logprob, g_entropy, g_lse, dz, dn, dp, dc, accumulate};
  BY_TYPE(type, logprobs_bwd, a, g, stream);
  return semseg_launch_status();
}

size_t semseg_distill_scratch_bytes(int type, long long n, long long p, int C, long long sc) {
  if (n <= 0 || p <= 0 || C <= 0) return 0;
  return distill_need(type, n * p, C, sc);
}

int semseg_distill_fwd(const void* z, int type, long long n, long long p, int C, long long sn, long long sp, long long sc, const void* ids,
                       int ids64, const void* top, int top_type, int k, long long in, long long ip, long long ik, long long vn,
                       long long vp, long long vk, const float* weight, float T, int tail, int reduction, float* rows, float* stats,
                       double* acc2, float* loss, void* scratch, size_t scratch_bytes, hipStream_t stream) {
  if (!logits_ok(z, type, n, p, C, T) || !layout_ok(C, p, sp, sc) || !teacher_ok(ids, ids64, top, top_type, k) || !stats || reduction < 0 ||
      reduction > 2 || !scratch || scratch_bytes < distill_need(type, n * p, C, sc) ||
      (reduction == SEMSEG_REDUCE_NONE ? !rows : (!acc2 || !loss)))
    return SEMSEG_EINVAL;
  const Logits a = logits_of(z, n, p, C, sn, sp, sc, T);
  const Teacher t{ids, top, ids64, top_type, k, tail, in, ip, ik, vn, vp, vk, weight};
  const DistillOut o{rows, stats, reduction == SEMSEG_REDUCE_NONE ? nullptr : (double*)scratch, T * T};
  BY_TYPE(type, distill_fwd, a, t, o, type, distill_slices(scratch), stream);
  if (reduction != SEMSEG_REDUCE_NONE) {
    long long all;
    int split;
    const int blocks = type == SEMSEG_TYPE_F32 ? distill_blocks<float>(a, &all, &split) : distill_blocks<__bf16>(a, &all, &split);
    distill_finish_kernel<<<1, 1024, 0, stream>>>((const double*)scratch, blocks, acc2, loss, T * T, reduction == SEMSEG_REDUCE_MEAN);
  }
  return semseg_launch_status();
}

int semseg_distill_bwd(const void* z, int type, long long n, long long p, int C, long long sn, long long sp, long long sc, const void* ids,
                       int ids64, const void* top, int top_type, int k, long long in, long long ip, long long ik, long long vn,
                       long long vp, long long vk, const float* weight, float T, int tail, int reduction, const float* stats,
                       const double* acc2, const float* grad_loss, float grad_mul, void* dz, long long dn, long long dp, long long dc,
                       int accumulate, hipStream_t stream) {
  if (!logits_ok(z, type, n, p, C, T) || !layout_ok(C, p, sp, sc) || !teacher_ok(ids, ids64, top, top_type, k) || !stats || !dz ||
      reduction < 0 || reduction > 2 || (reduction == SEMSEG_REDUCE_MEAN && !acc2) || !(C == 1 || (sc == 1 ? dc == 1 : dp == 1)))
    return SEMSEG_EINVAL;
  const Logits a = logits_of(z, n, p, C, sn, sp, sc, T);
  const Teacher t{ids, top, ids64, top_type, k, tail, in, ip, ik, vn, vp, vk, weight};
  const DistillGrad g{stats, acc2, 0.0, grad_loss, grad_mul, T, reduction == SEMSEG_REDUCE_MEAN, reduction == SEMSEG_REDUCE_NONE,
                      accumulate, dz, dn, dp, dc};
  BY_TYPE(type, distill_bwd, a, t, g, stream);
  return semseg_launch_status();
}

int semseg_distill_fwd_bwd(const void* z, int type, long long n, long long p, int C, long long sn, long long sp, long long sc,
                           const void* ids, int ids64, const void* top, int top_type, int k, long long in, long long ip, long long ik,
                           long long vn, long long vp, long long vk, const float* weight, float T, int tail, int reduction,
                           float* stats, double* acc2, float* loss, float grad_mul, void* dz, long long dn, long long dp, long long dc,
                           int accumulate, void* scratch, size_t scratch_bytes, hipStream_t stream) {
  if (reduction != SEMSEG_REDUCE_MEAN && reduction != SEMSEG_REDUCE_SUM) return SEMSEG_EINVAL;
  if ((C == 1 || sc == 1) && C <= ROW_CLASSES) {       // rows held in registers: one read of the logits serves both
    if (!logits_ok(z, type, n, p, C, T) || !teacher_ok(ids, ids64, top, top_type, k) || !acc2 || !loss || !dz || !(C == 1 || dc == 1) ||
        !scratch || scratch_bytes < distill_need(type, n * p, C, sc))
      return SEMSEG_EINVAL;
    const Logits a = logits_of(z, n, p, C, sn, sp, sc, T);
    const Teacher t{ids, top, ids64, top_type, k, tail, in, ip, ik, vn, vp, vk, weight};
    const DistillOut o{nullptr, nullptr, (double*)scratch, T * T};
    const int mean = reduction == SEMSEG_REDUCE_MEAN;
    const DistillGrad g{nullptr, weight ? acc2 : nullptr, (double)a.R, nullptr, grad_mul, T, mean, 0, accumulate, dz, dn, dp, dc};
    long long all;
    int split;
    const int blocks = type == SEMSEG_TYPE_F32 ? distill_blocks<float>(a, &all, &split) : distill_blocks<__bf16>(a, &all, &split);
    if (weight && mean) {                              // the gradient needs their sum first
      const int wb = capped((a.R + 255) / 256, 256);
      weight_sum_kernel<<<wb, 256, 0, stream>>>(weight, a.R, (double*)scratch);
      distill_finish_kernel<<<1, 1024, 0, stream>>>((const double*)scratch, wb, acc2, nullptr, T * T, mean);
    }
    if (type == SEMSEG_TYPE_F32) distill_rows<float, true>(a, t, o, g, blocks, stream);
    else if (type == SEMSEG_TYPE_BF16) distill_rows<__bf16, true>(a, t, o, g, blocks, stream);
    else distill_rows<_Float16, true>(a, t, o, g, blocks, stream);
    distill_finish_kernel<<<1, 1024, 0, stream>>>((const double*)scratch, blocks, acc2, loss, T * T, mean);
    return semseg_launch_status();
  }
  const int rc = semseg_distill_fwd(z, type, n, p, C, sn, sp, sc, ids, ids64, top, top_type, k, in, ip, ik, vn, vp, vk, weight, T, tail,
                                    reduction, nullptr, stats, acc2, loss, scratch, scratch_bytes, stream);
  if (rc != SEMSEG_OK) return rc;
  return semseg_distill_bwd(z, type, n, p, C, sn, sp, sc, ids, ids64, top, top_type, k, in, ip, ik, vn, vp, vk, weight, T, tail,
                            reduction, stats, acc2, nullptr, grad_mul, dz, dn, dp, dc, accumulate, stream);
}

}  // extern "C"
