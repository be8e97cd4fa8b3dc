// Log probability of a given class, entropy and the k best classes of every row of logits, and their gradient (class_probs.h: the
// formulas and how rows lie in memory).
#include "class_probs.h"

namespace {

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

// One wave per row, lanes along the classes, every pass read again: planes of more classes than the kernel below can name in its keys
// (65536; fp16 8192), or more than 32 alternatives of a pixel, whose lists would not fit registers.
template <typename E>
__global__ __launch_bounds__(256) void logprobs_fwd_kernel(const Logits a, const LogprobOut o) {
  const int lane = threadIdx.x & 63;
  const long long waves = (long long)gridDim.x * 4;
  for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.R; r += waves) {
    const E* z = (const E*)a.z + a.at(r);
    const long long y = o.label ? o.label[r] : 0;
    const long long ot = row_at(a, r, o.tn, o.tp);
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
    m = group_max<64>(m);
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f, u = 0.f, lost_s = 0.f, lost_u = 0.f;
    for (int c = lane; c < a.C; c += 64) {
      const float d = (load1(z + c * a.sc) - base) * a.scale2, e = exp2_(d);
      add_group(s, lost_s, e);
      add_group(u, lost_u, e * fmaxf(d, -300.f));      // exp2(-300) = 0 in fp32; 0 * -inf would be NaN
    }
    s = at_least_one(group_sum<64>(s));
    u = not_positive(group_sum<64>(u));
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
      prev = group_max64<64>(best);
      if (lane == 0) {
        const int c = (int)~(unsigned)prev;
        o.top_ids[ot + j * o.tk] = c;
        o.top_lp[ot + j * o.tk] = s == 0.f ? -INFINITY : (load1(z + c * a.sc) - base) * a.invT - ls;
      }
    }
  }
}

// Rows of at most 2048 contiguous classes: G lanes (4 up to 160 classes, 8 up to 256, 64 beyond) hold a row in registers, NV chunks of
// 16 bytes each, so it is read once and its maximum, sums and alternatives are reductions over registers and a few data-parallel moves.
// Few lanes to a row, because most of an alternative's instructions cost the same whatever they serve: with 4 lanes 16 rows a wave.
// An alternative is one round: the lanes' chunk maxima, their largest, the lowest class that has it, that class taken out and its chunk's
// maximum renewed.  The chunks lie in LDS too, where a lane reads the one that it needs by its number (selecting it from registers, and
// changing it there, took twice the instructions: 57600 x 150, 8 alternatives: 22.9 us).  16 us now, bound by the instructions of this
// selection (100 a row, 85 % of the issue slots); its 39 MB would take 5.5.  Each alternative is a round behind the one before: k 64 takes 56.
template <typename E, int G, int NV, bool TOP>
__global__ __launch_bounds__(256) void logprobs_rows_kernel(const Logits a, const LogprobOut o) {
  constexpr int V = VEC<E>;
  constexpr bool SHORT = G < 64 && NV == 1;
  __shared__ __attribute__((aligned(16))) float keep[TOP ? NV : 1][TOP ? 256 : 1][V];
  const int l = threadIdx.x % G;
  const long long step = (long long)gridDim.x * (256 / G);
  for (long long r = (long long)blockIdx.x * (256 / G) + threadIdx.x / G; r < a.R; r += step) {
    const long long y = o.label ? o.label[r] : 0;
    const long long ot = o.k ? row_at(a, r, o.tn, o.tp) : 0;
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
    load_chunks<NV, SHORT>(z, l * V, G * V, a.C, x, b);
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
    if (!TOP) continue;
    if (s != s) {                                  // a NaN or +inf: the alternatives one by one, NaN above +inf
      unsigned long long prev = ~0ull;
      for (int j = 0; j < o.k; ++j) {
        unsigned long long best = 0;
        for (int c = l; c < a.C; c += G) {
          const unsigned long long key = pair_key(load1(z + c), c);
          if (key < prev && key > best) best = key;
        }
        prev = group_max64<G>(best);
        if (l == 0) {
          o.top_ids[ot + j * o.tk] = (int)~(unsigned)prev;
          o.top_lp[ot + j * o.tk] = s;
        }
      }
      continue;
    }
    // NaN is no candidate to the maxima below: it marks what is no class of this lane and what has been taken.
    float cm[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int first = (i * G + l) * V;
      if (first + V > a.C) {
#pragma unroll
        for (int e = 0; e < V; ++e) x[i][e] = b[i] + e >= first && b[i] + e < a.C ? x[i][e] : NAN;
      }
      cm[i] = x[i][0];
#pragma unroll
      for (int e = 1; e < V; ++e) cm[i] = fmaxf(cm[i], x[i][e]);
#pragma unroll
      for (int e = 0; e < V; e += 4) *reinterpret_cast<f32x4*>(&keep[i][threadIdx.x][e]) = f32x4{x[i][e], x[i][e + 1], x[i][e + 2], x[i][e + 3]};
    }
    int kid = 0;
    float kv = 0.f;
    for (int j = 0; j < o.k; ++j) {
      float best = cm[0];
#pragma unroll
      for (int i = 1; i < NV; ++i) best = fmaxf(best, cm[i]);
      best = group_max<G>(best);
      int ch = -1;                                 // the lane's first chunk that holds it
#pragma unroll
      for (int i = NV - 1; i >= 0; --i) ch = cm[i] == best ? i : ch;
      unsigned c = 0xffffffffu;
      float y[V];
      int at = 0;
      if (ch >= 0) {
#pragma unroll
        for (int e = 0; e < V; e += 4) *reinterpret_cast<f32x4*>(&y[e]) = *reinterpret_cast<const f32x4*>(&keep[ch][threadIdx.x][e]);
#pragma unroll
        for (int e = V - 1; e >= 0; --e) at = y[e] == best ? e : at;
        const int first = (ch * G + l) * V;
        c = (unsigned)((SHORT && a.C < V ? first : min(first, a.C - V)) + at);
      }
      const unsigned lowest = group_umin<G>(c);
      if (c == lowest) {
        float nm = NAN;
#pragma unroll
        for (int e = 0; e < V; ++e) nm = fmaxf(nm, e == at ? NAN : y[e]);
#pragma unroll
        for (int i = 0; i < NV; ++i) cm[i] = i == ch ? nm : cm[i];
        keep[ch][threadIdx.x][at] = NAN;
      }
      // G alternatives, one to a lane, are written together
      const int jl = j & (G - 1);
      kid = jl == l ? (int)lowest : kid;
      kv = jl == l ? best : kv;
      if ((jl == G - 1 || j == o.k - 1) && l <= jl) {
        o.top_ids[ot + (j - jl + l) * o.tk] = kid;
        o.top_lp[ot + (j - jl + l) * o.tk] = s == 0.f ? -INFINITY : (kv - base) * a.invT - ls;
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
// Bound by memory: 4096 x 50001 bf16, 16 alternatives: 96 us, 4.3 TB/s (a copy reaches 4.8); one row of 131072 in 32 slices: 8 us and 7.6
// for joining them.
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
  const long long ot = o.k ? row_at(a, r, o.tn, o.tp) : 0;
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
  RowSums sum;
  float lm = -INFINITY;
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
    float nm = sum.m;
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
        const int i = it + n;
        if (i < iters && ((i + 1) % t.join == 0 || i + 1 == iters)) {
          if ((tid & 7) == 0) line[(i / t.join) * 32 + g8] = order_key(lm);
          lm = -INFINITY;
        }
      }
    }
    const float base = sum.follow(nm, a.scale2);
    float gs = 0.f, gu = 0.f;
#pragma unroll
    for (int n = 0; n < UN; ++n)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = (x[n][e] - base) * a.scale2, w = exp2_(d);
        gs += w;
        gu += w * fmaxf(d, -300.f);
      }
    sum.add(gs, gu);
  }
  // join the lanes, then the waves
  const float wm = group_max<64>(sum.m);
  sum.settle(wm, a.scale2);
  float s = group_sum<64>(sum.s), u = group_sum<64>(sum.u);
  if (lane == 0) { red[0][wv] = wm; red[1][wv] = s; red[2][wv] = u; }
  if (tid == 0) nlines = ncand = 0;
  __syncthreads();
  const float m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3])), base = usable(m);
  s = u = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float sw = red[1][w], uw = red[2][w];
    rescale(sw, uw, red[0][w], base, a.scale2);
    s += sw;
    u += uw;
  }
  s = at_least_one(s);
  u = not_positive(u);
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
      top = group_max64<64>(top);
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
  extern __shared__ unsigned long long lists[];      // [k][64]: every slice's list, a column to a lane
  const int lane = threadIdx.x;
  const long long r = t.r0 + blockIdx.x;
  const long long y = o.label ? o.label[r] : 0;
  const long long ot = o.k ? row_at(a, r, o.tn, o.tp) : 0;
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
#pragma unroll 4
  for (int j = 0; j < o.k; ++j) lists[j * 64 + lane] = on ? keys[j] : 0;
  unsigned long long head = o.k ? lists[lane] : 0;
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
    const unsigned long long top = group_max64<64>(head);
    if (head == top) {
      ++at;
      head = at < o.k ? lists[at * 64 + lane] : 0;
    }
    if (lane == 0) {
      o.top_ids[ot + j * o.tk] = (int)~(unsigned)top;
      o.top_lp[ot + j * o.tk] = s == 0.f ? -INFINITY : (key_value((unsigned)(top >> 32)) - base) * a.invT - ls;
    }
  }
}

// Falling lists of the K best: order keys with their classes beside them (fp32), or key and class in one word: an fp32 value that was
// bf16 (fp16) leaves the 16 (13) last bits of its key to the class, counted down.  Classes come in rising order, so a key equal to one in
// the list goes behind it.  The median of (upper neighbour, entry, new key) is the entry's new key.  NaN is not looked for here: its row's
// sum tells of it, and its alternatives are taken once more.
__device__ __forceinline__ unsigned med3u(unsigned a, unsigned b, unsigned c) { return max(min(a, b), min(max(a, b), c)); }
__device__ __forceinline__ unsigned plain_key(float z) {
  const unsigned u = __float_as_uint(z + 0.f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
template <typename E> constexpr unsigned CLASS_BITS = 0;
template <> constexpr unsigned CLASS_BITS<__bf16> = 0xffffu;
template <> constexpr unsigned CLASS_BITS<_Float16> = 0x1fffu;
template <typename E, int K>
struct Best {
  static constexpr unsigned BITS = CLASS_BITS<E>;
  unsigned key[K > 0 ? K : 1];
  int id[K > 0 && BITS == 0 ? K : 1];
  __device__ __forceinline__ Best() {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      key[j] = 0;
      if constexpr (BITS == 0) id[j] = 0;
    }
  }
  __device__ __forceinline__ void add_key(unsigned k, int c) {
#pragma unroll
    for (int j = K - 1; j > 0; --j) {
      if constexpr (BITS == 0) id[j] = k > key[j - 1] ? id[j - 1] : k > key[j] ? c : id[j];
      key[j] = med3u(key[j - 1], key[j], k);
    }
    if constexpr (BITS == 0) id[0] = k > key[0] ? c : id[0];
    key[0] = max(key[0], k);
  }
  __device__ __forceinline__ void add(float z, int c) { add_key((plain_key(z) & ~BITS) | (BITS - (BITS ? (unsigned)c : 0u)), c); }
  __device__ __forceinline__ float value(int j) const { return key_value(BITS == 0 ? key[j] : key[j] & 0x80000000u ? key[j] & ~BITS : key[j] | BITS); }
  __device__ __forceinline__ int cls(int j) const { return BITS ? (int)(BITS - (key[j] & BITS)) : id[j]; }
};

constexpr int PLANE_K = 32;
template <typename E> constexpr int PLANE_CLASSES = CLASS_BITS<E> ? (int)CLASS_BITS<E> + 1 : 65536;

// One pass over a pixel's classes with a running maximum, 8 classes at a time, the lists beside it.  SPLIT = 4: a block's four waves share
// 64 * PV pixels and take a quarter of the classes each (images too small to fill the device).  Bound by memory up to a few alternatives:
// 8 x 150 x 473 x 473 fp32: 210 us without any (5.1 TB/s), 236 with 3; by the lists' instructions beyond: 334 with 8, 582 with 16, 939 with
// 32.  2 x 19 x 713 x 713 bf16, 3 alternatives: 21 us, 3.9 TB/s, memory and instructions alike.
template <typename E, int PV, int K, int SPLIT>
__global__ __launch_bounds__(256) void logprobs_planes_kernel(const Logits a, const LogprobOut o, const long long i0, const int tiles) {
  using B = Best<E, K>;
  constexpr bool IDS = B::BITS == 0 && K > 0;
  // The label's logit is kept as it comes by (fp32), or fetched afterwards (16 bits): the one costs two instructions a logit, the other a
  // memory line a pixel.  8 x 150 x 473 x 473 fp32: 6 % less time than the other way; 2 x 19 x 713 x 713 bf16, whose two pixels to a lane
  // leave no instructions to spare: 14 % more.
  constexpr bool ZY = sizeof(E) == 4;
  constexpr int LANES = 256 / SPLIT, UN = 8;
  __shared__ float red[SPLIT > 1 ? SPLIT - 1 : 1][4][PV][SPLIT > 1 ? 64 : 1];
  __shared__ unsigned lists[SPLIT > 1 ? SPLIT - 1 : 1][K > 0 ? K : 1][PV][SPLIT > 1 ? 64 : 1];
  __shared__ int ids[SPLIT > 1 && IDS ? SPLIT - 1 : 1][K > 0 ? K : 1][PV][SPLIT > 1 && IDS ? 64 : 1];
  const int wv = SPLIT > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0, pl = threadIdx.x & (LANES - 1);
  unsigned image, at;
  tile_of(blockIdx.x, tiles, image, at);      // reads alone, 1 KB a block: with neighbours on one XCD 3 % more time
  const long long i = i0 + image;
  const Px<PV> px((long long)at * (LANES * PV), pl, a.p);
  const E* zt = (const E*)a.z + i * a.sn + px.base;
  const unsigned bytes = px.template bytes<E>();
  const E* z = zt + (px.px - px.base);
  const int per = (a.C + SPLIT - 1) / SPLIT, c0 = wv * per, c1 = min(a.C, c0 + per);
  RowSums sum[PV];
  float zy[PV];
  int yc[PV];
  B best[PV];
#pragma unroll
  for (int v = 0; v < PV; ++v) {
    zy[v] = 0.f;
    if (ZY) {
      const long long y = o.logprob ? o.label[i * a.p + px.px + v] : -1;
      yc[v] = y >= 0 && y < a.C ? (int)y : -1;
    }
  }
  // The next classes are on their way while these are worked on: an image's waves are all resident at once, and without it they all wait
  // for memory at the same time.
  const auto load = [&](E(&q)[UN][PV], int c) {
#pragma unroll
    for (int n = 0; n < UN; ++n) load_px<E, PV>(zt + min(c + n, c1 - 1) * a.sc, bytes, q[n]);
  };
  const auto work = [&](const E(&q)[UN][PV], int c) {
    float x[UN][PV];
#pragma unroll
    for (int n = 0; n < UN; ++n)
#pragma unroll
      for (int v = 0; v < PV; ++v) x[n][v] = (float)q[n][v];
    if (c + UN > c1) {
#pragma unroll
      for (int n = 0; n < UN; ++n)
#pragma unroll
        for (int v = 0; v < PV; ++v) x[n][v] = c + n < c1 ? x[n][v] : -INFINITY;
    }
#pragma unroll
    for (int v = 0; v < PV; ++v) {
      float nm = sum[v].m;
#pragma unroll
      for (int n = 0; n < UN; ++n) nm = fmaxf(nm, x[n][v]);
      const float base = sum[v].follow(nm, a.scale2);
      float gs = 0.f, gu = 0.f;
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        const float d = (x[n][v] - base) * a.scale2, w = exp2_(d);
        gs += w;
        gu += w * fmaxf(d, -300.f);
      }
      sum[v].add(gs, gu);
    }
    if (ZY) {
#pragma unroll
      for (int n = 0; n < UN; ++n)
#pragma unroll
        for (int v = 0; v < PV; ++v) zy[v] = yc[v] == c + n ? x[n][v] : zy[v];
    }
    if (K > 0) {
#pragma unroll
      for (int n = 0; n < UN; ++n)
        if (c + n < c1) {
#pragma unroll
          for (int v = 0; v < PV; ++v) best[v].add(x[n][v], c + n);
        }
    }
  };
  E qa[UN][PV], qb[UN][PV];
  load(qa, c0);
  for (int c = c0; c < c1; c += 2 * UN) {
    if (c + UN < c1) load(qb, c + UN);
    work(qa, c);
    if (c + UN >= c1) break;
    if (c + 2 * UN < c1) load(qa, c + 2 * UN);
    work(qb, c + UN);
  }
  float m[PV], s[PV], u[PV];
#pragma unroll
  for (int v = 0; v < PV; ++v) {
    sum[v].settle(sum[v].m, a.scale2);
    m[v] = sum[v].m;
    s[v] = sum[v].s;
    u[v] = sum[v].u;
  }
  if constexpr (SPLIT > 1) {
    if (wv > 0) {
#pragma unroll
      for (int v = 0; v < PV; ++v) {
        red[wv - 1][0][v][pl] = m[v];
        red[wv - 1][1][v][pl] = s[v];
        red[wv - 1][2][v][pl] = u[v];
        if (ZY) red[wv - 1][3][v][pl] = zy[v];
#pragma unroll
        for (int j = 0; j < K; ++j) {
          lists[wv - 1][j][v][pl] = best[v].key[j];
          if constexpr (IDS) ids[wv - 1][j][v][pl] = best[v].cls(j);
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
        const int lo = (w + 1) * per;
        if (ZY) zy[v] = yc[v] >= lo && yc[v] < min(a.C, lo + per) ? red[w][3][v][pl] : zy[v];
        if (K > 0) {
          for (int j = 0; j < K; ++j) {        // the other waves' classes are higher: equal keys stay behind
            const unsigned k = lists[w][j][v][pl];
            int id = 0;
            if constexpr (IDS) id = ids[w][j][v][pl];
            best[v].add_key(k, id);
          }
        }
      }
    }
  }
  if (px.p0 >= a.p) return;
  const long long r = i * a.p + px.px, ot = i * o.tn + px.px * o.tp;
  float base[PV], ls[PV], out[PV];
  bool empty[PV], is_class[PV];
  long long y[PV];
#pragma unroll
  for (int v = 0; v < PV; ++v) {
    y[v] = o.label ? o.label[r + v] : 0;
    empty[v] = o.label && y[v] == o.ignore;
    is_class[v] = y[v] >= 0 && y[v] < a.C;
    base[v] = usable(m[v]);
    s[v] = at_least_one(s[v]);
    u[v] = not_positive(u[v]);
    ls[v] = log2_(s[v]) * LN2;
  }
  if (o.logprob) {
#pragma unroll
    for (int v = 0; v < PV; ++v) {
      if (!ZY) zy[v] = is_class[v] && !empty[v] ? load1(z + y[v] * a.sc + v) : 0.f;
      out[v] = empty[v] ? 0.f : !is_class[v] ? NAN : s[v] == 0.f ? -INFINITY : (zy[v] - base[v]) * a.invT - ls[v];
    }
    px.put(o.logprob + r, 1, out);
  }
  if (o.entropy) {
#pragma unroll
    for (int v = 0; v < PV; ++v) out[v] = empty[v] || s[v] == 0.f ? 0.f : ls[v] - u[v] / s[v] * LN2;
    px.put(o.entropy + r, 1, out);
  }
  if (o.lse) {
#pragma unroll
    for (int v = 0; v < PV; ++v) out[v] = empty[v] ? 0.f : base[v] * a.invT + ls[v];
    px.put(o.lse + r, 1, out);
  }
  if (o.stats) {
#pragma unroll
    for (int v = 0; v < PV; ++v) out[v] = empty[v] ? 0.f : base[v];
    px.put(o.stats + r, 1, out);
#pragma unroll
    for (int v = 0; v < PV; ++v) out[v] = empty[v] ? 0.f : ls[v];
    px.put(o.stats + a.R + r, 1, out);
  }
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (j < o.k) {
      int id[PV];
#pragma unroll
      for (int v = 0; v < PV; ++v) {
        id[v] = empty[v] ? -1 : best[v].cls(j);
        out[v] = empty[v] || s[v] == 0.f ? -INFINITY : (best[v].value(j) - base[v]) * a.invT - ls[v];
      }
      px.put(o.top_ids + ot + j * o.tk, o.tp, id);
      px.put(o.top_lp + ot + j * o.tk, o.tp, out);
    }
  if (K > 0) {
#pragma unroll
    for (int v = 0; v < PV; ++v)
      if (s[v] != s[v] && !empty[v] && px.own(v)) {      // a NaN or +inf: the alternatives once more
        unsigned long long prev = ~0ull;
        for (int j = 0; j < o.k; ++j) {
          unsigned long long top = 0;
          for (int c = 0; c < a.C; ++c) {
            const unsigned long long key = pair_key(load1(z + c * a.sc + v), c);
            top = key < prev && key > top ? key : top;
          }
          prev = top;
          o.top_ids[ot + v * o.tp + j * o.tk] = (int)~(unsigned)top;
        }
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
  __device__ __forceinline__ void init(const Logits& a, const LogprobGrad& g, long long r) {
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

// Contiguous classes: G lanes to a row (8, 64) or a block to a segment of SEG chunks a lane; one read, one write, no reductions.  Bound by
// memory: 4096 x 32000 bf16: 84 us, 6.3 TB/s (part of what the forward pass read is still in the last-level cache).
template <typename E, int G>
__global__ __launch_bounds__(256) void logprobs_bwd_rows_kernel(const Logits a, const LogprobGrad g) {
  constexpr int V = VEC<E>, SEG = 4;
  const int l = threadIdx.x % G;
  const int seg = blockIdx.x;              // G < 256: 0
  const long long step = (long long)gridDim.y * (256 / G);
  for (long long r = (long long)blockIdx.y * (256 / G) + threadIdx.x / G; r < a.R; r += step) {
    RowGrad f;
    f.init(a, g, r);
    const E* z = (const E*)a.z + a.at(r);
    E* dz = (E*)g.dz + row_at(a, r, g.dn, g.dp);
    const int c1 = G == 256 ? min(a.C, (seg + 1) * (SEG * G * V)) : a.C;
    for (int c0 = G == 256 ? seg * (SEG * G * V) : 0; c0 < c1; c0 += SEG * G * V) {
      Vec<E> q[SEG], old[SEG];
      int b[SEG];
#pragma unroll
      for (int i = 0; i < SEG; ++i) {
        b[i] = load_raw<G == 8>(z, c0 + (i * G + l) * V, a.C, q[i]);
        if (g.accumulate) load_raw<G == 8>((const E*)dz, c0 + (i * G + l) * V, a.C, old[i]);
      }
#pragma unroll
      for (int i = 0; i < SEG; ++i) {
        const int c = c0 + (i * G + l) * V;
        if (c >= c1) break;
        float x[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = f(a, (float)q[i][e], b[i] + e) + (g.accumulate ? (float)old[i][e] : 0.f);
        store_chunk(dz, c, b[i], a.C, x);
      }
    }
  }
}

// Planes: PV pixels and a slice of the classes to a lane.  Bound by memory: 4 x 21 x 473 x 473 fp32: 28 us, 6.3 TB/s (part of what the
// forward pass read is still in the last-level cache).
template <typename E, int PV>
__global__ __launch_bounds__(256) void logprobs_bwd_planes_kernel(const Logits a, const LogprobGrad g, const long long i0, const int tiles,
                                                                  const int slice) {
  constexpr int UN = 4;
  unsigned image, at;
  tile_of(xcd_remap(blockIdx.x, gridDim.x), tiles, image, at);
  const long long i = i0 + image;
  const Px<PV> px((long long)at * (256 * PV), threadIdx.x, a.p);
  if (px.p0 >= a.p) return;
  const E* z = (const E*)a.z + i * a.sn + px.base;
  E* dz = (E*)g.dz + i * g.dn + px.base;
  const unsigned bytes = px.template bytes<E>();
  RowGrad f[PV];
#pragma unroll
  for (int v = 0; v < PV; ++v) f[v].init(a, g, i * a.p + px.px + v);
  const int c0 = blockIdx.y * slice, c1 = min(a.C, c0 + slice);
  for (int c = c0; c < c1; c += UN) {
    E q[UN][PV], old[UN][PV];
#pragma unroll
    for (int n = 0; n < UN; ++n) {
      load_px<E, PV>(z + min(c + n, c1 - 1) * a.sc, bytes, q[n]);
      if (g.accumulate) load_px<E, PV>(dz + min(c + n, c1 - 1) * g.dc, bytes, old[n]);
    }
#pragma unroll
    for (int n = 0; n < UN; ++n) {
      if (c + n >= c1) break;
#pragma unroll
      for (int v = 0; v < PV; ++v) q[n][v] = (E)(f[v](a, (float)q[n][v], c + n) + (g.accumulate ? (float)old[n][v] : 0.f));
      if (px.own(0)) {
        store_px<E, PV>(dz + (c + n) * g.dc, bytes, q[n]);
      } else {
#pragma unroll
        for (int v = 1; v < PV; ++v)
          if (px.own(v)) store_at(dz + (c + n) * g.dc + v, bytes, q[n][v]);
      }
    }
  }
}

int row_blocks(long long R) {
  const long long b = (R + 3) / 4;
  return (int)(b < 8192 ? b : 8192);
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
    const int pv = a.p >= PV ? PV : 1;
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
  if (a.C <= 256) logprobs_bwd_rows_kernel<E, 8><<<dim3(1, capped((a.R + 31) / 32, 65535)), 256, 0, stream>>>(a, g);
  else if (a.C <= 4 * 64 * VEC<E>) logprobs_bwd_rows_kernel<E, 64><<<dim3(1, capped((a.R + 3) / 4, 65535)), 256, 0, stream>>>(a, g);
  else logprobs_bwd_rows_kernel<E, 256><<<seg_grid(a.R, a.C, 4 * 256 * VEC<E>), 256, 0, stream>>>(a, g);
}

template <typename E>
void logprobs_fwd(const Logits& a, const LogprobOut& o, int type, void* scratch, hipStream_t stream) {
  if (a.C > 1 && a.sc != 1) {
    if (o.k > PLANE_K || a.C > PLANE_CLASSES<E>) {
      logprobs_fwd_kernel<E><<<row_blocks(a.R), 256, 0, stream>>>(a, o);
    } else {
      logprobs_planes<E>(a, o, stream);
    }
    return;
  }
  if (a.C <= ROW_CLASSES) {
    const int chunks = (a.C + VEC<E> - 1) / VEC<E>;
#define ROWS(G, NV)                                                                        \
  do {                                                                                      \
    const int blocks = capped((a.R + 256 / G - 1) / (256 / G), 16384);                       \
    if (o.k) logprobs_rows_kernel<E, G, NV, true><<<blocks, 256, 0, stream>>>(a, o);         \
    else logprobs_rows_kernel<E, G, NV, false><<<blocks, 256, 0, stream>>>(a, o);            \
  } while (0)
    constexpr bool W4 = VEC<E> == 4;
    if (chunks <= 4) ROWS(4, 1);
    else if (chunks <= 8) ROWS(4, 2);
    else if (chunks <= 12) ROWS(4, 3);
    else if (chunks <= 20) ROWS(4, 5);
    else if (W4 && chunks <= 40) ROWS(4, W4 ? 10 : 1);           // a form that only the other type reaches names one of this type's
    else if (chunks <= (W4 ? 64 : 32)) ROWS(8, W4 ? 8 : 4);      // 256 classes
    else if (!W4 && chunks <= 64) ROWS(64, W4 ? 2 : 1);
    else if (chunks <= 128) ROWS(64, 2);
    else if (chunks <= 256) ROWS(64, 4);
    else ROWS(64, W4 ? 8 : 1);
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
    if (s.nsplit > 1) logprobs_join_kernel<E><<<rows, 64, o.k * 64 * sizeof(unsigned long long), stream>>>(a, o, t);
  }
}

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
  if (!layout_ok(C, n, p, sp, sc)) return SEMSEG_EINVAL;
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
  if (!layout_ok(C, n, p, sp, sc) || !(C == 1 || (sc == 1 ? dc == 1 : dp == 1))) return SEMSEG_EINVAL;
  const Logits a = logits_of(z, n, p, C, sn, sp, sc, T);
  const LogprobGrad g{label, ignore_index, stats, entropy, g_logprob, g_entropy, g_lse, dz, dn, dp, dc, accumulate};
  BY_TYPE(type, logprobs_bwd, a, g, stream);
  return semseg_launch_status();
}

}  // extern "C"
