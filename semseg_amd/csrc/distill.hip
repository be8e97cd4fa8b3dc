// Distillation from a teacher's stored top logits: the loss T^2 mean_w KL(teacher || student) over the rows of a student's logits, its
// gradient, and both at once (class_probs.h: how rows lie in memory, and the softmax statistics).
//   q = softmax(top / T) over a row's entries (or q = exp(top) and q_rest = 1 - sum q for everything else), p = softmax(z / T)
//   loss = sum_j q_j (log q_j - log p_{id_j}) [+ q_rest (log q_rest - log p_rest)]
#include "class_probs.h"

namespace {

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
  // ids and values on their way, before anything else of the row is waited for
  long long c_[NE];
  __device__ __forceinline__ RowTeacher(const Teacher& t, const Logits& a, long long r, int l) {
    const long long io = row_at(a, r, t.in, t.ip), vo = row_at(a, r, t.vn, t.vp);
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int j = i * TG + l;
      c_[i] = -1;
      lq[i] = -INFINITY;
      if (j < t.k) {
        c_[i] = t.id(io, j);
        lq[i] = t.value(vo, j);
      }
    }
  }
  __device__ __forceinline__ void classes(const Logits& a) {
    unsigned flags = 0;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      if (c_[i] >= a.C) flags |= 2u;
      id[i] = c_[i] >= 0 && c_[i] < a.C ? (int)c_[i] : -1;
      if (id[i] >= 0) flags |= 1u;
      else lq[i] = -INFINITY;
    }
    flags = group_reduce<TG>(flags, [](unsigned x, unsigned y) { return x | y; });
    any = flags & 1u;
    bad = flags & 2u;
  }
  __device__ __forceinline__ void softmax(const Teacher& t, const Logits& a) {
    float s = 0.f;
    if (t.tail) {
#pragma unroll
      for (int i = 0; i < NE; ++i) s += q[i] = exp2_(lq[i] * LOG2E);
      qsum = group_sum<TG>(s);
      qrest = fmaxf(1.f - qsum, 0.f);
    } else {
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < NE; ++i) m = fmaxf(m, lq[i]);
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
  // sums of q over all entries of each element's class; what the other lanes hold comes by shuffles, once for all elements
  __device__ __forceinline__ void of_class(int k, float (&sum)[NE]) const {
#pragma unroll
    for (int i = 0; i < NE; ++i) sum[i] = 0.f;
#pragma unroll
    for (int n = 0; n < NE; ++n)
      if (n * TG < k)
        for (int src = 0; src < TG; ++src) {
          const int o = __shfl(id[n], src, TG);
          const float v = __shfl(q[n], src, TG);
#pragma unroll
          for (int i = 0; i < NE; ++i) sum[i] += o == id[i] ? v : 0.f;
          if (n * TG + src + 1 >= k) break;
        }
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

// Rows of at most 2048 contiguous classes: G lanes hold a row in registers (8 up to 256 classes; 4 lanes to a row save instructions, but
// what bounds this kernel is the way from the entries' ids to the logits gathered there, and with them fewer waves share it: 57600 x 150,
// k 8: 26.8 us, with 8 lanes 21; with the ids fetched before the logits 20, where 73 MB would take 10.4; k 32: 42, k 64: 58).  GRAD: loss and gradient from
// one read of the logits.
template <typename E, int G, int NV, int NE, bool GRAD, bool TAIL>
__global__ __launch_bounds__(256) void distill_rows_kernel(const Logits a, const Teacher t, const DistillOut o, const DistillGrad g) {
  constexpr int V = VEC<E>;
  constexpr bool SHORT = G < 64 && NV == 1;
  const int l = threadIdx.x % G;
  const long long step = (long long)gridDim.x * (256 / G);
  double loss = 0.0, wsum = 0.0;
  for (long long r = (long long)blockIdx.x * (256 / G) + threadIdx.x / G; r < a.R; r += step) {
    const float w = t.weight ? t.weight[r] : 1.f;
    E* dz = GRAD ? (E*)g.dz + row_at(a, r, g.dn, g.dp) : nullptr;
    bool dead = w == 0.f;
    if (!dead) {
      const E* z = (const E*)a.z + a.at(r);
      RowTeacher<G, NE> q(t, a, r, l);
      float x[NV][V];
      int b[NV];
      load_chunks<NV, SHORT>(z, l * V, G * V, a.C, x, b);
      q.classes(a);
      float zj[NE];
#pragma unroll
      for (int i = 0; i < NE; ++i) zj[i] = q.id[i] >= 0 ? load1(z + q.id[i]) : -INFINITY;
      q.softmax(t, a);
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) m = fmaxf(m, x[i][e]);
      m = group_max<G>(m);
      const float base = m == -INFINITY ? 0.f : m;
      float s = 0.f, st = 0.f;
      unsigned in = 0;             // of the lane's NV * V logits: those of the teacher's classes
      if (TAIL) {
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
          if (TAIL) st += in >> (i * V + e) & 1u ? 0.f : p;
        }
      s = group_sum<G>(s);
      const float ls = log2_(s) * LN2;
      float lpt = 0.f, rbase = base, rsum = s;
      bool rest = false;
      if (TAIL) {
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
          o.stats[2 * a.R + r] = TAIL && !rest ? INFINITY : lpt;
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
          float fix[NE], sum[NE];
          q.of_class(t.k, sum);
#pragma unroll
          for (int i = 0; i < NE; ++i) {
            fix[i] = 0.f;
            if (i * G < t.k) {
              fix[i] = coef * (Q * exp2_(zj[i] * LOG2E) - sum[i]);
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

// Longer rows: every block streams a slice and leaves its maximum and sum (with a tail: of the classes outside the entries.  A byte for
// every 16-byte chunk says which of its classes the teacher names, a bit for every load of a wave whether one of its chunks has any, so
// that most loads are done with a scalar test: 2048 x 131072 bf16, k 32: 160 us with a look at LDS for every chunk) ...
constexpr int MAP_CHUNKS = 16384;
struct DStream {
  long long r0;
  int nsplit, slice;
  float* part;               // [R][nsplit][2]
};
template <typename E, bool TAIL>
__global__ __launch_bounds__(256) void distill_stream_kernel(const Logits a, const Teacher t, const DStream d) {
  constexpr int V = VEC<E>, UN = 4;
  __shared__ unsigned map[TAIL ? MAP_CHUNKS / 4 : 1];
  __shared__ unsigned loads[4][2];           // of a wave: bit it of [it / 32]
  __shared__ float red[2][4];
  const int tid = threadIdx.x;
  const int sp = (int)(blockIdx.x % (unsigned)d.nsplit);
  const long long r = d.r0 + blockIdx.x / (unsigned)d.nsplit;
  if (t.weight && t.weight[r] == 0.f) return;
  const E* z = (const E*)a.z + a.at(r);
  int id = -1;
  if (TAIL && tid < t.k) {
    const long long c = t.id(row_at(a, r, t.in, t.ip), tid);
    id = c >= 0 && c < a.C ? (int)c : -1;
  }
  const int first = sp * d.slice, last = min(a.C, first + d.slice);
  float m = -INFINITY, b = -INFINITY, s = 0.f, lost = 0.f;      // maximum, base of the sum, sum, what it lost
  constexpr int TURN = TAIL ? MAP_CHUNKS * V : 1 << 30;
  for (int c0 = first; c0 < last; c0 += TURN) {
    const int c1 = last - c0 > TURN ? c0 + TURN : last;
    const int iters = (c1 - c0 + 256 * V - 1) / (256 * V);
    unsigned long long named = 0;
    if (TAIL) {
      __syncthreads();
      for (int i = tid; i < iters * 64; i += 256) map[i] = 0;
      if (tid < 8) loads[tid >> 1][tid & 1] = 0;
      __syncthreads();
      if (id >= c0 && id < c1) {
        const int ch = (id - c0) / V, c = c0 + ch * V, e = id - min(c, a.C - V);      // e: where load_chunk has it
        atomicOr(&map[ch >> 2], 1u << ((ch & 3) * 8 + e));
        atomicOr(&loads[(ch >> 6) & 3][ch >> 13], 1u << ((ch >> 8) & 31));
      }
      __syncthreads();
      named = (unsigned long long)__builtin_amdgcn_readfirstlane(loads[tid >> 6][1]) << 32 |
              (unsigned)__builtin_amdgcn_readfirstlane(loads[tid >> 6][0]);
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
      if (TAIL && (named >> it & 15u)) {
#pragma unroll
        for (int n = 0; n < UN; ++n)
          if (named >> (it + n) & 1u) {
            const int ch = (it + n) * 256 + tid;
            const unsigned in = map[ch >> 2] >> ((ch & 3) * 8);
#pragma unroll
            for (int e = 0; e < V; ++e) x[n][e] = in >> e & 1u ? -INFINITY : x[n][e];
          }
      }
      float nm = m;
#pragma unroll
      for (int n = 0; n < UN; ++n)
#pragma unroll
        for (int e = 0; e < V; ++e) nm = fmaxf(nm, x[n][e]);
      m = nm;
      const bool mv = must_move(m, b, a.scale2);
      if (__any(mv)) {
        const float to = mv ? m : b, f = exp2_((b - usable(to)) * a.scale2);
        s *= f;
        lost *= f;
        b = to;
      }
      const float base = usable(b);
      float gs = 0.f;
#pragma unroll
      for (int n = 0; n < UN; ++n)
#pragma unroll
        for (int e = 0; e < V; ++e) gs += exp2_((x[n][e] - base) * a.scale2);
      add_group(s, lost, gs);
    }
  }
  const float wm = group_max<64>(m);
  s = group_sum<64>(s * exp2_((b - usable(wm)) * a.scale2));
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
// ... and one wave a row joins them, adds the entries' logits and takes the loss.  2048 x 131072 bf16, k 32 with a tail: 120 us (4.5 TB/s)
// and 9.
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
    RowTeacher<64, 1> q(t, a, r, lane);
    q.classes(a);
    q.softmax(t, a);
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
    s = at_least_one(group_sum<64>(s));
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

// The gradient from the forward call's statistics: G lanes to a row (8, 64), or a block to a segment of SEG chunks a lane.  Bound by
// memory: 2048 x 131072 bf16: 210 us, 5.1 TB/s.
template <typename E, int G, int NE>
__global__ __launch_bounds__(256) void distill_bwd_rows_kernel(const Logits a, const Teacher t, const DistillGrad g) {
  constexpr int V = VEC<E>, SEG = 4, TG = G < 64 ? G : 64;
  const int l = threadIdx.x % G;
  const int seg = blockIdx.x;              // G < 256: 0
  const long long step = (long long)gridDim.y * (256 / G);
  for (long long r = (long long)blockIdx.y * (256 / G) + threadIdx.x / G; r < a.R; r += step) {
    const float w = t.weight ? t.weight[r] : 1.f, base = g.stats[r], ls = g.stats[a.R + r], lpt = g.stats[2 * a.R + r];
    E* dz = (E*)g.dz + row_at(a, r, g.dn, g.dp);
    const int c0 = G == 256 ? seg * (SEG * G * V) : 0, c1 = G == 256 ? min(a.C, c0 + SEG * G * V) : a.C;
    RowTeacher<TG, NE> q(t, a, r, threadIdx.x % TG);
    q.classes(a);
    q.softmax(t, a);
    const bool dead = w == 0.f || q.bad || !q.any || ls == -INFINITY;
    const E* z = (const E*)a.z + a.at(r);
    const bool rest = t.tail && lpt != INFINITY;
    const float coef = g.coef(r, w), Q = rest ? q.qsum + q.qrest : q.qsum;
    const float off = rest ? ls + lpt : ls, f = coef * (rest ? Q * exp2_(lpt * LOG2E) - q.qrest : Q);
    float fix[NE], sum[NE];
    bool mine[NE], named = false;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      mine[i] = !dead && q.id[i] >= c0 && q.id[i] < c1 && (G < 256 || threadIdx.x < 64);
      named |= mine[i];
    }
    if (__any(named)) {                  // most segments of a long row hold no entry
      q.of_class(t.k, sum);
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (mine[i]) {
          fix[i] = coef * (Q * exp2_(((load1(z + q.id[i]) - base) * a.invT - ls) * LOG2E) - sum[i]);
          if (g.accumulate) fix[i] += load1(dz + q.id[i]);
        }
    }
    if (G == 256) __syncthreads();       // with accumulate: the entries' old values are read before the row is written
    if (dead) {
      if (!g.accumulate) {
        float x[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = 0.f;
        for (int c = c0 + l * V; c < c1; c += G * V) store_chunk(dz, c, G == 8 && a.C < V ? c : min(c, a.C - V), a.C, x);
      }
    } else {
      for (int cs = c0; cs < c1; cs += SEG * G * V) {
        Vec<E> q[SEG], old[SEG];
        int b[SEG];
#pragma unroll
        for (int i = 0; i < SEG; ++i) {
          b[i] = load_raw<G == 8>(z, cs + (i * G + l) * V, a.C, q[i]);
          if (g.accumulate) load_raw<G == 8>((const E*)dz, cs + (i * G + l) * V, a.C, old[i]);
        }
#pragma unroll
        for (int i = 0; i < SEG; ++i) {
          const int c = cs + (i * G + l) * V;
          if (c >= c1) break;
          float x[V];
#pragma unroll
          for (int e = 0; e < V; ++e)
            x[e] = f * exp2_(((float)q[i][e] - base) * a.scale2 - off * LOG2E) + (g.accumulate ? (float)old[i][e] : 0.f);
          store_chunk(dz, c, b[i], a.C, x);
        }
      }
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

// ---- planes.  A lane walks through all classes of its PV pixels, CH at a time, and needs its own teacher's classes on the way: the CH
// logits (forward) or q (backward) lie in the lane's own columns of a small LDS tile, where an entry's class is found by its number (no
// other lane touches them: no barrier, no conflict).  That is one LDS access per logit instead of k comparisons.
constexpr int CH = 16;

// The teacher of one pixel; KR > 0: k <= KR entries, kept in registers, 0: read again whenever they are needed.
template <int KR>
struct PixTeacher {
  float m, ls, qsum, qrest, qlogq;
  bool any, bad, none;
  int id_[KR > 0 ? KR : 1];
  float q_[KR > 0 ? KR : 1];
  __device__ __forceinline__ float logq(const Teacher& t, const Logits& a, float v) const { return t.tail ? v : (v - m) * a.invT - ls; }
  // f(class, value or q) for every entry present
  template <typename F>
  __device__ __forceinline__ void each(const Teacher& t, const Logits& a, long long io, long long vo, F f) {
    if constexpr (KR > 0) {
#pragma unroll
      for (int j = 0; j < KR; ++j)
        if (id_[j] >= 0) f(id_[j], q_[j]);
    } else {
      for (int j = 0; j < t.k; ++j) {
        const long long c = t.id(io, j);
        if (c >= 0 && c < a.C) {
          float v = t.value(vo, j);
          f((int)c, v);
        }
      }
    }
  }
  __device__ __forceinline__ void init(const Teacher& t, const Logits& a, long long io, long long vo) {
    bad = any = false;
    if constexpr (KR > 0) {
      long long c[KR];
#pragma unroll
      for (int j = 0; j < KR; ++j) {
        c[j] = j < t.k ? t.id(io, j) : -1;
        q_[j] = j < t.k ? t.value(vo, j) : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < KR; ++j) {
        bad |= c[j] >= a.C;
        id_[j] = c[j] < 0 || c[j] >= a.C ? -1 : (int)c[j];
      }
    } else {
      for (int j = 0; j < t.k; ++j) bad |= t.id(io, j) >= a.C;
    }
    m = -INFINITY;
    each(t, a, io, vo, [&](int, float& v) {
      any = true;
      m = fmaxf(m, v);
    });
    if (m == -INFINITY) m = 0.f;
    ls = 0.f;
    none = false;
    if (!t.tail) {
      float s = 0.f;
      each(t, a, io, vo, [&](int, float& v) { s += exp2_((v - m) * a.scale2); });
      none = s == 0.f;
      ls = none ? 0.f : log2_(s) * LN2;
    }
    qsum = qlogq = 0.f;
    each(t, a, io, vo, [&](int, float& v) {
      const float lq = logq(t, a, v);
      v = exp2_(lq * LOG2E);             // KR: from here on q stands in the value's place
      qlogq += v == 0.f ? 0.f : v * lq;
      qsum += v;
    });
    qrest = t.tail ? fmaxf(1.f - qsum, 0.f) : 0.f;
    if (!t.tail) qsum = none ? 0.f : 1.f;
  }
  // f(n, q) for every entry of class c0 + n, 0 <= n < CH
  template <typename F>
  __device__ __forceinline__ void in_chunk(const Teacher& t, const Logits& a, long long io, long long vo, int c0, F f) {
    each(t, a, io, vo, [&](int c, float& v) {
      if ((unsigned)(c - c0) < (unsigned)CH) f(c - c0, KR > 0 ? v : exp2_(logq(t, a, v) * LOG2E));
    });
  }
};

// Loss: S about the running maximum, the mass outside the entries about the same one, sum q d as it goes.  A wave has 64 * PV pixels;
// with SPLIT = 4 four waves share them and take a quarter of the classes each.  4 x 150 x 473 x 473 fp32, k 4: 122 to 159 us for 537 MB; k 8:
// 152.  Beyond 8 entries (KR = 0) they are read again with every CH classes: k 16: 562 us, k 64: 2107.
template <typename E, int PV, int KR, int SPLIT, bool TAIL>
__global__ __launch_bounds__(64 * SPLIT) void distill_planes_kernel(const Logits a, const Teacher t, const DistillOut o, const int tiles,
                                                                    const long long all) {
  constexpr int COLS = 64 * PV;
  __shared__ float tiles_s[SPLIT][CH][COLS];
  __shared__ float red[SPLIT > 1 ? SPLIT - 1 : 1][5][SPLIT > 1 ? COLS : 1];
  const int wv = SPLIT > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0, lane = threadIdx.x & 63;
  float(*tile)[COLS] = tiles_s[wv];
  const int per = SPLIT > 1 ? ((a.C + SPLIT - 1) / SPLIT + CH - 1) / CH * CH : a.C;
  const int c_lo = wv * per, c_hi = min(a.C, c_lo + per);
  double loss = 0.0, wsum = 0.0;
  for (long long it = xcd_remap(blockIdx.x, gridDim.x); it < all; it += gridDim.x) {
    unsigned image, at;
    tile_of((unsigned)it, tiles, image, at);
    const long long i = image;
    const Px<PV> px((long long)at * COLS, lane, a.p);
    const E* zt = (const E*)a.z + i * a.sn + px.base;
    const unsigned bytes = px.template bytes<E>();
    const E* z = zt + (px.px - px.base);
    const long long r0 = i * a.p + px.px, io = i * t.in + px.px * t.ip, vo = i * t.vn + px.px * t.vp;
    // maximum, base, sums about it and what they lost: all classes, those outside the entries, q (z - base) of the entries; q so far
    float m[PV], base[PV], s[PV], st[PV], dot[PV], lost_s[PV], lost_t[PV], lost_d[PV], qacc[PV];
    PixTeacher<KR> q[PV];
#pragma unroll
    for (int v = 0; v < PV; ++v) {
      q[v].init(t, a, io + v * t.ip, vo + v * t.vp);
      m[v] = base[v] = -INFINITY;
      s[v] = st[v] = dot[v] = lost_s[v] = lost_t[v] = lost_d[v] = qacc[v] = 0.f;
    }
    // everything of pixel v about the base `to`
    const auto move = [&](int v, float to) {
      const float f = exp2_((base[v] - usable(to)) * a.scale2);
      s[v] *= f;
      lost_s[v] *= f;
      if (TAIL) {
        st[v] *= f;
        lost_t[v] *= f;
      }
      if (qacc[v] != 0.f) {
        add_group(dot[v], lost_d[v], qacc[v] * (usable(base[v]) - usable(to)));
        if (!(fabsf(dot[v]) < INFINITY)) lost_d[v] = 0.f;      // an entry on a class of -inf: -inf stays
      }
      base[v] = to;
    };
    for (int c0 = c_lo; c0 < c_hi; c0 += CH) {
      E x[CH][PV];
#pragma unroll
      for (int n = 0; n < CH; ++n) load_px<E, PV>(zt + min(c0 + n, c_hi - 1) * a.sc, bytes, x[n]);
#pragma unroll
      for (int v = 0; v < PV; ++v) {
        float y[CH], nm = m[v];
#pragma unroll
        for (int n = 0; n < CH; ++n) {
          y[n] = c0 + n < c_hi ? (float)x[n][v] : -INFINITY;
          nm = fmaxf(nm, y[n]);
          tile[n][lane * PV + v] = y[n];
        }
        m[v] = nm;
        const bool mv = must_move(nm, base[v], a.scale2);
        if (__any(mv)) move(v, mv ? nm : base[v]);
        const float nb = usable(base[v]);
        unsigned in = 0;
        q[v].in_chunk(t, a, io + v * t.ip, vo + v * t.vp, c0, [&](int n, float qc) {
          in |= 1u << n;
          dot[v] += qc == 0.f ? 0.f : qc * (tile[n][lane * PV + v] - nb);
          qacc[v] += qc;
        });
        float gs = 0.f, gt = 0.f;
#pragma unroll
        for (int n = 0; n < CH; ++n) {
          const float p = exp2_((y[n] - nb) * a.scale2);
          gs += p;
          if (TAIL) gt += in >> n & 1u ? 0.f : p;
        }
        add_group(s[v], lost_s[v], gs);
        if (TAIL) add_group(st[v], lost_t[v], gt);
      }
    }
#pragma unroll
    for (int v = 0; v < PV; ++v) {
      move(v, m[v]);
      base[v] = usable(m[v]);
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
    if (px.p0 >= a.p) continue;
    float s0[PV], s1[PV], s2[PV], lr[PV];
#pragma unroll
    for (int v = 0; v < PV; ++v) {
      const float w = t.weight ? t.weight[r0 + v] : 1.f;
      s[v] = at_least_one(s[v]);
      const float ls = log2_(s[v]) * LN2;
      float lpt = 0.f, kl = s[v] == 0.f ? (q[v].qsum > 0.f ? INFINITY : 0.f) : q[v].qlogq - (dot[v] * a.invT - q[v].qsum * ls);
      bool rest = TAIL;
      if (TAIL) {
        lpt = log2_(st[v]) * LN2 - ls;
        if (st[v] < 1e-20f) {          // the rest is far below the row's maximum: once more, about its own
          float mt = -INFINITY, sum = 0.f, lost = 0.f;
          for (int c = 0; c < a.C; ++c) {
            const float y = load1(z + c * a.sc + v);
            bool in = false;
            for (int j = 0; j < t.k; ++j) in |= t.id(io + v * t.ip, j) == c;
            if (in || y == -INFINITY) continue;
            if (must_move(y, mt, a.scale2)) {
              const float f = exp2_((mt - y) * a.scale2);
              sum *= f;
              lost *= f;
              mt = y;
            }
            add_group(sum, lost, exp2_((y - mt) * a.scale2));
          }
          rest = mt != -INFINITY;
          lpt = rest ? (mt - base[v]) * a.invT + log2_(sum) * LN2 - ls : 0.f;
        }
        if (rest && q[v].qrest > 0.f) kl += q[v].qrest * (log2_(q[v].qrest) * LN2 - lpt);
      }
      if (!q[v].any) kl = 0.f;
      if (q[v].bad) kl = NAN;
      const bool on = w != 0.f;        // a masked row's logits have been read, but nothing of them goes on
      s0[v] = on ? base[v] : 0.f;
      s1[v] = on ? ls : 0.f;
      s2[v] = !on ? 0.f : TAIL && !rest ? INFINITY : lpt;
      lr[v] = on ? o.T2 * w * kl : 0.f;
      if (on && px.own(v)) {
        loss += (double)w * (double)kl;
        wsum += (double)w;
      }
    }
    px.put(o.stats + r0, 1, s0);
    px.put(o.stats + a.R + r0, 1, s1);
    px.put(o.stats + 2 * a.R + r0, 1, s2);
    if (o.rows) px.put(o.rows + r0, 1, lr);
  }
  block_part<64 * SPLIT>(o.part, loss, wsum);
}

// 4 x 150 x 473 x 473 fp32, k 4: 227 us, 4.7 TB/s.
// The tile holds -coef * q; with a tail a class of the teacher is marked in the word's last bit (half a step of fp32 at most).
template <typename E, int PV, int KR, bool TAIL>
__global__ __launch_bounds__(64) void distill_bwd_planes_kernel(const Logits a, const Teacher t, const DistillGrad g, const long long i0,
                                                                const int tiles, const int slice) {
  constexpr int COLS = 64 * PV, UN = 8;
  __shared__ float tile[CH][COLS];
  const int lane = threadIdx.x;
  unsigned image, at;
  tile_of(xcd_remap(blockIdx.x, gridDim.x), tiles, image, at);
  const long long i = i0 + image;
  const Px<PV> px((long long)at * COLS, lane, a.p);
  if (px.p0 >= a.p) return;
  const E* z = (const E*)a.z + i * a.sn + px.base;
  E* dz = (E*)g.dz + i * g.dn + px.base;
  const unsigned bytes = px.template bytes<E>();
  const long long r0 = i * a.p + px.px, io = i * t.in + px.px * t.ip, vo = i * t.vn + px.px * t.vp;
  PixTeacher<KR> q[PV];
  float base[PV], ls2[PV], off2[PV], cq[PV], f[PV], coef[PV];
  bool dead[PV];
#pragma unroll
  for (int v = 0; v < PV; ++v) {
    q[v].init(t, a, io + v * t.ip, vo + v * t.vp);
    const float w = t.weight ? t.weight[r0 + v] : 1.f, ls = g.stats[a.R + r0 + v], lpt = g.stats[2 * a.R + r0 + v];
    base[v] = g.stats[r0 + v];
    const bool rest = TAIL && lpt != INFINITY;
    const float Q = rest ? q[v].qsum + q[v].qrest : q[v].qsum;
    dead[v] = w == 0.f || q[v].bad || !q[v].any || ls == -INFINITY;
    coef[v] = g.coef(r0 + v, w);
    cq[v] = coef[v] * Q;
    ls2[v] = ls * LOG2E;
    off2[v] = rest ? (ls + lpt) * LOG2E : ls2[v];
    f[v] = coef[v] * (rest ? Q * exp2_(lpt * LOG2E) - q[v].qrest : Q);
  }
  const int c_lo = blockIdx.y * slice, c_hi = min(a.C, c_lo + slice);
  for (int c0 = c_lo; c0 < c_hi; c0 += CH) {
#pragma unroll
    for (int n = 0; n < CH; ++n)
#pragma unroll
      for (int v = 0; v < PV; ++v) tile[n][lane * PV + v] = 0.f;
#pragma unroll
    for (int v = 0; v < PV; ++v)
      q[v].in_chunk(t, a, io + v * t.ip, vo + v * t.vp, c0, [&](int n, float qc) {
        float* p = &tile[n][lane * PV + v];
        *p = TAIL ? __uint_as_float(__float_as_uint(*p - coef[v] * qc) | 1u) : *p - coef[v] * qc;
      });
    for (int h = 0; h < CH && c0 + h < c_hi; h += UN) {
      E x[UN][PV], old[UN][PV];
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        load_px<E, PV>(z + min(c0 + h + n, c_hi - 1) * a.sc, bytes, x[n]);
        if (g.accumulate) load_px<E, PV>(dz + min(c0 + h + n, c_hi - 1) * g.dc, bytes, old[n]);
      }
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        if (c0 + h + n >= c_hi) break;
#pragma unroll
        for (int v = 0; v < PV; ++v) {
          const float tv = tile[h + n][lane * PV + v], d = ((float)x[n][v] - base[v]) * a.scale2;
          const bool in = TAIL && (__float_as_uint(tv) & 1u);
          float y = TAIL ? (in ? cq[v] : f[v]) * exp2_(d - (in ? ls2[v] : off2[v])) + (in ? tv : 0.f) : f[v] * exp2_(d - off2[v]) + tv;
          if (dead[v]) y = 0.f;
          x[n][v] = (E)(y + (g.accumulate ? (float)old[n][v] : 0.f));
        }
        if (px.own(0)) {
          store_px<E, PV>(dz + (c0 + h + n) * g.dc, bytes, x[n]);
        } else {
#pragma unroll
          for (int v = 1; v < PV; ++v)
            if (px.own(v)) store_at(dz + (c0 + h + n) * g.dc + v, bytes, x[n][v]);
        }
      }
    }
  }
}

bool teacher_ok(const void* ids, int ids64, const void* top, int top_type, int k) {
  return ids && top && (ids64 == 0 || ids64 == 1) && top_type >= 0 && top_type <= 2 && k >= 1 && k <= MAXK;
}

// Blocks of the loss kernels: one partial sum each
constexpr int PARTS = 16384;
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
  const int rows = a.C > 256 ? 4 : 32;      // of a block: distill_rows_t's choice of lanes to a row
  return capped((a.R + rows - 1) / rows, PARTS);
}

template <typename E, bool GRAD, bool TAIL>
void distill_rows_t(const Logits& a, const Teacher& t, const DistillOut& o, const DistillGrad& g, int blocks, hipStream_t stream) {
  const int chunks = (a.C + VEC<E> - 1) / VEC<E>;
#define DROWS(G, NV, NE) distill_rows_kernel<E, G, NV, NE, GRAD, TAIL><<<blocks, 256, 0, stream>>>(a, t, o, g)
  constexpr bool W4 = VEC<E> == 4;
  // entries per lane: one, two or eight, each at the cost of all it could hold (57600 x 150 fp32, k 9: 21 us with two, 29 with eight; 64
  // lanes with an entry each 47)
#define DROWS8(NV) do { if (t.k <= 8) DROWS(8, NV, 1); else if (t.k <= 16) DROWS(8, NV, 2); else DROWS(8, NV, 8); } while (0)
  if (chunks <= 8) DROWS8(1);
  else if (chunks <= 16) DROWS8(2);
  else if (chunks <= 24) DROWS8(3);
  else if (W4 && chunks <= 40) DROWS8(W4 ? 5 : 1);
  else if (chunks <= (W4 ? 64 : 32)) DROWS8(W4 ? 8 : 4);
  else if (!W4 && chunks <= 64) DROWS(64, W4 ? 2 : 1, 1);
  else if (chunks <= 128) DROWS(64, 2, 1);
  else if (chunks <= 256) DROWS(64, 4, 1);
  else DROWS(64, W4 ? 8 : 1, 1);
#undef DROWS8
#undef DROWS
}
template <typename E, bool GRAD>
void distill_rows(const Logits& a, const Teacher& t, const DistillOut& o, const DistillGrad& g, int blocks, hipStream_t stream) {
  if (t.tail) distill_rows_t<E, GRAD, true>(a, t, o, g, blocks, stream);
  else distill_rows_t<E, GRAD, false>(a, t, o, g, blocks, stream);
}

// Loss and statistics; partial sums to o.part
template <typename E>
void distill_fwd(const Logits& a, const Teacher& t, const DistillOut& o, int type, float* scratch, hipStream_t stream) {
  long long all;
  int split;
  const int blocks = distill_blocks<E>(a, &all, &split);
  if (a.C > 1 && a.sc != 1) {
    constexpr int PV = sizeof(E) == 2 ? 2 : 1;
    const int pv = a.p >= PV ? PV : 1, tiles = (int)((a.p + 64 * pv - 1) / (64 * pv));
#define DPLANES(PV_, KR, SP)                                                                                              \
  do {                                                                                                                    \
    if (t.tail) distill_planes_kernel<E, PV_, KR, SP, true><<<blocks, 64 * SP, 0, stream>>>(a, t, o, tiles, all);         \
    else distill_planes_kernel<E, PV_, KR, SP, false><<<blocks, 64 * SP, 0, stream>>>(a, t, o, tiles, all);               \
  } while (0)
    if (PV > 1 && pv == 1) DPLANES(1, 0, 4);
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
  for (d.r0 = 0; d.r0 < a.R; d.r0 += most) {
    const int blocks = (int)(a.R - d.r0 < most ? a.R - d.r0 : most) * s.nsplit;
    if (t.tail) distill_stream_kernel<E, true><<<blocks, 256, 0, stream>>>(a, t, d);
    else distill_stream_kernel<E, false><<<blocks, 256, 0, stream>>>(a, t, d);
  }
  distill_join_kernel<E><<<blocks, 256, 0, stream>>>(a, t, o, d);
}

template <typename E>
void distill_bwd(const Logits& a, const Teacher& t, const DistillGrad& g, hipStream_t stream) {
  if (a.C > 1 && a.sc != 1) {
    // two pixels to a lane: 8 bytes a load and store of fp32 (4 x 150 x 473 x 473: 10 % less time than with one; four take 2 % less still, but
    // more on small images)
    constexpr int PV = 2;
    const int pv = a.p >= PV ? PV : 1;
    const long long tiles = (a.p + 64 * pv - 1) / (64 * pv), blocks = a.R / a.p * tiles;
    // slices of the classes until there are about 16 waves a compute unit
    const int tc = (a.C + CH - 1) / CH, slices = blocks >= 4096 ? 1 : (int)(4096 / blocks < tc ? 4096 / blocks : tc);
    const int slice = (tc + slices - 1) / slices * CH;
    by_images(a, tiles * slices, [&](long long i0, int n) {
      const dim3 grid(n * (unsigned)tiles, (a.C + slice - 1) / slice);
#define DPLANES(PV_, KR)                                                                                                      \
  do {                                                                                                                        \
    if (t.tail) distill_bwd_planes_kernel<E, PV_, KR, true><<<grid, 64, 0, stream>>>(a, t, g, i0, (int)tiles, slice);          \
    else distill_bwd_planes_kernel<E, PV_, KR, false><<<grid, 64, 0, stream>>>(a, t, g, i0, (int)tiles, slice);                \
  } while (0)
      if (pv != PV) DPLANES(1, 0);
      else if (t.k <= 4) DPLANES(PV, 4);
      else if (t.k <= 8) DPLANES(PV, 8);
      else DPLANES(PV, 0);
#undef DPLANES
    });
    return;
  }
  if (a.C <= 256 && t.k <= 8) distill_bwd_rows_kernel<E, 8, 1><<<dim3(1, capped((a.R + 31) / 32, 65535)), 256, 0, stream>>>(a, t, g);
  else if (a.C <= 256 && t.k <= 16) distill_bwd_rows_kernel<E, 8, 2><<<dim3(1, capped((a.R + 31) / 32, 65535)), 256, 0, stream>>>(a, t, g);
  else if (a.C <= 256) distill_bwd_rows_kernel<E, 8, 8><<<dim3(1, capped((a.R + 31) / 32, 65535)), 256, 0, stream>>>(a, t, g);
  else if (a.C <= 4 * 64 * VEC<E>) distill_bwd_rows_kernel<E, 64, 1><<<dim3(1, capped((a.R + 3) / 4, 65535)), 256, 0, stream>>>(a, t, g);
  else distill_bwd_rows_kernel<E, 256, 1><<<seg_grid(a.R, a.C, 4 * 256 * VEC<E>), 256, 0, stream>>>(a, t, g);
}

// Scratch of a distillation call: partial sums, then the slices' maxima and sums of long rows
size_t distill_need(int type, long long R, int C, long long sc) {
  size_t need = (size_t)PARTS * 2 * sizeof(double);
  if ((C == 1 || sc == 1) && C > ROW_CLASSES) need += (size_t)R * split_rows(type, R, C).nsplit * 2 * sizeof(float);
  return need;
}
float* distill_slices(void* scratch) { return (float*)((double*)scratch + 2 * PARTS); }

}  // namespace

extern "C" {

size_t semseg_distill_scratch_bytes(int type, long long n, long long p, int C, long long sc) {
  if (n <= 0 || p <= 0 || C <= 0) return 0;
  return distill_need(type, n * p, C, sc);
}

int semseg_distill_fwd(const void* z, int type, long long n, long long p, int C, long long sn, long long sp, long long sc, const void* ids,
                       int ids64, const void* top, int top_type, int k, long long in, long long ip, long long ik, long long vn,
                       long long vp, long long vk, const float* weight, float T, int tail, int reduction, float* rows, float* stats,
                       double* acc2, float* loss, void* scratch, size_t scratch_bytes, hipStream_t stream) {
  if (!logits_ok(z, type, n, p, C, T) || !layout_ok(C, n, p, sp, sc) || !teacher_ok(ids, ids64, top, top_type, k) || !stats || reduction < 0 ||
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
  if (!logits_ok(z, type, n, p, C, T) || !layout_ok(C, n, p, sp, sc) || !teacher_ok(ids, ids64, top, top_type, k) || !stats || !dz ||
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
