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
  return z != z ? 0xffffffffu : k;
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

struct Logits {
  const void* z;
  long long R, p, sn, sp, sc;
  int C;
  float invT, scale2;      // 1 / T, log2(e) / T
  __device__ __forceinline__ long long at(long long r) const { return (r / p) * sn + (r % p) * sp; }
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

// One wave per row, lanes along the classes: any strides.
template <typename E>
__global__ __launch_bounds__(256) void logprobs_fwd_kernel(const Logits a, const LogprobOut o) {
  const int lane = threadIdx.x & 63;
  const long long waves = (long long)gridDim.x * 4;
  for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.R; r += waves) {
    const E* z = (const E*)a.z + a.at(r);
    const long long y = o.label ? o.label[r] : 0;
    const long long ot = (r / a.p) * o.tn + (r % a.p) * o.tp;
    if (o.label && y == o.ignore) {            // a void row is not read
      if (lane == 0) {
        if (o.logprob) o.logprob[r] = 0.f;
        if (o.entropy) o.entropy[r] = 0.f;
        if (o.lse) o.lse[r] = 0.f;
        if (o.stats) o.stats[r] = o.stats[a.R + r] = 0.f;
      }
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
      const float d = (load1(z + c * a.sc) - base) * a.scale2, e = exp2f(d);
      s += e;
      u += e * fmaxf(d, -300.f);               // exp2(-300) = 0 in fp32; 0 * -inf would be NaN
    }
    s = wave_sum(s);
    u = wave_sum(u);
    const bool none = s == 0.f;                // every logit -inf
    const float ls = logf(s);
    if (lane == 0) {
      if (o.stats) { o.stats[r] = base; o.stats[a.R + r] = ls; }
      if (o.lse) o.lse[r] = base * a.invT + ls;
      if (o.entropy) o.entropy[r] = none ? 0.f : ls - u / s * LN2;
      if (o.logprob)
        o.logprob[r] = (y < 0 || y >= a.C) ? NAN : none ? -INFINITY : (load1(z + y * a.sc) - base) * a.invT - ls;
    }
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
        o.top_lp[ot + j * o.tk] = none ? -INFINITY : (load1(z + c * a.sc) - base) * a.invT - ls;
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
template <typename E>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(const Logits a, const LogprobGrad g) {
  const int lane = threadIdx.x & 63;
  const long long waves = (long long)gridDim.x * 4;
  for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.R; r += waves) {
    const E* z = (const E*)a.z + a.at(r);
    E* dz = (E*)g.dz + (r / a.p) * g.dn + (r % a.p) * g.dp;
    const long long y = g.label ? g.label[r] : -1;
    const float m = g.stats[r], ls = g.stats[a.R + r];
    if ((g.label && y == g.ignore) || ls == -INFINITY) {
      if (!g.accumulate)
        for (int c = lane; c < a.C; c += 64) store1(dz + c * g.dc, 0.f);
      continue;
    }
    const bool has = g.g_logprob && y >= 0 && y < a.C;
    const float G = has ? g.g_logprob[r] * a.invT : 0.f;
    const float B = g.g_entropy ? -g.g_entropy[r] * a.invT : 0.f;
    const float A = (g.g_lse ? g.g_lse[r] * a.invT : 0.f) - G + (g.g_entropy ? B * g.entropy[r] : 0.f);
    for (int c = lane; c < a.C; c += 64) {
      const float lp = (load1(z + c * a.sc) - m) * a.invT - ls;
      float v = expf(lp) * (A + B * fmaxf(lp, -200.f));      // exp(-200) = 0 in fp32; 0 * -inf would be NaN
      if (c == y) v += G;
      if (g.accumulate) v += load1(dz + c * g.dc);
      store1(dz + c * g.dc, v);
    }
  }
}

struct Teacher {
  const void* ids;
  const void* top;
  int ids64, top_type, k, tail;
  long long in, ip, ik, vn, vp, vk;
  const float* weight;
  __device__ __forceinline__ long long id(long long r, long long p, int j) const {
    const long long o = (r / p) * in + (r % p) * ip + j * ik;
    return ids64 ? ((const long long*)ids)[o] : ((const int*)ids)[o];
  }
  __device__ __forceinline__ float value(long long r, long long p, int j) const {
    const long long o = (r / p) * vn + (r % p) * vp + j * vk;
    return top_type == SEMSEG_TYPE_F32 ? ((const float*)top)[o]
         : top_type == SEMSEG_TYPE_BF16 ? (float)((const __bf16*)top)[o] : (float)((const _Float16*)top)[o];
  }
};

// The teacher's distribution of one row, entry j in lane j (k <= 64): q, log q; qsum = sum q, qrest = what is left of 1 (tail).
// id -1 where the entry is absent (negative id, lane >= k); *bad: an id >= C.
__device__ __forceinline__ void teacher_row(const Teacher& t, long long r, long long p, int C, float invT, int lane, int& id, float& q,
                                            float& lq, float& qsum, float& qrest, bool& bad) {
  long long i = -1;
  float v = -INFINITY;
  if (lane < t.k) {
    i = t.id(r, p, lane);
    if (i >= 0) v = t.value(r, p, lane);
  }
  bad = __any(i >= C);
  id = i < 0 || i >= C ? -1 : (int)i;
  if (id < 0) v = -INFINITY;
  if (t.tail) {
    lq = v;
    q = expf(v);
    qsum = wave_sum(q);
    qrest = fmaxf(1.f - qsum, 0.f);
  } else {
    const float m = wave_max(v);
    const float d = (v - (m == -INFINITY ? 0.f : m)) * invT;
    const float e = expf(d), s = wave_sum(e);
    lq = d - logf(s);
    q = s == 0.f ? 0.f : e / s;
    qsum = s == 0.f ? 0.f : 1.f;
    qrest = 0.f;
  }
}

struct DistillOut {
  float *rows, *stats;       // [R] loss per row (or null), stats [3][R]: m, log S, log p_rest (0 without a tail)
  double* part;              // [2][blocks]: weighted loss, weights
  float T2;
};

template <typename E>
__global__ __launch_bounds__(256) void distill_fwd_kernel(const Logits a, const Teacher t, const DistillOut o) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const long long waves = (long long)gridDim.x * 4;
  double loss = 0.0, wsum = 0.0;
  for (long long r = (long long)blockIdx.x * 4 + wv; r < a.R; r += waves) {
    const E* z = (const E*)a.z + a.at(r);
    const float w = t.weight ? t.weight[r] : 1.f;
    if (w == 0.f) {                            // a masked row is not read
      if (lane == 0) {
        if (o.rows) o.rows[r] = 0.f;
        o.stats[r] = o.stats[a.R + r] = o.stats[2 * a.R + r] = 0.f;
      }
      continue;
    }
    int id;
    float q, lq, qsum, qrest;
    bool bad;
    teacher_row(t, r, a.p, a.C, a.invT, lane, id, q, lq, qsum, qrest, bad);
    float m = -INFINITY, mt = -INFINITY;
    for (int c0 = 0; c0 < a.C; c0 += 64) {
      const int c = c0 + lane;
      const float v = c < a.C ? load1(z + c * a.sc) : -INFINITY;
      m = fmaxf(m, v);
      if (t.tail) {
        bool in = false;
        for (int j = 0; j < t.k; ++j) in |= __shfl(id, j) == c;
        if (!in) mt = fmaxf(mt, v);
      }
    }
    m = wave_max(m);
    mt = wave_max(mt);
    const float base = m == -INFINITY ? 0.f : m, baset = mt == -INFINITY ? 0.f : mt;
    float s = 0.f, st = 0.f;
    for (int c0 = 0; c0 < a.C; c0 += 64) {
      const int c = c0 + lane;
      const float v = c < a.C ? load1(z + c * a.sc) : -INFINITY;
      s += expf((v - base) * a.invT);
      if (t.tail) {
        bool in = false;
        for (int j = 0; j < t.k; ++j) in |= __shfl(id, j) == c;
        if (!in) st += expf((v - baset) * a.invT);
      }
    }
    s = wave_sum(s);
    st = wave_sum(st);
    const float ls = logf(s);
    const float lp = id < 0 || s == 0.f ? -INFINITY : (load1(z + id * a.sc) - base) * a.invT - ls;
    float kl = wave_sum(q == 0.f ? 0.f : q * (lq - lp));
    float lpt = 0.f;
    if (t.tail && mt != -INFINITY) {           // a tail without a finite logit is no class
      lpt = (baset - base) * a.invT + logf(st) - ls;
      if (qrest > 0.f) kl += qrest * (logf(qrest) - lpt);
    }
    if (!__any(id >= 0)) kl = 0.f;             // no entry
    if (bad) kl = NAN;
    if (lane == 0) {
      o.stats[r] = base;
      o.stats[a.R + r] = ls;
      o.stats[2 * a.R + r] = t.tail && mt == -INFINITY ? INFINITY : lpt;      // +inf: no tail
      if (o.rows) o.rows[r] = o.T2 * w * kl;
    }
    loss += (double)w * (double)kl;
    wsum += (double)w;
  }
  __shared__ double sl[4], sw[4];
  if (lane == 0) { sl[wv] = loss; sw[wv] = wsum; }
  __syncthreads();
  if (threadIdx.x == 0 && o.part) {
    o.part[blockIdx.x] = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    o.part[gridDim.x + blockIdx.x] = (sw[0] + sw[1]) + (sw[2] + sw[3]);
  }
}

// acc = {sum of weighted losses, sum of weights} from the blocks' partials, added in a fixed order; loss = T^2 acc0 [/ acc1]
__global__ __launch_bounds__(256) void distill_finish_kernel(const double* part, int blocks, double* acc, float* loss, float T2, int mean) {
  double l = 0.0, w = 0.0;
  for (int i = threadIdx.x; i < blocks; i += 256) { l += part[i]; w += part[blocks + i]; }
  for (int o = 32; o; o >>= 1) { l += shfl_xor_f64(l, o); w += shfl_xor_f64(w, o); }
  __shared__ double sl[4], sw[4];
  if ((threadIdx.x & 63) == 0) { sl[threadIdx.x >> 6] = l; sw[threadIdx.x >> 6] = w; }
  __syncthreads();
  if (threadIdx.x == 0) {
    l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    w = (sw[0] + sw[1]) + (sw[2] + sw[3]);
    acc[0] = l;
    acc[1] = w;
    loss[0] = (float)((double)T2 * (mean ? l / w : l));
  }
}

struct DistillGrad {
  const float* stats;
  const double* acc;
  const float* g;            // one gradient (or one per row), null: 1
  float gmul, T;
  int mean, per_row, accumulate;
  void* dz;
  long long dn, dp, dc;
};

// dz_c = coef (p_c Q - sum_{j: id_j = c} q_j) for the teacher's classes, coef p_c Q for the others; with a tail Q counts it, and the
// others are coef exp(log p_c - log p_rest) (Q p_rest - q_rest): one exponential, and no overflow where p_rest is tiny.
template <typename E>
__global__ __launch_bounds__(256) void distill_bwd_kernel(const Logits a, const Teacher t, const DistillGrad g) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const long long waves = (long long)gridDim.x * 4;
  for (long long r = (long long)blockIdx.x * 4 + wv; r < a.R; r += waves) {
    const E* z = (const E*)a.z + a.at(r);
    E* dz = (E*)g.dz + (r / a.p) * g.dn + (r % a.p) * g.dp;
    const float w = t.weight ? t.weight[r] : 1.f;
    const float base = g.stats[r], ls = g.stats[a.R + r], lpt = g.stats[2 * a.R + r];
    int id;
    float q, lq, qsum, qrest;
    bool bad;
    teacher_row(t, r, a.p, a.C, a.invT, lane, id, q, lq, qsum, qrest, bad);
    float coef = g.gmul * g.T * w * (g.g ? g.g[g.per_row ? r : 0] : 1.f);
    if (g.mean) coef = g.acc[1] == 0.0 ? 0.f : (float)((double)coef / g.acc[1]);
    if (w == 0.f || bad || ls == -INFINITY || !__any(id >= 0)) {
      if (!g.accumulate)
        for (int c = lane; c < a.C; c += 64) store1(dz + c * g.dc, 0.f);
      continue;
    }
    const bool tail = t.tail && lpt != INFINITY;
    const float Q = tail ? qsum + qrest : qsum;
    const float off = tail ? ls + lpt : ls, fac = tail ? Q * expf(lpt) - qrest : Q;
    for (int c0 = 0; c0 < a.C; c0 += 64) {
      const int c = c0 + lane;
      float qc = 0.f;
      bool in = false;
      for (int j = 0; j < t.k; ++j) {
        const int ij = __shfl(id, j);
        const float qj = __shfl(q, j);
        if (ij == c) { in = true; qc += qj; }
      }
      if (c >= a.C) continue;
      const float d = (load1(z + c * a.sc) - base) * a.invT;
      float v = coef * (in ? Q * expf(d - ls) - qc : fac * expf(d - off));
      if (g.accumulate) v += load1(dz + c * g.dc);
      store1(dz + c * g.dc, v);
    }
  }
}

int row_blocks(long long R) {
  const long long b = (R + 3) / 4;
  return (int)(b < 8192 ? b : 8192);
}

bool logits_ok(const void* z, int type, long long n, long long p, int C, float T) {
  return z && type >= 0 && type <= 2 && n > 0 && p > 0 && C > 0 && p <= (1ll << 40) / n && T > 0.f && T <= 3e38f;
}
bool teacher_ok(const void* ids, int ids64, const void* top, int top_type, int k) {
  return ids && top && (ids64 == 0 || ids64 == 1) && top_type >= 0 && top_type <= 2 && k >= 1 && k <= MAXK;
}

Logits logits_of(const void* z, long long n, long long p, int C, long long sn, long long sp, long long sc, float T) {
  return Logits{z, n * p, p, sn, sp, sc, C, 1.f / T, LOG2E / T};
}

#define BY_TYPE(type, K, ...)                            \
  do {                                                   \
    if (type == SEMSEG_TYPE_F32) K<float> __VA_ARGS__;   \
    else if (type == SEMSEG_TYPE_BF16) K<__bf16> __VA_ARGS__; \
    else K<_Float16> __VA_ARGS__;                        \
  } while (0)

}  // namespace

extern "C" {

int semseg_class_logprobs_fwd(const void* z, int type, long long n, long long p, int C, long long sn, long long sp, long long sc,
                              const long long* label, long long ignore_index, float T, int k, float* logprob, float* entropy,
                              float* lse, float* stats, int* top_ids, float* top_logprobs, long long tn, long long tp, long long tk,
                              hipStream_t stream) {
  if (!logits_ok(z, type, n, p, C, T) || k < 0 || k > MAXK || k > C || (k && (!top_ids || !top_logprobs)) || (logprob && !label))
    return SEMSEG_EINVAL;
  const Logits a = logits_of(z, n, p, C, sn, sp, sc, T);
  const LogprobOut o{label, ignore_index, logprob, entropy, lse, stats, top_ids, top_logprobs, k, tn, tp, tk};
  BY_TYPE(type, logprobs_fwd_kernel, <<<row_blocks(a.R), 256, 0, stream>>>(a, o));
  return semseg_launch_status();
}

int semseg_class_logprobs_bwd(const void* z, int type, long long n, long long p, int C, long long sn, long long sp, long long sc,
                              const long long* label, long long ignore_index, float T, const float* stats, const float* entropy,
                              const float* g_logprob, const float* g_entropy, const float* g_lse, void* dz, long long dn,
                              long long dp, long long dc, int accumulate, hipStream_t stream) {
  if (!logits_ok(z, type, n, p, C, T) || !stats || !dz || (g_entropy && !entropy) || (g_logprob && !label)) return SEMSEG_EINVAL;
  const Logits a = logits_of(z, n, p, C, sn, sp, sc, T);
  const LogprobGrad g{label, ignore_index, stats, entropy, g_logprob, g_entropy, g_lse, dz, dn, dp, dc, accumulate};
  BY_TYPE(type, logprobs_bwd_kernel, <<<row_blocks(a.R), 256, 0, stream>>>(a, g));
  return semseg_launch_status();
}

size_t semseg_distill_scratch_bytes(long long n, long long p, int C) {
  if (n <= 0 || p <= 0 || C <= 0) return 0;
  return (size_t)row_blocks(n * p) * 2 * sizeof(double);
}

int semseg_distill_fwd(const void* z, int type, long long n, long long p, int C, long long sn, long long sp, long long sc, const void* ids,
                       int ids64, const void* top, int top_type, int k, long long in, long long ip, long long ik, long long vn,
                       long long vp, long long vk, const float* weight, float T, int tail, int reduction, float* rows, float* stats,
                       double* acc2, float* loss, void* scratch, size_t scratch_bytes, hipStream_t stream) {
  if (!logits_ok(z, type, n, p, C, T) || !teacher_ok(ids, ids64, top, top_type, k) || !stats || reduction < 0 || reduction > 2)
    return SEMSEG_EINVAL;
  if (reduction == SEMSEG_REDUCE_NONE ? !rows : (!acc2 || !loss || !scratch || scratch_bytes < semseg_distill_scratch_bytes(n, p, C)))
    return SEMSEG_EINVAL;
  const Logits a = logits_of(z, n, p, C, sn, sp, sc, T);
  const Teacher t{ids, top, ids64, top_type, k, tail, in, ip, ik, vn, vp, vk, weight};
  const int blocks = row_blocks(a.R);
  const DistillOut o{rows, stats, reduction == SEMSEG_REDUCE_NONE ? nullptr : (double*)scratch, T * T};
  BY_TYPE(type, distill_fwd_kernel, <<<blocks, 256, 0, stream>>>(a, t, o));
  if (reduction != SEMSEG_REDUCE_NONE)
    distill_finish_kernel<<<1, 256, 0, stream>>>((const double*)scratch, blocks, acc2, loss, T * T, reduction == SEMSEG_REDUCE_MEAN);
  return semseg_launch_status();
}

int semseg_distill_bwd(const void* z, int type, long long n, long long p, int C, long long sn, long long sp, long long sc, const void* ids,
                       int ids64, const void* top, int top_type, int k, long long in, long long ip, long long ik, long long vn,
                       long long vp, long long vk, const float* weight, float T, int tail, int reduction, const float* stats,
                       const double* acc2, const float* grad_loss, float grad_mul, void* dz, long long dn, long long dp, long long dc,
                       int accumulate, hipStream_t stream) {
  if (!logits_ok(z, type, n, p, C, T) || !teacher_ok(ids, ids64, top, top_type, k) || !stats || !dz || reduction < 0 || reduction > 2 ||
      (reduction == SEMSEG_REDUCE_MEAN && !acc2))
    return SEMSEG_EINVAL;
  const Logits a = logits_of(z, n, p, C, sn, sp, sc, T);
  const Teacher t{ids, top, ids64, top_type, k, tail, in, ip, ik, vn, vp, vk, weight};
  const DistillGrad g{stats, acc2, grad_loss, grad_mul, T, reduction == SEMSEG_REDUCE_MEAN, reduction == SEMSEG_REDUCE_NONE,
                      accumulate, dz, dn, dp, dc};
  BY_TYPE(type, distill_bwd_kernel, <<<row_blocks(a.R), 256, 0, stream>>>(a, t, g));
  return semseg_launch_status();
}

int semseg_distill_fwd_bwd(const void* z, int type, long long n, long long p, int C, long long sn, long long sp, long long sc,
                           const void* ids, int ids64, const void* top, int top_type, int k, long long in, long long ip, long long ik,
                           long long vn, long long vp, long long vk, const float* weight, float T, int tail, int reduction,
                           float* stats, double* acc2, float* loss, float grad_mul, void* dz, long long dn, long long dp, long long dc,
                           int accumulate, void* scratch, size_t scratch_bytes, hipStream_t stream) {
  if (reduction != SEMSEG_REDUCE_MEAN && reduction != SEMSEG_REDUCE_SUM) return SEMSEG_EINVAL;
  const int rc = semseg_distill_fwd(z, type, n, p, C, sn, sp, sc, ids, ids64, top, top_type, k, in, ip, ik, vn, vp, vk, weight, T, tail,
                                    reduction, nullptr, stats, acc2, loss, scratch, scratch_bytes, stream);
  if (rc != SEMSEG_OK) return rc;
  return semseg_distill_bwd(z, type, n, p, C, sn, sp, sc, ids, ids64, top, top_type, k, in, ip, ik, vn, vp, vk, weight, T, tail,
                            reduction, stats, acc2, nullptr, grad_mul, dz, dn, dp, dc, accumulate, stream);
}

}  // extern "C"
