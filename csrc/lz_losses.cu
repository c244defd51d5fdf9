// Vocabulary losses: token log-probabilities, a clipped policy loss with a KL
// term, distillation from a teacher's top logits (and, from log-probabilities,
// a preference loss), forward and backward.
//
// With z = logits / T, lse = log sum_j exp z_j and p = softmax(z), every one of
// them needs the sum of a row, a few of its entries and then the gradient
//     dlogits_j = slope / T * (t_j - p_j),
// where slope is the loss's derivative in sum_j t_j (z_j - lse) and t is one
// token (LOGP, POLICY) or the teacher's distribution over its top entries
// (DISTILL). Only the row's scalars differ. Everything is held in base 2:
// c = log2(e) / T, p_j = 2^(x_j c - lse2), so an element costs one FMA and one
// exponential. Sums run in 32 bits a thread; what is per row (lse2, the slope,
// the loss) in 64 bits, since a log-probability enters the KL term and the
// ratio as a difference and costs nothing per element.
#include <atomic>
#include <type_traits>

#include "lz_common.cuh"
#include "lz_internal.h"
#include "lz_losses.h"

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr double kLn2 = 0.693147180559945309417;
constexpr double kLog2e = 1.44269504088896340736;

// 2^x; results below 2^-126 are zero.
LZ_DEV float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int N = 4;  // elements of a 16-byte vector
  LZ_DEV static float get(float v) { return v; }
  LZ_DEV static float put(float v) { return v; }
  LZ_DEV static void unpack(uint4 v, float* f) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  LZ_DEV static uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int N = 8;
  LZ_DEV static float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  LZ_DEV static __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
  LZ_DEV static void unpack(uint4 v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  LZ_DEV static uint4 pack(const float* f) {
    uint4 v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    return v;
  }
};
template <>
struct Elem<__half> {
  static constexpr int N = 8;
  LZ_DEV static float get(__half v) { return __half2float(v); }
  LZ_DEV static __half put(float v) { return __float2half_rn(v); }
  LZ_DEV static void unpack(uint4 v, float* f) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(h[i]);
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  }
  LZ_DEV static uint4 pack(const float* f) {
    uint4 v;
    __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    return v;
  }
};

// Running maximum and sum of a softmax: sum_j 2^(x_j c - ref), where ref is the
// maximum, rounded to an integer so that sums are brought to another reference
// without a rounding (0 while it is -inf, so that rows of -inf sum to 0 and not
// to NaN). A NaN or +inf among the logits makes the sum NaN.
struct Running {
  float max, ref, sum;
  LZ_DEV void init() { max = -INFINITY, ref = 0.f, sum = 0.f; }
  LZ_DEV void raise(float m) {
    if (m > max + 0.5f) {
      m = rintf(m);
      sum *= exp2_fast(max - m);
      max = m, ref = m;
    }
  }
  LZ_DEV void join(float omax, float osum) {
    if (omax > max) {
      sum = sum * (max == -INFINITY ? 1.f : exp2_fast(max - omax)) + osum;
      max = omax, ref = omax;
    } else {
      sum += osum * (omax == -INFINITY ? 1.f : exp2_fast(omax - max));
    }
  }
};

template <typename T>
LZ_DEV void take_vector(Running& s, uint4 v, float c) {
  constexpr int N = Elem<T>::N;
  float f[N];
  Elem<T>::unpack(v, f);
  float m = f[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, f[i]);
  s.raise(m * c);
#pragma unroll
  for (int i = 0; i < N; ++i) s.sum += exp2_fast(fmaf(f[i], c, -s.ref));
}

template <typename T>
LZ_DEV void take_one(Running& s, T v, float c) {
  const float f = Elem<T>::get(v);
  s.raise(f * c);
  s.sum += exp2_fast(fmaf(f, c, -s.ref));
}

// A row as [0, lead) single elements, `vecs` 16-byte vectors, single elements.
template <typename T>
struct Split {
  int lead, vecs;
  LZ_DEV Split(const T* p, long long n) {
    const int off = (int)((uintptr_t)p % 16) / (int)sizeof(T);
    const int l = off ? Elem<T>::N - off : 0;
    lead = l < n ? l : (int)n;
    vecs = (int)((n - lead) / Elem<T>::N);
  }
};

// One thread's share of the row's sum.
template <typename T>
LZ_DEV Running row_sum(const T* x, long long n, float c) {
  constexpr int N = Elem<T>::N, U = 4;
  Running s;
  s.init();
  const Split<T> sp(x, n);
  const uint4* v = reinterpret_cast<const uint4*>(x + sp.lead);
  int i = threadIdx.x;
  for (; i + (U - 1) * kThreads < sp.vecs; i += U * kThreads) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = __ldg(v + i + u * kThreads);
#pragma unroll
    for (int u = 0; u < U; ++u) take_vector<T>(s, w[u], c);
  }
  for (; i < sp.vecs; i += kThreads) take_vector<T>(s, __ldg(v + i), c);
  const long long tail = sp.lead + (long long)sp.vecs * N;
  const int singles = sp.lead + (int)(n - tail);
  if (threadIdx.x < singles) take_one<T>(s, x[threadIdx.x < sp.lead ? threadIdx.x : tail + threadIdx.x - sp.lead], c);
  return s;
}

// The row's (max, sum) in every thread; `buf` holds kWarps pairs. The order of
// the additions depends on nothing but the row's length and alignment.
LZ_DEV Running block_join(Running s, float2* buf) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float m = __shfl_xor_sync(~0u, s.max, o), q = __shfl_xor_sync(~0u, s.sum, o);
    s.join(m, q);
  }
  if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = make_float2(s.max, s.sum);
  __syncthreads();
  Running t;
  t.init();
  for (int w = 0; w < kWarps; ++w) t.join(buf[w].x, buf[w].y);
  __syncthreads();
  return t;
}

LZ_DEV float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float m = red[0];
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, red[w]);
  __syncthreads();
  return m;
}

template <typename V>
LZ_DEV V block_sum(V v, V* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  V s = red[0];
  for (int w = 1; w < kWarps; ++w) s += red[w];
  __syncthreads();
  return s;
}

// p_j = 2^((x_j - base) c - lse2). base is 0 but in rows whose maximum times c
// is beyond 32 bits (all of a row masked with the type's lowest value): there it
// is that maximum, and the row takes the slow loops.
struct Norm {
  float base;
  double lse2;
};

template <typename T>
LZ_DEV double row_log2p(const T* x, long long i, const Norm& n, float c) {
  return ((double)Elem<T>::get(x[i]) - (double)n.base) * (double)c - n.lse2;
}

// The row's normaliser in every thread, from the block's (max, sum).
template <typename T>
LZ_DEV Norm row_norm(const Running& s, const T* x, long long n, float c, float* red) {
  if (!isinf(s.max)) return {0.f, (double)s.max + log2((double)s.sum)};
  float m = -INFINITY;
  for (long long i = threadIdx.x; i < n; i += kThreads) m = fmaxf(m, Elem<T>::get(x[i]));
  m = block_max(m, red);
  float t = 0.f;
  for (long long i = threadIdx.x; i < n; i += kThreads) t += exp2_fast((Elem<T>::get(x[i]) - m) * c);
  t = block_sum(t, red);  // NaN where m is infinite
  return {m, log2((double)t)};
}

// Writes -slope / T p_j, rounded once to the logits' type; zeros without a look
// at x where the slope is zero. lse2 is taken in 32 bits and the factor makes up
// for what that rounding leaves.
template <typename T>
LZ_DEV void row_dense(const T* x, T* out, long long n, double slope, float inv_t, const Norm& norm, float c) {
  constexpr int N = Elem<T>::N;
  const float l = (float)norm.lse2;
  const double left = (double)l - norm.lse2;  // at most half a step of l: 2^left is 1 + left ln 2
  const float a = slope == 0.0 ? 0.f : (float)(-slope * inv_t * (1.0 + left * kLn2));
  if (a == 0.f) {
    const Split<T> sp(out, n);
    uint4* v = reinterpret_cast<uint4*>(out + sp.lead);
    for (int i = threadIdx.x; i < sp.vecs; i += kThreads) st_cs_v4(v + i, make_uint4(0, 0, 0, 0));
    const long long tail = sp.lead + (long long)sp.vecs * N;
    const int singles = sp.lead + (int)(n - tail);
    if (threadIdx.x < singles) out[threadIdx.x < sp.lead ? threadIdx.x : tail + threadIdx.x - sp.lead] = Elem<T>::put(0.f);
    return;
  }
  // one element at a time where the two rows start at different offsets from a 16-byte border
  if (norm.base != 0.f || ((uintptr_t)x ^ (uintptr_t)out) % 16) {
    for (long long i = threadIdx.x; i < n; i += kThreads)
      out[i] = Elem<T>::put(a * exp2_fast(fmaf(Elem<T>::get(x[i]) - norm.base, c, -l)));
    return;
  }
  const Split<T> sp(x, n);
  const uint4* v = reinterpret_cast<const uint4*>(x + sp.lead);
  uint4* o = reinterpret_cast<uint4*>(out + sp.lead);
  constexpr int U = 4;
  for (int i = threadIdx.x; i < sp.vecs; i += U * kThreads) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kThreads < sp.vecs) w[u] = __ldg(v + i + u * kThreads);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[N];
      Elem<T>::unpack(w[u], f);
#pragma unroll
      for (int k = 0; k < N; ++k) f[k] = a * exp2_fast(fmaf(f[k], c, -l));
      if (i + u * kThreads < sp.vecs) st_cs_v4(o + i + u * kThreads, Elem<T>::pack(f));
    }
  }
  const long long tail = sp.lead + (long long)sp.vecs * N;
  const int singles = sp.lead + (int)(n - tail);
  if (threadIdx.x < singles) {
    const long long i = threadIdx.x < sp.lead ? threadIdx.x : tail + threadIdx.x - sp.lead;
    out[i] = Elem<T>::put(a * exp2_fast(fmaf(Elem<T>::get(x[i]), c, -l)));
  }
}

LZ_DEV long long load_id(const void* ids, int ids64, long long i) {
  return ids64 ? static_cast<const long long*>(ids)[i] : (long long)static_cast<const int*>(ids)[i];
}

LZ_DEV float load_any(const void* p, int dtype, long long i) {
  if (dtype == LZ_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == LZ_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}

template <typename T>
LZ_DEV const T* row_of(const LzLossArgs& a, long long r) {
  const T* x = static_cast<const T*>(a.logits);
  if (a.inner == a.rows) return x + r * a.inner_stride;
  return x + (r / a.inner) * a.outer_stride + (r % a.inner) * a.inner_stride;
}

// The parts of `work`.
LZ_DEV double2* work_norm(const LzLossArgs& a) { return reinterpret_cast<double2*>(a.work + LZ_LOSS_WORK_HEAD); }
LZ_DEV double* work_slope(const LzLossArgs& a) { return a.work + LZ_LOSS_WORK_HEAD + 2 * a.rows; }
LZ_DEV double* work_loss(const LzLossArgs& a) { return a.work + LZ_LOSS_WORK_HEAD + 3 * a.rows; }
LZ_DEV int* work_order(const LzLossArgs& a) { return reinterpret_cast<int*>(a.work + LZ_LOSS_WORK_HEAD + 4 * a.rows); }
LZ_DEV unsigned* work_ticket(const LzLossArgs& a) { return reinterpret_cast<unsigned*>(a.work + 1); }
LZ_DEV int* work_active(const LzLossArgs& a) { return reinterpret_cast<int*>(a.work + 1) + 1; }

// Whether a row counts: its token is not negative and its weight not zero.
template <int KIND>
LZ_DEV bool row_counts(const LzLossArgs& a, long long r) {
  return (KIND == LZ_LOSS_DISTILL || load_id(a.ids, a.ids64, r) >= 0) &&
         (KIND == LZ_LOSS_LOGP || !a.weights || a.weights[r] != 0.f);
}

// The teacher's list of one row in shared memory.
struct Top {
  float q[LZ_LOSS_MAX_TOP];     // the teacher's probabilities; 0 for padding
  int id[LZ_LOSS_MAX_TOP];      // -1: padding
  float red[kWarps];
};

LZ_DEV float top_value(const LzLossArgs& a, long long r, int k) {
  return load_any(a.teacher, a.teacher_dtype, r * a.top + k) * a.inv_temperature;
}

// q = softmax(teacher / T) over the entries whose id is not negative. Returns
// the log of the sum, and the maximum through `tmax`: -inf where the list is
// empty, NaN where an id is beyond the vocabulary.
LZ_DEV double top_softmax(const LzLossArgs& a, long long r, Top& t, float* tmax) {
  float m = -INFINITY;
  bool bad = false;
  for (int k = threadIdx.x; k < a.top; k += kThreads) {
    const long long id = load_id(a.ids, a.ids64, r * a.top + k);
    const float v = id < 0 ? -INFINITY : top_value(a, r, k);
    bad |= id >= a.vocab;
    t.id[k] = id < 0 || id >= a.vocab ? -1 : (int)id;
    t.q[k] = v;
    m = fmaxf(m, v);
  }
  m = block_max(m, t.red);
  bad = __syncthreads_or(bad);
  float s = 0.f;
  for (int k = threadIdx.x; k < a.top; k += kThreads) {
    const float e = m == -INFINITY ? 0.f : expf(t.q[k] - m);
    t.q[k] = e;
    s += e;
  }
  s = block_sum(s, t.red);
  const float inv = bad ? NAN : (s > 0.f || s != s ? 1.f / s : 0.f);
  for (int k = threadIdx.x; k < a.top; k += kThreads) t.q[k] *= inv;
  __syncthreads();
  *tmax = bad ? NAN : m;
  return log((double)s);
}

// The entries where t_j is not zero, over what row_dense wrote (a barrier
// between the two is the caller's).
template <typename T>
LZ_DEV void row_sparse_token(const LzLossArgs& a, const T* x, T* out, long long y, double slope, const Norm& n, float c) {
  if (threadIdx.x == 0 && slope != 0.0) {
    const double p = exp2(row_log2p(x, y, n, c));
    out[y] = Elem<T>::put((float)(slope * a.inv_temperature * (1.0 - p)));
  }
}

template <typename T>
LZ_DEV void row_sparse_top(const LzLossArgs& a, const T* x, T* out, const Top& t, double slope, const Norm& n, float c) {
  if (slope == 0.0) return;
  for (int k = threadIdx.x; k < a.top; k += kThreads) {
    const int id = t.id[k];
    if (id < 0) continue;
    float q = t.q[k];
    bool first = true;
    for (int o = 0; o < a.top; ++o) {  // an index that stands in the list twice gets both shares
      if (t.id[o] != id || o == k) continue;
      if (o < k) first = false;
      q += t.q[o];
    }
    if (!first) continue;
    const double p = exp2(row_log2p(x, id, n, c));
    out[id] = Elem<T>::put((float)(slope * a.inv_temperature * ((double)q - p)));
  }
}

// Scalars of a LOGP or POLICY row from its sum; one thread. Returns the slope.
template <typename T, int KIND>
LZ_DEV double token_scalars(const LzLossArgs& a, const T* x, long long r, long long y, const Norm& n, float c) {
  const bool there = y < a.vocab;  // otherwise every output of the row is NaN
  const double logp = there ? row_log2p(x, y, n, c) * kLn2 : (double)NAN;
  a.logp[r] = (float)logp;
  if (KIND == LZ_LOSS_LOGP) return logp;
  const double w = (a.weights ? (double)a.weights[r] : 1.0) * a.work[0];
  const double adv = a.advantages[r], ratio = exp(logp - (double)a.old_logp[r]);
  const double lo = 1.0 - (double)a.clip_low, hi = 1.0 + (double)a.clip_high;
  const bool clipped = (adv > 0.0 && ratio > hi) || (adv < 0.0 && ratio < lo);
  double each = -adv * (clipped ? (adv > 0.0 ? hi : lo) : ratio);
  double slope = clipped ? 0.0 : -adv * ratio;
  if (a.ref_logp) {
    const double d = (double)a.ref_logp[r] - logp, e = expm1(d);
    a.kl[r] = (float)(e - d);
    each += (double)a.kl_coef * (e - d);
    slope -= (double)a.kl_coef * e;
  }
  a.clipped[r] = clipped;
  work_loss(a)[r] = w * each;
  return w * slope;
}

// One CTA a row at a time: the sum, the row's scalars, then the gradient from
// a second look at the row, which L2 still holds. Masked rows are not read.
template <typename T, int KIND, bool GRAD>
__global__ void __launch_bounds__(kThreads) forward_kernel(const __grid_constant__ LzLossArgs a) {
  __shared__ float2 buf[kWarps];
  __shared__ double dred[kWarps];
  __shared__ double row_slope;
  __shared__ bool last;
  extern __shared__ char dynamic[];
  const float c = (float)(kLog2e * (double)a.inv_temperature);
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = row_of<T>(a, r);
    const bool weighted = KIND == LZ_LOSS_LOGP || !a.weights || a.weights[r] != 0.f;
    const long long y = KIND == LZ_LOSS_DISTILL ? 0 : load_id(a.ids, a.ids64, r);
    double slope = 0.0;
    Norm n = {0.f, 0.0};
    Top* top = reinterpret_cast<Top*>(dynamic);
    if (weighted && y >= 0) {
      const Running s = block_join(row_sum<T>(x, a.vocab, c), buf);
      n = row_norm(s, x, a.vocab, c, reinterpret_cast<float*>(buf));
      if (KIND == LZ_LOSS_DISTILL) {
        float tmax;
        const double logsum = top_softmax(a, r, *top, &tmax);
        double kl = 0.0;
        for (int k = threadIdx.x; k < a.top; k += kThreads) {
          if (top->q[k] == 0.f) continue;
          const double logq = (double)top_value(a, r, k) - tmax - logsum;
          const double logp = top->id[k] < 0 ? (double)NAN : row_log2p(x, top->id[k], n, c) * kLn2;
          kl += (double)top->q[k] * (logq - logp);
        }
        kl = block_sum(kl, dred);
        const double w = (a.weights ? (double)a.weights[r] : 1.0) * a.work[0];
        slope = tmax == -INFINITY ? 0.0 : isnan(tmax) ? (double)NAN : -w;
        if (threadIdx.x == 0) {
          a.kl[r] = (float)kl;
          work_loss(a)[r] = w * kl;
        }
      } else {
        if (threadIdx.x == 0) row_slope = token_scalars<T, KIND>(a, x, r, y, n, c);
        __syncthreads();
        slope = row_slope;
      }
    } else if (threadIdx.x == 0) {
      if (KIND == LZ_LOSS_DISTILL) a.kl[r] = 0.f;
      else a.logp[r] = 0.f;
      if (KIND == LZ_LOSS_POLICY) {
        if (a.ref_logp) a.kl[r] = 0.f;
        a.clipped[r] = 0;
      }
      if (KIND != LZ_LOSS_LOGP) work_loss(a)[r] = 0.0;
    }
    if (threadIdx.x == 0) {
      work_norm(a)[r] = make_double2(n.base, n.lse2);
      work_slope(a)[r] = slope;
    }
    if (GRAD) {
      T* out = static_cast<T*>(a.grad) + r * a.vocab;
      row_dense<T>(x, out, a.vocab, slope, a.inv_temperature, n, c);
      __syncthreads();
      if (KIND == LZ_LOSS_DISTILL) row_sparse_top<T>(a, x, out, *top, slope, n, c);
      else if (y < a.vocab) row_sparse_token<T>(a, x, out, y, slope, n, c);
    }
    __syncthreads();  // the next row's scalars and list overwrite this one's
  }
  if (KIND == LZ_LOSS_LOGP) return;
  // The CTA that is done last adds the rows' losses up, in the rows' order.
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0)
    last = atomicAdd(work_ticket(a), 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
  for (long long r = threadIdx.x; r < a.rows; r += kThreads) s += __ldcg(work_loss(a) + r);
  s = block_sum(s, dred);
  if (threadIdx.x == 0) *a.loss = (float)s;
}

// 1 / denominator (0 where that is not positive: nothing counts), the ticket and,
// where `order` is set, the rows that count in front of those that do not, each
// in their order: taken in turns, every cluster of stream_kernel gets as many.
template <int KIND>
__global__ void __launch_bounds__(kThreads) head_kernel(const __grid_constant__ LzLossArgs a, bool order) {
  __shared__ double red[kWarps];
  __shared__ int counts[2][kWarps];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  double s = 0.0;
  if (KIND != LZ_LOSS_LOGP) {
    if (a.denom_ptr) {
      s = (double)*a.denom_ptr;
    } else if (a.denom >= 0.0) {
      s = a.denom;
    } else {
      for (long long r = threadIdx.x; r < a.rows; r += kThreads)
        if (KIND == LZ_LOSS_DISTILL || load_id(a.ids, a.ids64, r) >= 0) s += a.weights ? (double)a.weights[r] : 1.0;
      s = block_sum(s, red);
    }
  }
  if (threadIdx.x == 0) {
    a.work[0] = s > 0.0 || s != s ? 1.0 / s : 0.0;
    *work_ticket(a) = 0u;
    if (KIND != LZ_LOSS_LOGP && a.rows == 0) *a.loss = 0.f;
  }
  if (!order) return;
  const int n = (int)a.rows;
  int front = 0, back = 0;  // rows placed at either end
  for (int first = 0, k = 0; first < n; first += kThreads, k ^= 1) {
    const int r = first + threadIdx.x;
    const bool counts_ = r < n && row_counts<KIND>(a, r);
    const unsigned m = __ballot_sync(~0u, counts_);
    if (lane == 0) counts[k][warp] = __popc(m);
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
      before += w < warp ? counts[k][w] : 0;
      all += counts[k][w];
    }
    before += __popc(m & ((1u << lane) - 1));
    if (r < n) work_order(a)[counts_ ? front + before : n - 1 - (back + (int)threadIdx.x - before)] = r;
    front += all;
    back += min(kThreads, n - first) - all;
  }
  if (threadIdx.x == 0) *work_active(a) = front;
}

// A row's slope for the given upstream.
template <int KIND>
LZ_DEV double row_slope_for(const LzLossArgs& a, long long r, long long y, float up) {
  if (y >= a.vocab) return NAN;
  if (KIND == LZ_LOSS_LOGP) return y < 0 ? 0.0 : (double)up * (double)a.row_upstream[r];
  const double slope = work_slope(a)[r];
  return slope == 0.0 ? 0.0 : (double)up * slope;
}

// The gradient from the rows' saved sums and slopes, a CTA a row. POLICY and
// DISTILL: where `grad` holds the gradient for upstream 1 and the upstream is 1,
// it stands.
template <typename T, int KIND>
__global__ void __launch_bounds__(kThreads) backward_kernel(const __grid_constant__ LzLossArgs a) {
  extern __shared__ char dynamic[];
  const float up = a.upstream ? *a.upstream : 1.f;
  if (!a.fresh && up == 1.f) return;
  const float c = (float)(kLog2e * (double)a.inv_temperature);
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = row_of<T>(a, r);
    T* out = static_cast<T*>(a.grad) + r * a.vocab;
    const Norm n = {(float)work_norm(a)[r].x, work_norm(a)[r].y};
    const long long y = KIND == LZ_LOSS_DISTILL ? 0 : load_id(a.ids, a.ids64, r);
    const double slope = row_slope_for<KIND>(a, r, y, up);
    Top* top = reinterpret_cast<Top*>(dynamic);
    if (KIND == LZ_LOSS_DISTILL && slope != 0.0) {
      float tmax;
      top_softmax(a, r, *top, &tmax);
    }
    row_dense<T>(x, out, a.vocab, slope, a.inv_temperature, n, c);
    __syncthreads();
    if (KIND == LZ_LOSS_DISTILL) row_sparse_top<T>(a, x, out, *top, slope, n, c);
    else if (y < a.vocab) row_sparse_token<T>(a, x, out, y, slope, n, c);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Large vocabularies: a cluster of CTAs a row, each with a slice of it.
//
// A row goes through shared memory once. One warp streams the slices of the
// cluster's rows into a ring of chunks by bulk copies and runs ahead as far as
// the ring has room. W warps take a chunk's part of the row's sum, and for the
// gradient take the chunks a second time, from shared memory, and hand each back
// to the ring. So HBM sees a row read once and its gradient written once, and
// reads of the next row run under the writes of this one. One more warp keeps
// what is per row off that path: it joins the warps' sums, exchanges them with
// the cluster's CTAs through distributed shared memory, works out the row's
// scalars from values fetched a row ahead (and the teacher's list), writes the
// row's outputs, and puts the few entries with t_j != 0 over the dense gradient
// once that is written. While it does, the W warps take the first chunks of the
// next row, as many as fit beside this one.
// ---------------------------------------------------------------------------

constexpr int kMaxSlots = 64;
constexpr int kMaxCluster = 8;
constexpr int kSmallList = 128;  // teacher's lists up to here look for equal ids entry by entry, longer ones by a hash table
constexpr unsigned long long kWaitNs = 4000000000ull;  // bound of every wait

struct StreamPlan {
  int slots;    // of the ring, a chunk each
  int early;    // chunks of the next row taken before this one's gradient
  int ordered;  // rows by work_order; otherwise one row a cluster
  int hash;     // entries of the hash table of DISTILL, a power of two; 0 where the list is short
};

struct RowParams {
  float xy, adv;
  double old_logp2, ref_logp2;  // base 2
  double weight;  // over the denominator
  int token;      // -1: beyond the vocabulary
  float slope;    // DISTILL
  double q_logq, q_z, q_sum;  // DISTILL: sums over the list (z in base 2)
};

// Which row, and this CTA's slice of it.
struct RowHead {
  long long row;  // -1: no more
  int lead, vecs, first, count, chunks;
};

// What the dense gradient of a row takes: f 2^((x - base) c - ref).
struct RowDense {
  float f, base, ref;
};

// The teacher's list of a row: entries and, with equal ids joined, what the gradient takes from them.
struct TopView {
  int* id;
  float *z, *q, *share;  // share < 0: another entry of the same id has it
};

// Both rows' lists (id, z, q, share) and the hash table.
__host__ __device__ inline int list_bytes(int kind, int top, int hash) {
  return kind == LZ_LOSS_DISTILL ? (top * 32 + hash * 4 + 127) / 128 * 128 : 0;
}

struct alignas(128) StreamShared {
  uint64_t full[kMaxSlots], empty[kMaxSlots];
  uint64_t parts[2], peers[2], dense[2], ready[2], used[2];  // of every other row
  float2 warp_part[2][16];
  float2 peer_part[2][kMaxCluster];
  RowHead heads[4];
  RowDense row_dense[2];
  RowParams params[2];
  int failed;
};

LZ_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
LZ_DEV uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
LZ_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
LZ_DEV void mbar_arrive(uint64_t* bar) {
  asm volatile("{\n\t.reg .b64 t;\n\tmbarrier.arrive.shared::cta.b64 t, [%0];\n\t}" ::"r"(smem_addr(bar)) : "memory");
}
// Sends v to `slot` of CTA `rank`'s shared memory; its 8 bytes count there on
// `bar`. (A remote arrive with release semantics would first wait for this
// thread's outputs to reach global memory.)
LZ_DEV void send_to_peer(float2* slot, float2 v, uint64_t* bar, uint32_t rank) {
  asm volatile(
      "{\n\t.reg .b32 s, b;\n\t"
      "mapa.shared::cluster.u32 s, %0, %2;\n\t"
      "mapa.shared::cluster.u32 b, %1, %2;\n\t"
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [s], {%3, %4}, [b];\n\t}" ::"r"(smem_addr(slot)),
      "r"(smem_addr(bar)), "r"(rank), "f"(v.x), "f"(v.y)
      : "memory");
}
// Arrives at this CTA's `bar` and has it wait for `bytes` besides.
LZ_DEV void mbar_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("{\n\t.reg .b64 t;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 t, [%0], %1;\n\t}" ::"r"(smem_addr(bar)),
               "r"(bytes)
               : "memory");
}

// Waits for phase `parity` of `bar`, 4 s at most. A wait that gives up sets
// `failed`, and the CTA's other waits then return at once: the kernel runs to its
// end and leaves NaN.
template <bool CLUSTER>
LZ_DEV bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  if (CLUSTER)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
  return done != 0;
}

template <bool CLUSTER>
__device__ __noinline__ void ring_wait_on(uint32_t bar, uint32_t parity, volatile int* failed) {
  unsigned long long began = 0;
  for (uint32_t it = 1; it; ++it) {
    if (try_wait<CLUSTER>(bar, parity) || *failed) return;
    if (it % 64 == 0) {
      const unsigned long long now = globaltimer();
      if (!began) began = now;
      if (now - began > kWaitNs) break;
    }
  }
  *failed = 1;
}

template <bool CLUSTER>
LZ_DEV void ring_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
  if (!try_wait<CLUSTER>(smem_addr(bar), parity)) ring_wait_on<CLUSTER>(smem_addr(bar), parity, failed);
}

// After a wait that gave up: copies still in flight land before the CTA ends.
LZ_DEV void drain_copies() {
  const unsigned long long began = globaltimer();
  for (uint32_t it = 0; it < 100000000u && globaltimer() - began < 20000000ull; ++it) {
  }
}

// Two fp32 operations an instruction.
LZ_DEV uint64_t pair(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
LZ_DEV void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
LZ_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
LZ_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
LZ_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The largest element of a vector; NaN only if all are.
template <typename T>
LZ_DEV float vector_max(uint4 v);
template <>
LZ_DEV float vector_max<float>(uint4 v) {
  return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
template <>
LZ_DEV float vector_max<__nv_bfloat16>(uint4 v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  return fmaxf(m.x, m.y);
}
template <>
LZ_DEV float vector_max<__half>(uint4 v) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
  const float2 m = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  return fmaxf(m.x, m.y);
}

template <typename T>
LZ_DEV void unpack_pairs(uint4 v, uint64_t* p) {
  float f[Elem<T>::N];
  Elem<T>::unpack(v, f);
#pragma unroll
  for (int i = 0; i < Elem<T>::N / 2; ++i) p[i] = pair(f[2 * i], f[2 * i + 1]);
}

// A rank's share of a row: vectors [first, first + count) of those between the
// 16-byte borders; the single elements outside of these are rank 0's.
template <typename T>
LZ_DEV RowHead slice_of(const T* x, long long row, long long vocab, uint32_t rank, uint32_t ranks, int chunk_vecs) {
  const Split<T> sp(x, vocab);
  RowHead h;
  h.row = row, h.lead = sp.lead, h.vecs = sp.vecs;
  const int per = (sp.vecs + (int)ranks - 1) / (int)ranks;
  h.first = min((int)rank * per, sp.vecs);
  h.count = min(per, sp.vecs - h.first);
  h.chunks = (h.count + chunk_vecs - 1) / chunk_vecs;
  return h;
}

// Index of the t-th single element, or -1.
template <typename T>
LZ_DEV long long single_of(const RowHead& h, int t, long long vocab) {
  const long long tail = h.lead + (long long)h.vecs * Elem<T>::N;
  if (t < h.lead) return t;
  return t - h.lead < vocab - tail ? tail + t - h.lead : -1;
}

// log2 of a sum as an integer and a part in [-1/2, 1/2], so that neither is rounded away.
LZ_DEV void log2_parts(float s, float* whole, float* part) {
  const int bits = __float_as_int(s), e = (bits - 0x3f3504f3) >> 23;  // mantissa in [1/sqrt 2, sqrt 2)
  const bool normal = s >= 0x1p-126f && s < INFINITY;
  *whole = normal ? (float)e : 0.f;
  *part = log2f(normal ? __int_as_float(bits - (e << 23)) : s);
}

// A row's normaliser: p_j = 2^((x_j - base) c - ref) / sum.
struct RowSum {
  float base, ref, sum;
  LZ_DEV Norm norm() const {
    float whole, part;
    log2_parts(sum, &whole, &part);
    return {base, (double)ref + (double)whole + (double)part};
  }
};

// What a POLICY row's scalars give; logp2: the token's log-probability in base 2.
struct PolicyOut {
  float ratio, slope;
  bool clipped;
};
LZ_DEV PolicyOut policy_out(const LzLossArgs& a, const RowParams& p, double logp2) {
  PolicyOut o;
  o.ratio = exp2f((float)(logp2 - p.old_logp2));
  o.clipped = (p.adv > 0.f && o.ratio > 1.f + a.clip_high) || (p.adv < 0.f && o.ratio < 1.f - a.clip_low);
  float slope = o.clipped ? 0.f : -p.adv * o.ratio;
  if (a.ref_logp) slope -= a.kl_coef * expm1f((float)((p.ref_logp2 - logp2) * kLn2));
  o.slope = (float)(p.weight * (double)slope);
  return o;
}

// (max, sum) over the `n` lanes' values, n a power of two; the same in every lane.
LZ_DEV void lanes_join(float& m, float& s, int n) {
  float top = m;
  for (int o = n / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  s *= m == -INFINITY ? 1.f : exp2_fast(m - top);  // a sum without a maximum is 0 or NaN
  for (int o = n / 2; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  m = top;
}

// Maximum and sum of a row whose scaled maximum is beyond 32 bits, by one warp.
template <typename T>
LZ_DEV RowSum slow_sum(const T* x, long long n, float c) {
  const int lane = threadIdx.x % 32;
  float m = -INFINITY, s = 0.f;
#pragma unroll 8
  for (long long i = lane; i < n; i += 32) m = fmaxf(m, Elem<T>::get(x[i]));
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
#pragma unroll 8
  for (long long i = lane; i < n; i += 32) s += exp2_fast((Elem<T>::get(x[i]) - m) * c);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  return {m, 0.f, s};
}

// Two rows ahead the teacher's list goes to L2, and then the logits at its ids:
// read only when they are needed, each took up to 3 us behind the rows' stream.
LZ_DEV void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

LZ_DEV void touch_list(const LzLossArgs& a, long long r) {
  const int id_bytes = a.ids64 ? 8 : 4, t_bytes = a.teacher_dtype == LZ_F32 ? 4 : 2;
  for (int k = threadIdx.x % 32 * 16; k < a.top; k += 512) {  // one entry of each 128 bytes at least
    prefetch_l2(static_cast<const char*>(a.ids) + (r * a.top + k) * id_bytes);
    prefetch_l2(static_cast<const char*>(a.teacher) + (r * a.top + k) * t_bytes);
  }
}

template <typename T>
LZ_DEV void touch_logits(const LzLossArgs& a, const T* x, long long r) {
#pragma unroll 4
  for (int k = threadIdx.x % 32; k < a.top; k += 32) {
    const long long id = load_id(a.ids, a.ids64, r * a.top + k);
    if (id >= 0 && id < a.vocab) prefetch_l2(x + id);
  }
}

// A row's scalars, fetched a row ahead.
template <typename T, int KIND>
LZ_DEV void prepare_params(const LzLossArgs& a, const StreamPlan& p, const T* x, long long r, RowParams& out, TopView t,
                           int* hash, float c) {
  const int lane = threadIdx.x % 32;
  if (KIND != LZ_LOSS_DISTILL) {
    if (lane == 0) {
      const long long y = load_id(a.ids, a.ids64, r);
      out.token = y < a.vocab ? (int)y : -1;
      out.xy = y < a.vocab ? Elem<T>::get(x[y]) : 0.f;
      if (KIND == LZ_LOSS_POLICY) {
        out.adv = a.advantages[r];
        out.old_logp2 = (double)a.old_logp[r] * kLog2e;
        out.ref_logp2 = a.ref_logp ? (double)a.ref_logp[r] * kLog2e : 0.0;
        out.weight = (a.weights ? (double)a.weights[r] : 1.0) * a.work[0];
      }
    }
    __syncwarp();
    return;
  }
  float m = -INFINITY;
  bool bad = false;
  for (int first = 0; first < a.top; first += 128) {  // four entries a lane at a time: their loads run together
    long long id[4];
    float v[4];
    T z[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = first + 32 * u + lane;
      id[u] = k < a.top ? load_id(a.ids, a.ids64, r * a.top + k) : -1;
      v[u] = k < a.top ? top_value(a, r, k) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) z[u] = id[u] >= 0 && id[u] < a.vocab ? x[id[u]] : Elem<T>::put(0.f);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = first + 32 * u + lane;
      if (k >= a.top) break;
      if (id[u] < 0) v[u] = -INFINITY;
      bad |= id[u] >= a.vocab;
      t.id[k] = id[u] >= 0 && id[u] < a.vocab ? (int)id[u] : -1;
      t.z[k] = Elem<T>::get(z[u]);
      t.q[k] = v[u];
      m = fmaxf(m, v[u]);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  bad = __any_sync(~0u, bad);
  // Sums over e = exp(v - m); q = e / s.
  float s = 0.f;
  double e_v = 0.0, e_z = 0.0;
  for (int k = lane; k < a.top; k += 32) {
    const float v = t.q[k] - m, e = m == -INFINITY ? 0.f : expf(v);
    t.q[k] = e;
    if (e != 0.f) {  // NaN counts
      s += e;
      e_v += (double)e * (double)v;
      e_z += (double)e * ((double)t.z[k] * (double)c);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s += __shfl_xor_sync(~0u, s, o);
    e_v += __shfl_xor_sync(~0u, e_v, o);
    e_z += __shfl_xor_sync(~0u, e_z, o);
  }
  const float inv = s > 0.f || s != s ? 1.f / s : 0.f;
  for (int k = lane; k < a.top; k += 32) {
    const float q = t.q[k] * inv;
    t.q[k] = q;
    t.share[k] = t.id[k] < 0 ? -1.f : q;
  }
  __syncwarp();
  // Does an id stand in the list twice? Then its first entry gets all shares.
  bool twice = false;
  if (a.top <= kSmallList) {
    for (int k = lane; k < a.top; k += 32) {
      const int id = t.id[k];
      int same = 0;
#pragma unroll 8
      for (int o = 0; o < a.top; ++o) same += t.id[o] == id;
      twice |= id >= 0 && same > 1;
    }
  } else {
    for (int k = lane; k < p.hash; k += 32) hash[k] = -1;
    __syncwarp();
    for (int k = lane; k < a.top; k += 32) {
      const int id = t.id[k];
      if (id < 0) continue;
      for (unsigned h = (unsigned)id * 2654435761u >> 7;; ++h) {  // ends: the table is twice the list
        const int was = atomicCAS(hash + (h & (p.hash - 1)), -1, id);
        twice |= was == id;
        if (was == -1 || was == id) break;
      }
    }
  }
  if (__any_sync(~0u, twice)) {
    for (int k = lane; k < a.top; k += 32) {
      if (t.id[k] < 0) continue;
      float q = t.q[k];
      bool first = true;
      for (int o = 0; o < a.top; ++o) {
        if (t.id[o] != t.id[k] || o == k) continue;
        first &= o > k;
        q += t.q[o];
      }
      t.share[k] = first ? q : -1.f;
    }
  }
  float whole, part;
  log2_parts(s, &whole, &part);
  const double q_sum = (double)s * (double)inv;
  const double q_logq = s == 0.f ? 0.0 : e_v * (double)inv - q_sum * ((double)whole + (double)part) * kLn2, q_z = e_z * (double)inv;
  if (lane == 0) {
    out.weight = (a.weights ? (double)a.weights[r] : 1.0) * a.work[0];
    out.slope = bad ? NAN : m == -INFINITY ? 0.f : (float)-out.weight;
    out.q_logq = q_logq, out.q_z = q_z, out.q_sum = q_sum;
  }
  __syncwarp();
}

constexpr int kBatch = 3;  // vectors a thread has in work at a time

// Sum over a thread's elements of 2^(x c - ref). ref is not the running maximum:
// it is taken from the first batch (as an integer, as above) and moves only when a batch's maximum is more
// than 2^16 above it, which fp32 has room for (2^16 times the vocabulary), so the
// exponentials of a batch wait for no maximum and the branch is seldom taken.
struct LazySum {
  float ref, limit;  // in units of x c, of x; ref is -inf (and taken as 0) before the first batch
  uint64_t neg_ref, sum[2];
  LZ_DEV void init(float c) {
    ref = -INFINITY, neg_ref = 0, sum[0] = sum[1] = 0;
    limit = -3e38f / fmaxf(c, 1.f);  // below this x c is beyond 32 bits: such entries count nothing
  }
  LZ_DEV void raise(float m, float c) {
    const float to = rintf(m * c), f = exp2_fast(ref - to);
    sum[0] = mul2(sum[0], pair(f, f)), sum[1] = mul2(sum[1], pair(f, f));
    ref = to, neg_ref = pair(-ref, -ref);
    limit = m + 16.f / c;
  }
};

template <typename T, int U>
LZ_DEV void batch_sum(const uint4* w, uint64_t c2, uint64_t neg_ref, uint64_t* out) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    uint64_t p[Elem<T>::N / 2];
    unpack_pairs<T>(w[u], p);
#pragma unroll
    for (int i = 0; i < Elem<T>::N / 2; ++i) {
      float lo, hi;
      unpair(fma2(p[i], c2, neg_ref), lo, hi);
      out[i % 2] = add2(out[i % 2], pair(exp2_fast(lo), exp2_fast(hi)));
    }
  }
}

// `first` (of a row): nothing to go by, so the maximum comes first.
template <typename T, int U>
LZ_DEV void take_batch(LazySum& s, const uint4* w, float c, bool first) {
  const uint64_t c2 = pair(c, c);
  float m = vector_max<T>(w[0]);
#pragma unroll
  for (int u = 1; u < U; ++u) m = fmaxf(m, vector_max<T>(w[u]));
  if (first && m > s.limit) s.raise(m, c);
  uint64_t part[2] = {0, 0};
  batch_sum<T, U>(w, c2, s.neg_ref, part);
  if (m > s.limit) {
    s.raise(m, c);
    part[0] = part[1] = 0;
    batch_sum<T, U>(w, c2, s.neg_ref, part);
  }
  s.sum[0] = add2(s.sum[0], part[0]), s.sum[1] = add2(s.sum[1], part[1]);
}

// Warps beside the W that take chunks: one feeds the ring, one has the rows'
// scalars; DISTILL's lists take one more (about 9000 cycles for 64 entries, of
// the 15000 that a slice of 150 KB takes; on one warp they were the bound).
template <int KIND>
constexpr int kHelpers = KIND == LZ_LOSS_DISTILL ? 3 : 2;

template <typename T, int KIND, bool GRAD, int W>
__global__ void __launch_bounds__((W + kHelpers<KIND>) * 32, 1) stream_kernel(const __grid_constant__ LzLossArgs a,
                                                                 const __grid_constant__ StreamPlan plan) {
  constexpr int N = Elem<T>::N, kTake = W * 32;
  constexpr int kChunkVecs = kBatch * kTake, kChunk = 16 * kChunkVecs;
  extern __shared__ __align__(128) char smem[];
  StreamShared& sh = *reinterpret_cast<StreamShared*>(smem);
  char* const lists = smem + sizeof(StreamShared);
  char* const ring = lists + list_bytes(KIND, a.top, plan.hash);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const long long cluster = blockIdx.x / ranks, clusters = gridDim.x / ranks;
  const float c = (float)(kLog2e * (double)a.inv_temperature);
  volatile int* const failed = &sh.failed;
  // Rows of this cluster: i = cluster, cluster + clusters, ... below `limit`, those that count first.
  const long long limit = plan.ordered ? a.rows : min(a.rows, clusters);
  const int active = plan.ordered ? *work_active(a) : 0;
  auto row_at = [&](long long i, long long* r) {
    if (i >= limit) return false;
    *r = plan.ordered ? (long long)work_order(a)[i] : i;
    return plan.ordered ? i < active : row_counts<KIND>(a, i);
  };
  auto head_at = [&](long long i) {
    RowHead h;
    long long r;
    if (row_at(i, &r)) h = slice_of(row_of<T>(a, r), r, a.vocab, rank, ranks, kChunkVecs);
    else h.row = -1;
    return h;
  };
  auto view = [&](int k) {
    float* f = reinterpret_cast<float*>(lists) + k * 4 * a.top;
    return TopView{reinterpret_cast<int*>(f), f + a.top, f + 2 * a.top, f + 3 * a.top};
  };
  if (tid == 0) {
    for (int s = 0; s < plan.slots; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], W);
    }
    for (int k = 0; k < 2; ++k) {
      mbar_init(&sh.parts[k], W);
      mbar_init(&sh.peers[k], 1);
      mbar_init(&sh.dense[k], 1);
      mbar_init(&sh.ready[k], 1);
      mbar_init(&sh.used[k], 1);
    }
    fence_mbar_init();
    *failed = 0;
  }
  if (warp == W + 1 && lane < 2) sh.heads[lane] = head_at(cluster + lane * clusters);
  cluster_sync();

  if (warp == W) {  // ---- streams the slices into the ring
    if (lane == 0) {
      uint32_t slot = 0, round = 0;
      RowHead h = sh.heads[0];
      for (long long i = cluster; h.row >= 0; i += clusters) {
        const RowHead next = head_at(i + clusters);
        const char* from = reinterpret_cast<const char*>(row_of<T>(a, h.row) + h.lead) + (size_t)h.first * 16;
        for (int k = 0; k < h.chunks && !*failed; ++k) {
          if (round) ring_wait<false>(&sh.empty[slot], (round - 1) & 1, failed);
          if (*failed) break;
          const int vecs = min(kChunkVecs, h.count - k * kChunkVecs);
          bulk_g2s(ring + (size_t)slot * kChunk, from + (size_t)k * kChunk, vecs * 16, &sh.full[slot]);
          if (++slot == (uint32_t)plan.slots) slot = 0, ++round;
        }
        h = next;
      }
      if (*failed) drain_copies();
    }
    __syncwarp();
  } else if (warp < W) {  // ---- sums, then the dense gradient
    uint32_t slot = 0, round = 0;      // where the sums are
    uint32_t again = 0;                // where the gradient is
    LazySum sum;
    sum.init(c);
    int done = 0;  // chunks of the row that are in `sum`
    // Chunks [done, upto) of a row, two at a time.
    auto take = [&](const RowHead& h, int upto) {
      for (; done < upto; ++done) {
        const int vecs = h.count - done * kChunkVecs;
        ring_wait<false>(&sh.full[slot], round & 1, failed);
        const uint4* v = reinterpret_cast<const uint4*>(ring + (size_t)slot * kChunk) + tid;
        if (vecs >= kChunkVecs) {
          uint4 w[kBatch];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) w[u] = v[u * kTake];
          take_batch<T, kBatch>(sum, w, c, done == 0);
        } else {
          for (int j = tid; j < vecs; j += kTake, v += kTake) take_batch<T, 1>(sum, v, c, true);
        }
        if (!GRAD) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.empty[slot]);
        }
        if (++slot == (uint32_t)plan.slots) slot = 0, ++round;
      }
    };
    uint32_t turn = 0;
    for (;; ++turn) {
      // The row's head is there, and its place in `warp_part` free, when the row two before it is done with.
      const int k = turn & 1;
      if (!GRAD && turn >= 2) ring_wait<false>(&sh.dense[k], ((turn - 2) >> 1) & 1, failed);
      const RowHead h = sh.heads[turn & 3];
      if (h.row < 0) break;
      const long long single = rank == 0 && tid < 2 * N ? single_of<T>(h, tid, a.vocab) : -1;
      float alone = 0.f;
      if (single >= 0) alone = Elem<T>::get(row_of<T>(a, h.row)[single]);
      take(h, h.chunks);
      if (single >= 0) {
        if (alone > sum.limit) sum.raise(alone, c);
        float neg_ref, unused;
        unpair(sum.neg_ref, neg_ref, unused);
        sum.sum[0] = add2(sum.sum[0], pair(exp2_fast(fmaf(alone, c, neg_ref)), 0.f));
      }
      float s0, s1, s2, s3;
      unpair(sum.sum[0], s0, s1), unpair(sum.sum[1], s2, s3);
      float m = sum.ref, all = (s0 + s1) + (s2 + s3);
      lanes_join(m, all, 32);
      if (lane == 0) {
        sh.warp_part[k][warp] = make_float2(m, all);
        mbar_arrive(&sh.parts[k]);
      }
      sum.init(c);
      done = 0;
      if (!GRAD) continue;
      const RowHead& next = sh.heads[(turn + 1) & 3];
      if (next.row >= 0) take(next, min(plan.early, next.chunks));
      ring_wait<false>(&sh.dense[k], (turn >> 1) & 1, failed);
      const RowDense d = sh.row_dense[k];
      T* out = static_cast<T*>(a.grad) + h.row * a.vocab;
      const uint64_t c2 = pair(c, c), f2 = pair(d.f, d.f), off2 = pair(-d.ref, -d.ref);
      for (int ch = 0; ch < h.chunks; ++ch) {
        const uint4* v = reinterpret_cast<const uint4*>(ring + (size_t)again * kChunk);
        uint4* o = reinterpret_cast<uint4*>(out + h.lead) + h.first + (long long)ch * kChunkVecs;
        const int vecs = h.count - ch * kChunkVecs;
        if (d.f == 0.f) {
#pragma unroll
          for (int j = tid; j < kChunkVecs; j += kTake)
            if (j < vecs) st_cs_v4(o + j, make_uint4(0, 0, 0, 0));
        } else if (d.base == 0.f) {
          uint4 w[kBatch];
#pragma unroll
          for (int u = 0; u < kBatch; ++u)
            if (tid + u * kTake < vecs) w[u] = v[tid + u * kTake];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            if (u * kTake >= vecs) break;
            uint64_t p[N / 2];
            float e[N];
            unpack_pairs<T>(w[u], p);
#pragma unroll
            for (int q = 0; q < N / 2; ++q) {
              float lo, hi;
              unpair(fma2(p[q], c2, off2), lo, hi);
              unpair(mul2(f2, pair(exp2_fast(lo), exp2_fast(hi))), e[2 * q], e[2 * q + 1]);
            }
            if (tid + u * kTake < vecs) st_cs_v4(o + tid + u * kTake, Elem<T>::pack(e));
          }
        } else {
          for (int j = tid; j < min(vecs, kChunkVecs); j += kTake) {
            float e[N];
            Elem<T>::unpack(v[j], e);
#pragma unroll
            for (int q = 0; q < N; ++q) e[q] = d.f * exp2_fast((e[q] - d.base) * c);
            st_cs_v4(o + j, Elem<T>::pack(e));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[again]);
        if (++again == (uint32_t)plan.slots) again = 0;
      }
      if (single >= 0)
        out[single] = Elem<T>::put(d.f == 0.f ? 0.f : d.f * exp2_fast(fmaf(alone - d.base, c, -d.ref)));
    }
    __syncwarp();
    if (GRAD) {
      if (lane == 0) mbar_arrive(&sh.parts[turn & 1]);  // the last row is written
      for (long long i = (plan.ordered ? active : 0) + cluster; i < limit; i += clusters) {
        long long r;
        if (row_at(i, &r)) continue;
        T* out = static_cast<T*>(a.grad) + r * a.vocab;
        const RowHead h = slice_of(out, r, a.vocab, rank, ranks, kChunkVecs);
        uint4* o = reinterpret_cast<uint4*>(out + h.lead) + h.first;
        for (int j = tid; j < h.count; j += kTake) st_cs_v4(o + j, make_uint4(0, 0, 0, 0));
        const long long single = rank == 0 && tid < 2 * N ? single_of<T>(h, tid, a.vocab) : -1;
        if (single >= 0) out[single] = Elem<T>::put(0.f);
      }
    }
  } else if (KIND == LZ_LOSS_DISTILL && warp == W + 2) {  // ---- the teacher's lists, a row ahead
    int* const hash = reinterpret_cast<int*>(lists) + 8 * a.top;
    long long r, to_come;
    for (uint32_t turn = 0; row_at(cluster + (long long)turn * clusters, &r); ++turn) {
      const int k = turn & 1;
      if (row_at(cluster + (long long)(turn + 2) * clusters, &to_come)) touch_list(a, to_come);
      if (turn >= 2) ring_wait<false>(&sh.used[k], ((turn - 2) >> 1) & 1, failed);
      prepare_params<T, KIND>(a, plan, row_of<T>(a, r), r, sh.params[k], view(k), hash, c);
      if (lane == 0) mbar_arrive(&sh.ready[k]);
      if (row_at(cluster + (long long)(turn + 1) * clusters, &to_come))
        touch_logits(a, row_of<T>(a, to_come), to_come);
    }
    __syncwarp();
  } else {  // ---- joins the sums; the rows' scalars, outputs and sparse entries
    double loss = 0.0;
    RowHead before = {-1};  // the row whose dense part is being written, its slope, token and sum
    float before_slope = 0.f, before_xy = 0.f;
    int before_token = -1;
    RowSum before_n = {0.f, 0.f, 1.f};
    auto sparse = [&](int k) {
      if (!GRAD || before.row < 0 || before_slope == 0.f) return;
      T* out = static_cast<T*>(a.grad) + before.row * a.vocab;
      const long long lo = before.lead + (long long)before.first * N, hi = lo + (long long)before.count * N;
      const long long tail = before.lead + (long long)before.vecs * N;
      const float inv = 1.f / before_n.sum;
      auto put = [&](int id, float z, float t) {
        if (!((id >= lo && id < hi) || (rank == 0 && (id < before.lead || id >= tail)))) return;
        const float p = exp2_fast(fmaf(z - before_n.base, c, -before_n.ref)) * inv;
        out[id] = Elem<T>::put(before_slope * a.inv_temperature * (t - p));
      };
      if (KIND == LZ_LOSS_DISTILL) {
        const TopView t = view(k);
        for (int j = lane; j < a.top; j += 32)
          if (!(t.share[j] < 0.f)) put(t.id[j], t.z[j], t.share[j]);
      } else if (lane == 0 && before_token >= 0) {
        put(before_token, before_xy, 1.f);
      }
    };
    auto prepare = [&](const RowHead& h, int k) {
      if (KIND != LZ_LOSS_DISTILL && h.row >= 0)
        prepare_params<T, KIND>(a, plan, row_of<T>(a, h.row), h.row, sh.params[k], TopView{}, nullptr, c);
    };
    prepare(sh.heads[0], 0);
    uint32_t turn = 0;
    for (;; ++turn) {
      const RowHead h = sh.heads[turn & 3];
      if (h.row < 0) break;
      const int k = turn & 1;
      const RowHead later = head_at(cluster + (long long)(turn + 2) * clusters);
      ring_wait<false>(&sh.parts[k], (turn >> 1) & 1, failed);
      float2 v = sh.warp_part[k][lane % W];
      lanes_join(v.x, v.y, W);
      if (ranks > 1) {
        if (lane == 0) mbar_expect(&sh.peers[k], ranks * (uint32_t)sizeof(float2));
        if (lane < ranks) send_to_peer(&sh.peer_part[k][rank], v, &sh.peers[k], lane);
        __syncwarp();
        ring_wait<true>(&sh.peers[k], (turn >> 1) & 1, failed);
        v = sh.peer_part[k][lane % ranks];
        lanes_join(v.x, v.y, (int)ranks);
      }
      RowSum n = {0.f, v.x, v.y};
      if (isinf(v.x)) n = slow_sum(row_of<T>(a, h.row), a.vocab, c);
      if (KIND == LZ_LOSS_DISTILL) ring_wait<false>(&sh.ready[k], (turn >> 1) & 1, failed);
      const RowParams& p = sh.params[k];
      const Norm norm = n.norm();
      const double logp2 = p.token < 0 ? (double)NAN : ((double)p.xy - (double)norm.base) * (double)c - norm.lse2;
      PolicyOut o = {0.f, 0.f, false};
      if (KIND == LZ_LOSS_POLICY) o = policy_out(a, p, logp2);
      const float slope = KIND == LZ_LOSS_DISTILL ? p.slope : o.slope;
      if (lane == 0) {
        sh.row_dense[k] = {slope == 0.f ? 0.f : -slope * a.inv_temperature / n.sum, n.base, n.ref};
        sh.heads[(turn + 2) & 3] = later;
        mbar_arrive(&sh.dense[k]);
      }
      sparse(k ^ 1);
      __syncwarp();
      if (KIND == LZ_LOSS_DISTILL && turn && lane == 0) mbar_arrive(&sh.used[k ^ 1]);  // by the row before
      double kl = 0.0;
      if (KIND == LZ_LOSS_DISTILL) {
        kl = p.q_logq - kLn2 * (p.q_z - p.q_sum * norm.lse2);
        if (norm.base != 0.f) {
          const TopView t = view(k);
          kl = 0.0;
          for (int j = lane; j < a.top; j += 32)
            if (t.q[j] != 0.f)
              kl += (double)t.q[j] * (log((double)t.q[j]) -
                                      (((double)t.z[j] - (double)norm.base) * (double)c - norm.lse2) * kLn2);
#pragma unroll
          for (int o2 = 16; o2; o2 >>= 1) kl += __shfl_xor_sync(~0u, kl, o2);
        }
        if (isnan(p.slope)) kl = NAN;
      }
      if (rank == 0 && lane == 0) {
        double each = kl;
        if (KIND != LZ_LOSS_DISTILL) a.logp[h.row] = (float)(logp2 * kLn2);
        if (KIND == LZ_LOSS_POLICY) {
          const double lo = 1.0 - (double)a.clip_low, hi = 1.0 + (double)a.clip_high;
          each = -(double)p.adv * (o.clipped ? (p.adv > 0.f ? hi : lo) : (double)o.ratio);
          if (a.ref_logp) {
            const double d = (double)a.ref_logp[h.row] - logp2 * kLn2, e = expm1(d) - d;
            a.kl[h.row] = (float)e;
            each += (double)a.kl_coef * e;
          }
          a.clipped[h.row] = o.clipped;
        }
        if (KIND == LZ_LOSS_DISTILL) a.kl[h.row] = (float)kl;
        if (KIND != LZ_LOSS_LOGP) loss += p.weight * each;
        work_norm(a)[h.row] = make_double2(norm.base, norm.lse2);
        work_slope(a)[h.row] = KIND == LZ_LOSS_LOGP ? logp2 * kLn2 : (double)slope;
      }
      before = h, before_n = n, before_slope = slope, before_xy = p.xy, before_token = p.token;
      __syncwarp();
      prepare(sh.heads[(turn + 1) & 3], k ^ 1);
    }
    if (GRAD) {
      ring_wait<false>(&sh.parts[turn & 1], (turn >> 1) & 1, failed);
      sparse((turn & 1) ^ 1);
    }
    if (rank == 0) {
      long long r;
      for (long long i = (plan.ordered ? active : 0) + cluster + lane * clusters; i < limit; i += 32 * clusters) {
        if (row_at(i, &r)) continue;
        if (KIND != LZ_LOSS_DISTILL) a.logp[r] = 0.f;
        if (KIND == LZ_LOSS_DISTILL || (KIND == LZ_LOSS_POLICY && a.ref_logp)) a.kl[r] = 0.f;
        if (KIND == LZ_LOSS_POLICY) a.clipped[r] = 0;
        work_norm(a)[r] = make_double2(0.0, 0.0);
        work_slope(a)[r] = 0.0;
      }
      if (*failed) {
        loss = NAN;
        for (long long i = cluster + lane * clusters; i < limit; i += 32 * clusters) {
          row_at(i, &r);
          if (KIND != LZ_LOSS_DISTILL) a.logp[r] = NAN;
          if (KIND == LZ_LOSS_DISTILL || (KIND == LZ_LOSS_POLICY && a.ref_logp)) a.kl[r] = NAN;
        }
      }
      if (KIND != LZ_LOSS_LOGP) {  // the cluster that is done last adds the losses up, in the clusters' order
        int last = 0;
        if (lane == 0) {
          work_loss(a)[cluster] = loss;
          __threadfence();
          last = atomicAdd(work_ticket(a), 1u) == (unsigned)clusters - 1;
        }
        if (__shfl_sync(~0u, last, 0)) {
          __threadfence();
          double s = 0.0;
          for (long long j = lane; j < clusters; j += 32) s += __ldcg(work_loss(a) + j);
#pragma unroll
          for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
          if (lane == 0) *a.loss = (float)s;
        }
      }
    }
    __syncwarp();
  }
  cluster_sync();  // no CTA leaves while a peer may still write to it
}

// The gradient alone, for rows whose sums and slopes are known (LOGP, POLICY). A
// chunk is a piece of work of its own: what it takes from its row travels in the
// ring slot's head. The feeding warp works the heads of its next 32 chunks out
// at once, a lane each, and issues them in turn.
struct ChunkHead {
  void* out;             // first vector of the chunk
  const void* row;       // logits of the row and, with `singles`, its gradient row
  void* out_row;
  int vecs, token_vec, token_at;  // the vector that holds the token (-1: none) and its place in it
  int singles, lead, tail;        // 1: the row's single elements go with this chunk
  float f, base, ref, token_value;
  int token;
};

struct alignas(128) GradShared {
  uint64_t full[kMaxSlots], empty[kMaxSlots];
  ChunkHead heads[kMaxSlots];
  int failed;
};

template <typename T, int KIND, int W>
__global__ void __launch_bounds__((W + 1) * 32, 1) stream_grad_kernel(const __grid_constant__ LzLossArgs a, int slots) {
  constexpr int N = Elem<T>::N, kTake = W * 32;
  constexpr int kChunkVecs = kBatch * kTake, kChunk = 16 * kChunkVecs;
  extern __shared__ __align__(128) char smem[];
  GradShared& sh = *reinterpret_cast<GradShared*>(smem);
  char* const ring = smem + sizeof(GradShared);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const float c = (float)(kLog2e * (double)a.inv_temperature);
  volatile int* const failed = &sh.failed;
  const float up = a.upstream ? *a.upstream : 1.f;
  if (!a.fresh && up == 1.f) return;
  if (tid == 0) {
    for (int s = 0; s < slots; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], W);
    }
    fence_mbar_init();
    *failed = 0;
  }
  __syncthreads();
  const int per_row = (int)((a.vocab / N + kChunkVecs - 1) / kChunkVecs);  // chunks of a row, the last of them maybe empty
  const long long all = a.rows * per_row;

  if (warp == W) {
    uint32_t slot = 0, round = 0;
    for (long long first = blockIdx.x; first < all; first += 32ll * gridDim.x) {
      const long long g = first + (long long)lane * gridDim.x;
      ChunkHead h = {};
      const char* from = nullptr;
      if (g < all) {
        const long long r = g / per_row;
        const int piece = (int)(g % per_row);
        const T* x = row_of<T>(a, r);
        T* out = static_cast<T*>(a.grad) + r * a.vocab;
        const double2 norm = work_norm(a)[r];
        const long long y = load_id(a.ids, a.ids64, r);
        const double slope = row_slope_for<KIND>(a, r, y, up);
        const Split<T> sp(x, a.vocab);
        h.vecs = max(0, min(kChunkVecs, sp.vecs - piece * kChunkVecs));
        const long long at = sp.lead + (long long)piece * kChunkVecs * N;
        h.out = out + at;
        h.row = x, h.out_row = out;
        h.singles = piece == 0, h.lead = sp.lead, h.tail = (int)(a.vocab - sp.lead) % N;
        h.base = (float)norm.x, h.ref = (float)norm.y;
        const double left = (double)h.ref - norm.y;  // at most half a step of ref: 2^left is 1 + left ln 2
        h.f = slope == 0.0 ? 0.f : (float)(-slope * a.inv_temperature * (1.0 + left * kLn2));
        h.token = -1, h.token_vec = -1;
        if (y >= 0 && y < a.vocab && h.f != 0.f) {
          const long long in = y - at;
          if (in >= 0 && in < (long long)h.vecs * N) h.token_vec = (int)(in / N), h.token_at = (int)(in % N);
          else if (h.singles && (y < sp.lead || y >= a.vocab - h.tail)) h.token = (int)y;
          if (h.token_vec >= 0 || h.token >= 0) {
            const float p = exp2_fast(fmaf(Elem<T>::get(x[y]) - h.base, c, -h.ref)) * (float)(1.0 + left * kLn2);
            h.token_value = (float)(slope * a.inv_temperature) * (1.f - p);
          }
        }
        from = reinterpret_cast<const char*>(x + at);
      }
      for (int l = 0; l < 32 && first + (long long)l * gridDim.x < all; ++l) {
        if (lane == l) {
          if (round) ring_wait<false>(&sh.empty[slot], (round - 1) & 1, failed);
          if (!*failed) {
            sh.heads[slot] = h;
            if (h.f != 0.f && h.vecs > 0) bulk_g2s(ring + (size_t)slot * kChunk, from, h.vecs * 16, &sh.full[slot]);
            else mbar_arrive(&sh.full[slot]);  // nothing to read
          }
        }
        __syncwarp();
        if (++slot == (uint32_t)slots) slot = 0, ++round;
      }
    }
    if (*failed) drain_copies();
    __syncwarp();
  } else {
    uint32_t slot = 0, round = 0;
    for (long long g = blockIdx.x; g < all; g += gridDim.x) {
      ring_wait<false>(&sh.full[slot], round & 1, failed);
      const ChunkHead& h = sh.heads[slot];
      const uint4* v = reinterpret_cast<const uint4*>(ring + (size_t)slot * kChunk) + tid;
      uint4* o = static_cast<uint4*>(h.out) + tid;
      const int vecs = *failed ? 0 : h.vecs;
      const float f = *failed ? 0.f : h.f, base = h.base, ref = h.ref;
      const int token_vec = h.token_vec;
      if (f == 0.f) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (tid + u * kTake < vecs) st_cs_v4(o + u * kTake, make_uint4(0, 0, 0, 0));
      } else {
        uint4 w[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (tid + u * kTake < vecs) w[u] = v[u * kTake];
        const uint64_t c2 = pair(c, c), f2 = pair(f, f), off2 = pair(-ref, -ref);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (u * kTake >= vecs) break;
          float e[N];
          if (base == 0.f) {
            uint64_t p[N / 2];
            unpack_pairs<T>(w[u], p);
#pragma unroll
            for (int q = 0; q < N / 2; ++q) {
              float lo, hi;
              unpair(fma2(p[q], c2, off2), lo, hi);
              unpair(mul2(f2, pair(exp2_fast(lo), exp2_fast(hi))), e[2 * q], e[2 * q + 1]);
            }
          } else {
            Elem<T>::unpack(w[u], e);
#pragma unroll
            for (int q = 0; q < N; ++q) e[q] = f * exp2_fast(fmaf(e[q] - base, c, -ref));
          }
          if (tid + u * kTake < vecs) st_cs_v4(o + u * kTake, Elem<T>::pack(e));
        }
        if (token_vec >= 0 && token_vec % kTake == tid)  // over its vector, by the thread that wrote it
          reinterpret_cast<T*>(static_cast<uint4*>(h.out) + token_vec)[h.token_at] = Elem<T>::put(h.token_value);
      }
      if (h.singles && tid < h.lead + h.tail && !*failed) {
        const long long i = tid < h.lead ? tid : a.vocab - h.tail + tid - h.lead;
        float e = 0.f;
        if (f != 0.f) e = i == h.token ? h.token_value : f * exp2_fast(fmaf(Elem<T>::get(static_cast<const T*>(h.row)[i]) - base, c, -ref));
        static_cast<T*>(h.out_row)[i] = Elem<T>::put(e);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[slot]);
      if (++slot == (uint32_t)slots) slot = 0, ++round;
    }
    if (*failed)  // a wait gave up: the gradient is NaN, not stale
      for (long long i = tid; i < a.rows * a.vocab; i += kTake)
        static_cast<T*>(a.grad)[i] = Elem<T>::put(NAN);
  }
}

// Preference loss of one pair a CTA: sums of its two sequences' log-probabilities
// (means where `normalized`), h = beta ((c - ref_c) - (r - ref_r)), loss
// -(1 - eps) log sigmoid(h) - eps log sigmoid(-h), and the slope of every row
// that counts (the others' are zero before the launch).
__global__ void __launch_bounds__(kThreads) pair_kernel(const __grid_constant__ LzPairArgs a) {
  __shared__ double red[kWarps];
  __shared__ bool last;
  const long long n = a.rows;
  const long long pair = blockIdx.x;
  float* slope = reinterpret_cast<float*>(a.work + 1 + a.pairs);
  const double* logp = a.logp_work + LZ_LOSS_WORK_HEAD + 2 * n;  // as work_slope
  auto offset = [&](long long s) { return a.offsets ? load_id(a.offsets, a.offsets64, s) : s * a.length; };
  long long begin[2], end[2];
  double reward[2], per[2];
  bool bad = false;
  for (int k = 0; k < 2; ++k) {
    const long long s = pair + k * a.pairs;
    begin[k] = offset(s), end[k] = offset(s + 1);
    // offsets that do not rise within the rows: the loss is NaN, nothing outside is touched
    if (begin[k] < 0 || begin[k] > end[k] || end[k] > n) bad = true, begin[k] = end[k] = 0;
    double sum = 0.0, count = 0.0;
    for (long long r = begin[k] + threadIdx.x; r < end[k]; r += kThreads)
      if (load_id(a.ids, a.ids64, r) >= 0) sum += logp[r], count += 1.0;
    sum = block_sum(sum, red);
    count = block_sum(count, red);
    per[k] = a.normalized ? 1.0 / (count > 1.0 ? count : 1.0) : 1.0;
    reward[k] = a.beta * (sum * per[k] - (a.ref_logp ? (double)a.ref_logp[s] : 0.0));
    if (threadIdx.x == 0) a.rewards[s] = bad ? NAN : (float)reward[k];
  }
  const double h = bad ? (double)NAN : reward[0] - reward[1], soft = log1p(exp(-fabs(h)));
  const double up = soft + (h < 0.0 ? -h : 0.0), down = soft + (h > 0.0 ? h : 0.0);
  const double dh = (a.smoothing / (1.0 + exp(-h)) - (1.0 - a.smoothing) / (1.0 + exp(h))) * a.beta / (double)a.pairs;
  for (int k = 0; k < 2; ++k)
    for (long long r = begin[k] + threadIdx.x; r < end[k]; r += kThreads)
      if (load_id(a.ids, a.ids64, r) >= 0) slope[r] = (float)((k ? -dh : dh) * per[k]);
  if (threadIdx.x == 0) a.work[1 + pair] = (1.0 - a.smoothing) * up + a.smoothing * down;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(reinterpret_cast<unsigned*>(a.work), 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
  for (long long p = threadIdx.x; p < a.pairs; p += kThreads) s += __ldcg(a.work + 1 + p);
  s = block_sum(s, red);
  if (threadIdx.x == 0) *a.loss = (float)(s / (double)a.pairs);
}

// Makes the tensors' device current for a launch and the caller's again after it.
struct OnDevice {
  int before = -1;
  cudaError_t rc;
  explicit OnDevice(int device) {
    rc = cudaGetDevice(&before);
    if (rc == cudaSuccess && before != device) rc = cudaSetDevice(device);
    else before = -1;
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

int grid_for(int device, long long rows, int* grid) {
  int sms = 0;
  LZ_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  const long long cap = (long long)sms * 4;  // 4 CTAs of 512 threads fill an SM
  *grid = (int)(rows < cap ? rows : cap);
  return LZE_OK;
}

size_t top_bytes(const LzLossArgs* a) { return a->kind == LZ_LOSS_DISTILL ? sizeof(Top) : 0; }

// The stream kernel's launch for these arguments, or false where a CTA a row
// does better or is the only way: rows that fit no cluster's shared memory,
// rows and gradient rows at different offsets from a 16-byte border, small rows.
struct StreamLaunch {
  StreamPlan plan;
  int clusters, ranks;
  size_t smem;
};

// Whether rows can be streamed: not small, and each row and its gradient at the
// same offset from a 16-byte border.
template <typename T>
bool streams(const LzLossArgs* a, bool grad) {
  const long long size = sizeof(T), row = a->vocab * size;
  if (row < 16384 || a->rows > INT32_MAX) return false;
  if (!grad) return true;
  return ((uintptr_t)a->logits ^ (uintptr_t)a->grad) % 16 == 0 &&
         (a->inner >= a->rows || (a->outer_stride * size - a->inner * row) % 16 == 0) &&
         (a->inner <= 1 || (a->inner_stride * size - row) % 16 == 0);
}

constexpr int kStreamWarps = 16;
constexpr int kChunk = 16 * kBatch * kStreamWarps * 32;  // bytes of a ring slot: a batch of every thread
constexpr int kSharedMax = 232448;
constexpr int kMaxDevices = 64;

template <typename T, int KIND, bool GRAD>
int plan_stream(const LzLossArgs* a, StreamLaunch* l, bool* fits) {
  *fits = false;
  const long long row = a->vocab * (long long)sizeof(T);
  if (!streams<T>(a, GRAD)) return LZE_OK;
  int hash = 0;
  if (KIND == LZ_LOSS_DISTILL && a->top > kSmallList)
    for (hash = 32; hash < 2 * a->top;) hash *= 2;
  const int fixed = (int)sizeof(StreamShared) + list_bytes(KIND, a->top, hash);
  const int slots = (kSharedMax - fixed) / kChunk < kMaxSlots ? (kSharedMax - fixed) / kChunk : kMaxSlots;
  auto kernel = stream_kernel<T, KIND, GRAD, kStreamWarps>;
  static std::atomic<bool> known[kMaxDevices];
  static std::atomic<int> resident[kMaxDevices][4];
  if (a->device < 0 || a->device >= kMaxDevices) return LZE_OK;
  if (!known[a->device].load(std::memory_order_acquire)) {
    LZ_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax));
    for (int k = 0; k < 4; ++k) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute at[1] = {};
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim = {1u << k, 1, 1};
      cfg.gridDim = dim3(148 * 8), cfg.blockDim = dim3((kStreamWarps + kHelpers<KIND>) * 32), cfg.dynamicSmemBytes = kSharedMax;
      cfg.attrs = at, cfg.numAttrs = 1;
      int g = 0;
      LZ_CUDA_TRY(cudaOccupancyMaxActiveClusters(&g, kernel, &cfg));
      resident[a->device][k].store(g, std::memory_order_relaxed);
    }
    known[a->device].store(true, std::memory_order_release);
  }
  double best = 0.0;
  int chunks = 0;
  for (int k = 0; k < 4; ++k) {
    const int ranks = 1 << k, g = resident[a->device][k].load(std::memory_order_relaxed);
    const long long slice = (row + ranks - 1) / ranks;
    if (g < 1 || (GRAD && (slice + 16 + kChunk - 1) / kChunk > slots)) continue;
    const double cost = (double)((a->rows + g - 1) / g) * ((double)slice * (GRAD ? 2 : 1) + 50e3);
    if (best != 0.0 && cost >= best) continue;
    best = cost;
    l->ranks = ranks;
    l->clusters = (int)(a->rows < g ? a->rows : g);
    chunks = (int)((slice + 16 + kChunk - 1) / kChunk);
  }
  if (best == 0.0) return LZE_OK;
  l->plan = {slots, slots - chunks, a->rows > l->clusters, hash};
  l->smem = fixed + (size_t)slots * kChunk;
  *fits = true;
  return LZE_OK;
}

template <typename T, int KIND, bool GRAD>
int launch_stream(const LzLossArgs* a, const StreamLaunch& l, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)l.ranks, 1, 1};
  cfg.gridDim = dim3(l.clusters * l.ranks), cfg.blockDim = dim3((kStreamWarps + kHelpers<KIND>) * 32);
  cfg.dynamicSmemBytes = l.smem, cfg.stream = s, cfg.attrs = at, cfg.numAttrs = 1;
  LZ_CUDA_TRY(cudaLaunchKernelEx(&cfg, stream_kernel<T, KIND, GRAD, kStreamWarps>, *a, l.plan));
  return LZE_OK;
}

template <typename T, int KIND, bool GRAD>
int launch_forward_as(const LzLossArgs* a, cudaStream_t s) {
  StreamLaunch l = {};
  bool fits = false;
  if (a->rows)
    if (const int rc = plan_stream<T, KIND, GRAD>(a, &l, &fits)) return rc;
  if (KIND != LZ_LOSS_LOGP || l.plan.ordered) {
    head_kernel<KIND><<<1, kThreads, 0, s>>>(*a, l.plan.ordered);
    LZ_CUDA_TRY(cudaGetLastError());
  }
  if (!a->rows) return LZE_OK;
  if (fits) return launch_stream<T, KIND, GRAD>(a, l, s);
  int grid = 0;
  if (const int rc = grid_for(a->device, a->rows, &grid)) return rc;
  forward_kernel<T, KIND, GRAD><<<grid, kThreads, top_bytes(a), s>>>(*a);
  LZ_CUDA_TRY(cudaGetLastError());
  return LZE_OK;
}

template <typename T, int KIND>
int launch_forward(const LzLossArgs* a, cudaStream_t s) {
  if constexpr (KIND == LZ_LOSS_LOGP) return launch_forward_as<T, KIND, false>(a, s);
  else return a->grad ? launch_forward_as<T, KIND, true>(a, s) : launch_forward_as<T, KIND, false>(a, s);
}

template <typename T, int KIND>
int launch_stream_grad(const LzLossArgs* a, cudaStream_t s) {
  auto kernel = stream_grad_kernel<T, KIND, kStreamWarps>;
  static std::atomic<int> sms[kMaxDevices];
  int n = sms[a->device].load(std::memory_order_acquire);
  if (!n) {
    LZ_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax));
    LZ_CUDA_TRY(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, a->device));
    sms[a->device].store(n, std::memory_order_release);
  }
  // Four chunks ahead: with nine, as many as fit, the reads queue in front of the
  // writes (4096 rows of 151936 in bf16, half of them read: 408 us a step against 432).
  constexpr int slots = 4;
  static_assert(slots * kChunk + sizeof(GradShared) <= kSharedMax && slots <= kMaxSlots, "ring");
  kernel<<<n, (kStreamWarps + 1) * 32, sizeof(GradShared) + (size_t)slots * kChunk, s>>>(*a, slots);
  LZ_CUDA_TRY(cudaGetLastError());
  return LZE_OK;
}

template <typename T, int KIND>
int launch_backward(const LzLossArgs* a, cudaStream_t s) {
  if (!a->rows) return LZE_OK;
  if constexpr (KIND != LZ_LOSS_DISTILL)
    if (streams<T>(a, true) && a->device < kMaxDevices) return launch_stream_grad<T, KIND>(a, s);
  int grid = 0;
  if (const int rc = grid_for(a->device, a->rows, &grid)) return rc;
  backward_kernel<T, KIND><<<grid, kThreads, top_bytes(a), s>>>(*a);
  LZ_CUDA_TRY(cudaGetLastError());
  return LZE_OK;
}

template <typename T>
int run_kind(const LzLossArgs* a, cudaStream_t s, bool forward) {
  switch (a->kind) {
    case LZ_LOSS_LOGP:
      return forward ? launch_forward<T, LZ_LOSS_LOGP>(a, s) : launch_backward<T, LZ_LOSS_LOGP>(a, s);
    case LZ_LOSS_POLICY:
      return forward ? launch_forward<T, LZ_LOSS_POLICY>(a, s) : launch_backward<T, LZ_LOSS_POLICY>(a, s);
    default:
      return forward ? launch_forward<T, LZ_LOSS_DISTILL>(a, s) : launch_backward<T, LZ_LOSS_DISTILL>(a, s);
  }
}

int run(const LzLossArgs* a, cudaStream_t s, bool forward) {
  if (a->kind < LZ_LOSS_LOGP || a->kind > LZ_LOSS_DISTILL || a->rows < 0 || a->vocab < 1 || a->vocab > INT32_MAX ||
      a->inner < 1 || a->inv_temperature <= 0.f ||
      (a->kind == LZ_LOSS_DISTILL && (a->top < 1 || a->top > LZ_LOSS_MAX_TOP))) {
    lz_set_error("loss: bad arguments (kind %d, rows %lld, vocabulary %lld, top %d)", a->kind, a->rows, a->vocab, a->top);
    return LZE_ARG;
  }
  const OnDevice on(a->device);
  LZ_CUDA_TRY(on.rc);
  switch (a->dtype) {
    case LZ_F32: return run_kind<float>(a, s, forward);
    case LZ_F16: return run_kind<__half>(a, s, forward);
    case LZ_BF16: return run_kind<__nv_bfloat16>(a, s, forward);
  }
  lz_set_error("loss: dtype %d", a->dtype);
  return LZE_ARG;
}

}  // namespace

extern "C" int lz_loss_forward(const LzLossArgs* a, cudaStream_t stream) { return run(a, stream, true); }

extern "C" int lz_loss_backward(const LzLossArgs* a, cudaStream_t stream) { return run(a, stream, false); }

extern "C" int lz_loss_pairs(const LzPairArgs* a, cudaStream_t stream) {
  if (a->pairs < 1 || a->pairs > INT32_MAX || a->rows < 0 || (!a->offsets && a->length * 2 * a->pairs != a->rows)) {
    lz_set_error("preference loss: bad arguments (%lld pairs, %lld rows)", a->pairs, a->rows);
    return LZE_ARG;
  }
  const OnDevice on(a->device);
  LZ_CUDA_TRY(on.rc);
  LZ_CUDA_TRY(cudaMemsetAsync(a->work, 0, sizeof(double) * (1 + a->pairs) + sizeof(float) * a->rows, stream));
  pair_kernel<<<(unsigned)a->pairs, kThreads, 0, stream>>>(*a);
  LZ_CUDA_TRY(cudaGetLastError());
  return LZE_OK;
}
