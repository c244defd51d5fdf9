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
// maximum (0 while it is -inf, so that rows of -inf sum to 0 and not to NaN).
// A NaN or +inf among the logits makes the sum NaN.
struct Running {
  float max, ref, sum;
  LZ_DEV void init() { max = -INFINITY, ref = 0.f, sum = 0.f; }
  LZ_DEV void raise(float m) {
    if (m > max) {
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
  const float a = slope == 0.0 ? 0.f : (float)(-slope * inv_t * exp2((double)l - norm.lse2));
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
#pragma unroll 4
  for (int i = threadIdx.x; i < sp.vecs; i += kThreads) {
    float f[N];
    Elem<T>::unpack(__ldg(v + i), f);
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = a * exp2_fast(fmaf(f[k], c, -l));
    st_cs_v4(o + i, Elem<T>::pack(f));
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
  return static_cast<const T*>(a.logits) + (r / a.inner) * a.outer_stride + (r % a.inner) * a.inner_stride;
}

// The parts of `work`.
LZ_DEV double2* work_norm(const LzLossArgs& a) { return reinterpret_cast<double2*>(a.work + LZ_LOSS_WORK_HEAD); }
LZ_DEV double* work_slope(const LzLossArgs& a) { return a.work + LZ_LOSS_WORK_HEAD + 2 * a.rows; }
LZ_DEV double* work_loss(const LzLossArgs& a) { return a.work + LZ_LOSS_WORK_HEAD + 3 * a.rows; }

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
  if (KIND == LZ_LOSS_LOGP) return 0.0;
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
    last = atomicAdd(reinterpret_cast<unsigned*>(a.work + 1), 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
  for (long long r = threadIdx.x; r < a.rows; r += kThreads) s += __ldcg(work_loss(a) + r);
  s = block_sum(s, dred);
  if (threadIdx.x == 0) *a.loss = (float)s;
}

// 1 / denominator (0 where that is not positive: nothing counts) and the ticket.
__global__ void __launch_bounds__(kThreads) head_kernel(const __grid_constant__ LzLossArgs a) {
  __shared__ double red[kWarps];
  double s = 0.0;
  if (a.denom_ptr) {
    s = (double)*a.denom_ptr;
  } else if (a.denom >= 0.0) {
    s = a.denom;
  } else {
    for (long long r = threadIdx.x; r < a.rows; r += kThreads)
      if (a.kind == LZ_LOSS_DISTILL || load_id(a.ids, a.ids64, r) >= 0) s += a.weights ? (double)a.weights[r] : 1.0;
    s = block_sum(s, red);
  }
  if (threadIdx.x == 0) {
    a.work[0] = s > 0.0 || s != s ? 1.0 / s : 0.0;
    *reinterpret_cast<unsigned*>(a.work + 1) = 0u;
    if (a.rows == 0) *a.loss = 0.f;
  }
}

// The gradient from the rows' saved sums and slopes. POLICY and DISTILL: where
// `grad` holds the gradient for upstream 1 and the upstream is 1, it stands.
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
    double slope = (double)up;
    if (KIND == LZ_LOSS_LOGP) slope = y < 0 ? 0.0 : slope * (double)a.row_upstream[r];
    else slope = work_slope(a)[r] == 0.0 ? 0.0 : slope * work_slope(a)[r];
    if (y >= a.vocab) slope = NAN;
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
      if (load_id(a.ids, a.ids64, r) >= 0) sum += (double)a.logp[r], count += 1.0;
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

template <typename T, int KIND>
int launch_forward(const LzLossArgs* a, cudaStream_t s) {
  if (KIND != LZ_LOSS_LOGP) {
    head_kernel<<<1, kThreads, 0, s>>>(*a);
    LZ_CUDA_TRY(cudaGetLastError());
  }
  if (!a->rows) return LZE_OK;
  int grid = 0;
  if (const int rc = grid_for(a->device, a->rows, &grid)) return rc;
  if (a->grad) forward_kernel<T, KIND, true><<<grid, kThreads, top_bytes(a), s>>>(*a);
  else forward_kernel<T, KIND, false><<<grid, kThreads, top_bytes(a), s>>>(*a);
  LZ_CUDA_TRY(cudaGetLastError());
  return LZE_OK;
}

template <typename T, int KIND>
int launch_backward(const LzLossArgs* a, cudaStream_t s) {
  if (!a->rows) return LZE_OK;
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
