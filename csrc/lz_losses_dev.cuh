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
#pragma once
#include <cfloat>
#include <type_traits>

#include "lz_common.cuh"
#include "lz_internal.h"
#include "lz_losses.h"

namespace {

constexpr double kLn2 = 0.693147180559945309417;
constexpr double kLog2e = 1.44269504088896340736;
constexpr int kMaxDevices = 64;
constexpr int kMaxCluster = 8;
constexpr int kSmallList = 128;  // teacher's lists up to here look for equal ids entry by entry, longer ones by a hash table

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

template <typename T>
LZ_DEV void unpack_pairs(uint4 v, uint64_t* p) {
  float f[Elem<T>::N];
  Elem<T>::unpack(v, f);
#pragma unroll
  for (int i = 0; i < Elem<T>::N / 2; ++i) p[i] = pair(f[2 * i], f[2 * i + 1]);
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

// `v` of CTA `rank` of this cluster.
template <typename V>
LZ_DEV V peer_value(const V* v, uint32_t rank) {
  static_assert(sizeof(V) == 16, "two words");
  uint64_t w[2];
  asm volatile(
      "{\n\t.reg .b32 p;\n\t"
      "mapa.shared::cluster.u32 p, %2, %3;\n\t"
      "ld.shared::cluster.v2.b64 {%0, %1}, [p];\n\t}"
      : "=l"(w[0]), "=l"(w[1])
      : "r"(smem_addr(v)), "r"(rank)
      : "memory");
  V out;
  memcpy(&out, w, 16);
  return out;
}

// Index of the t-th single element of a row of `n`, or -1.
LZ_DEV long long single_of(int lead, int vecs, int per_vec, int t, long long n) {
  const long long tail = lead + (long long)vecs * per_vec;
  if (t < lead) return t;
  return t - lead < n - tail ? tail + t - lead : -1;
}

// p_j = 2^((x_j - base) c - lse2). base is 0 but in rows whose maximum times c is
// no integer's neighbour in fp32 any more (all of a row masked, with -1e10 or the
// type's lowest value): there it is that maximum, and the row takes the slow loops.
struct Norm {
  float base;
  double lse2;
};

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

// What the gradient of a row takes: dlogits_j = scale t_j + f 2^((x_j - base) c - ref),
// with f = -scale inv and p_j = inv 2^(...). scale is the slope over T.
struct RowGrad {
  float f, base, ref, inv, scale;
  LZ_DEV RowGrad() {}
  LZ_DEV RowGrad(float slope, float inv_t, const RowSum& n) : base(n.base), ref(n.ref), inv(1.f / n.sum), scale(slope * inv_t) {
    f = slope == 0.f ? 0.f : -scale * inv;
  }
  LZ_DEV float dense(float x, float c) const { return f * exp2_fast(fmaf(x - base, c, -ref)); }
  LZ_DEV float sparse(float x, float t, float c) const { return scale * (t - inv * exp2_fast(fmaf(x - base, c, -ref))); }
};

// The dense gradient of a 16-byte vector (rows whose base is 0).
template <typename T>
LZ_DEV uint4 dense_vector(uint4 w, uint64_t c2, uint64_t neg_ref, uint64_t f2) {
  uint64_t p[Elem<T>::N / 2];
  float e[Elem<T>::N];
  unpack_pairs<T>(w, p);
#pragma unroll
  for (int q = 0; q < Elem<T>::N / 2; ++q) {
    float lo, hi;
    unpair(fma2(p[q], c2, neg_ref), lo, hi);
    unpair(mul2(f2, pair(exp2_fast(lo), exp2_fast(hi))), e[2 * q], e[2 * q + 1]);
  }
  return Elem<T>::pack(e);
}

constexpr int kBatch = 3;  // vectors a thread has in work at a time
constexpr float kExactRef = 8388608.f;  // 2^23: references up to here are exact integers, and so is x c - ref near them

// Sum over a thread's elements of 2^(x c - ref). ref is an integer, so that sums are
// brought to another reference without a rounding (with the maximum itself as the
// reference log-probabilities were low by 1.6e-7 on average). It is not the running
// maximum: it is taken from the first batch and moves only when a batch's maximum is
// more than 2^16 above it, which fp32 has room for (2^16 times the vocabulary), so
// the exponentials of a batch wait for no maximum and the branch is seldom taken.
// A thread that sees nothing above -kExactRef / c leaves the reference -inf and a sum
// of 0; a NaN or +inf makes the sum NaN.
struct LazySum {
  float ref, limit;  // in units of x c, of x; ref is -inf (and taken as 0) before the first batch
  uint64_t neg_ref, sum[2];
  LZ_DEV void init(float c) {
    ref = -INFINITY, neg_ref = 0, sum[0] = sum[1] = 0;
    limit = -kExactRef / c;  // entries below this count nothing beside 2^0
  }
  LZ_DEV float total() const {
    float s0, s1, s2, s3;
    unpair(sum[0], s0, s1), unpair(sum[1], s2, s3);
    return (s0 + s1) + (s2 + s3);
  }
  LZ_DEV void take_one(float x, float c) {
    if (x > limit) raise(x, c);
    float off, unused;
    unpair(neg_ref, off, unused);
    sum[0] = add2(sum[0], pair(exp2_fast(fmaf(x, c, off)), 0.f));
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

// The largest element of U vectors; NaN only if all are.
template <typename T, int U>
LZ_DEV float batch_max(const uint4* w) {
  if constexpr (sizeof(T) == 4) {
    const float* f = reinterpret_cast<const float*>(w);
    float m = f[0];
#pragma unroll
    for (int i = 1; i < 4 * U; ++i) m = fmaxf(m, f[i]);
    return m;
  } else {
    using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
    const T2* h = reinterpret_cast<const T2*>(w);
    T2 m = h[0];
#pragma unroll
    for (int i = 1; i < 4 * U; ++i) m = __hmax2(m, h[i]);
    return fmaxf(Elem<T>::get(m.x), Elem<T>::get(m.y));
  }
}

// `first` (of a row): nothing to go by, so the maximum comes first.
template <typename T, int U>
LZ_DEV void take_batch(LazySum& s, const uint4* w, float c, bool first) {
  const uint64_t c2 = pair(c, c);
  const float m = batch_max<T, U>(w);
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

// (reference, sum) over a warp's lanes; the same in every lane. Lanes beyond the
// first `n` (a power of two) hold (-inf, 0).
LZ_DEV void lanes_join(float& m, float& s, int n) {
  float top;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(m));
  s *= m == -INFINITY ? 1.f : exp2_fast(m - top);  // a sum without a reference is 0 or NaN
#pragma unroll
  for (int o = 16; o; o >>= 1)
    if (o < n) s += __shfl_xor_sync(~0u, s, o);
  if (n < 32) s = __shfl_sync(~0u, s, 0);
  m = top;
}

// Whether a joined reference is that of an ordinary row.
LZ_DEV bool exact_ref(float ref) { return fabsf(ref) <= kExactRef; }

// Maximum and sum of any other row, by one warp.
template <typename T>
LZ_DEV RowSum slow_sum(const T* x, long long n, float c) {
  const int lane = threadIdx.x % 32;
  float m = -INFINITY, s = 0.f, part[8] = {};
#pragma unroll 8
  for (long long i = lane; i < n; i += 32) m = fmaxf(m, Elem<T>::get(x[i]));
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  for (long long first = lane; first < n; first += 256)
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (first + 32 * u < n) part[u] += exp2_fast((Elem<T>::get(x[first + 32 * u]) - m) * c);
#pragma unroll
  for (int u = 0; u < 8; ++u) s += part[u];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  return {m, 0.f, s};
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
LZ_DEV float4* work_sum(const LzLossArgs& a) { return reinterpret_cast<float4*>(a.work + LZ_LOSS_WORK_HEAD); }
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

struct RowParams {
  float xy, adv;
  double old_logp2, ref_logp2;  // base 2
  double weight;  // over the denominator
  int token;      // -1: beyond the vocabulary
  float slope;    // DISTILL
  double q_logq, q_z, q_sum;  // DISTILL: sums over the list (z in base 2)
};

// The teacher's list of a row: entries and, with equal ids joined, what the gradient takes from them.
struct TopView {
  int* id;
  float *z, *q, *share;  // share < 0: another entry of the same id has it
};

LZ_DEV float top_value(const LzLossArgs& a, long long r, int k) { return load_any(a.teacher, a.teacher_dtype, r * a.top + k); }

// What a row's scalars give; logp2: the token's log-probability in base 2.
struct RowOut {
  double logp2;
  Norm norm;
  double ratio;
  float slope;
  bool clipped;
};

// A row's ratio and its slope over its weight in 64 bits. Where a ratio or a KL slope is beyond 2^64, the
// advantage, the weight or the denominator may still bring it back into the range of fp32, and its
// exponent has bits that fp32 does not hold. Out of line: in line, rows of 64 KB took 2 to 5 % longer.
struct FarRow {
  double ratio, slope;
};
__device__ __noinline__ FarRow far_row(double log_ratio2, double d, float adv, float kl_coef, bool clipped) {
  const double ratio = exp2(log_ratio2);
  double slope = clipped ? 0.0 : -(double)adv * ratio;
  if (kl_coef != 0.f) slope -= (double)kl_coef * expm1(d);
  return {ratio, slope};
}

template <int KIND>
LZ_DEV RowOut row_out(const LzLossArgs& a, const RowParams& p, const Norm& n, float c) {
  RowOut o;
  o.norm = n;
  o.logp2 = p.token < 0 ? (double)NAN : ((double)p.xy - (double)n.base) * (double)c - n.lse2;
  o.ratio = 0.0, o.clipped = false, o.slope = KIND == LZ_LOSS_DISTILL ? p.slope : 0.f;
  if (KIND == LZ_LOSS_POLICY) {
    const double log_ratio2 = o.logp2 - p.old_logp2, d = (p.ref_logp2 - o.logp2) * kLn2;
    const float ratio = exp2f((float)log_ratio2);
    o.clipped = (p.adv > 0.f && ratio > 1.f + a.clip_high) || (p.adv < 0.f && ratio < 1.f - a.clip_low);
    float slope = o.clipped ? 0.f : -p.adv * ratio;
    if (a.kl_coef != 0.f) slope -= a.kl_coef * expm1f((float)d);
    FarRow f = {(double)ratio, (double)slope};
    if (!(fabsf((float)log_ratio2) < 64.f && (a.kl_coef == 0.f || fabsf((float)d) < 64.f) && fabsf(slope) < INFINITY))
      f = far_row(log_ratio2, d, p.adv, a.kl_coef, o.clipped);
    o.ratio = f.ratio, o.slope = (float)(p.weight * f.slope);
  }
  return o;
}

// Writes (where `store`) a row's outputs and what the backward pass takes, from which it
// gets the same bits for upstream 1; returns its loss. `kl`: DISTILL's. One thread.
template <int KIND>
LZ_DEV double row_write(const LzLossArgs& a, const RowParams& p, const RowOut& o, const RowSum& n, double kl, long long r,
                        bool store) {
  double each = kl;
  if (KIND == LZ_LOSS_POLICY) {
    const double lo = 1.0 - (double)a.clip_low, hi = 1.0 + (double)a.clip_high;
    each = -(double)p.adv * (o.clipped ? (p.adv > 0.f ? hi : lo) : o.ratio);
    if (a.ref_logp) {
      const double d = (p.ref_logp2 - o.logp2) * kLn2;
      kl = expm1(d) - fmin(d, DBL_MAX);  // +inf where the token has probability zero
      if (a.kl_coef != 0.f) each += (double)a.kl_coef * kl;  // 0: watched alone, it may be infinite
    }
  }
  if (store) {
    if (KIND != LZ_LOSS_DISTILL) a.logp[r] = (float)(o.logp2 * kLn2);
    if (KIND == LZ_LOSS_DISTILL || (KIND == LZ_LOSS_POLICY && a.ref_logp)) a.kl[r] = (float)kl;
    if (KIND == LZ_LOSS_POLICY) a.clipped[r] = o.clipped;
    work_sum(a)[r] = make_float4(n.base, n.ref, n.sum, 0.f);
    work_slope(a)[r] = KIND == LZ_LOSS_LOGP ? o.logp2 * kLn2 : (double)o.slope;
  }
  return KIND == LZ_LOSS_LOGP ? 0.0 : p.weight * each;
}

// The same by one warp. `t`: the teacher's list.
template <int KIND>
LZ_DEV double row_outputs(const LzLossArgs& a, const RowParams& p, const RowOut& o, const RowSum& n, const TopView& t,
                          long long r, float c) {
  const int lane = threadIdx.x % 32;
  double kl = 0.0;
  if (KIND == LZ_LOSS_DISTILL) {
    kl = p.q_logq - kLn2 * (p.q_z - p.q_sum * o.norm.lse2);
    if (o.norm.base != 0.f) {  // differences of what is beyond 32 bits: entry by entry
      kl = 0.0;
      for (int j = lane; j < a.top; j += 32)
        if (t.q[j] != 0.f)
          kl += (double)t.q[j] * (log((double)t.q[j]) -
                                  (((double)t.z[j] - (double)o.norm.base) * (double)c - o.norm.lse2) * kLn2);
#pragma unroll
      for (int s = 16; s; s >>= 1) kl += __shfl_xor_sync(~0u, kl, s);
    }
    if (p.q_sum == 0.0) kl = 0.0;  // an empty list shields its row, whatever the logits are
    if (isnan(p.slope)) kl = NAN;
  }
  return row_write<KIND>(a, p, o, n, kl, r, lane == 0);
}

// A row's slope for the given upstream; zero where the row does not count or has no upstream of its own,
// whatever its token. One beyond the vocabulary is NaN otherwise (POLICY's saved slope is that already).
template <int KIND>
LZ_DEV double row_slope_for(const LzLossArgs& a, long long r, long long y, float up) {
  const double slope = KIND != LZ_LOSS_LOGP ? work_slope(a)[r] : y < 0 ? 0.0 : (double)a.row_upstream[r];
  if (slope == 0.0) return 0.0;
  return KIND == LZ_LOSS_LOGP && y >= a.vocab ? (double)NAN : (double)up * slope;
}

// Outputs of a row that does not count.
template <int KIND>
LZ_DEV void no_outputs(const LzLossArgs& a, long long r) {
  if (KIND != LZ_LOSS_DISTILL) a.logp[r] = 0.f;
  if (KIND == LZ_LOSS_DISTILL || (KIND == LZ_LOSS_POLICY && a.ref_logp)) a.kl[r] = 0.f;
  if (KIND == LZ_LOSS_POLICY) a.clipped[r] = 0;
  work_sum(a)[r] = make_float4(0.f, 0.f, 1.f, 0.f);
  work_slope(a)[r] = 0.0;
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

// A row's scalars (LOGP, POLICY).
template <typename T, int KIND>
LZ_DEV void token_params(const LzLossArgs& a, const T* x, long long r, RowParams& out) {
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

// A row's scalars and, for DISTILL, the teacher's list; `hash` has `hashed` entries, a
// power of two, where the list is long. One warp.
template <typename T, int KIND>
LZ_DEV void prepare_params(const LzLossArgs& a, const T* x, long long r, RowParams& out, TopView t, int* hash, int hashed,
                           float c) {
  const int lane = threadIdx.x % 32;
  if (KIND != LZ_LOSS_DISTILL) {
    if (lane == 0) token_params<T, KIND>(a, x, r, out);
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
  // Sums over e = exp((v - m) / T); q = e / s. The difference comes first: a type's lowest value over T may
  // be -inf. An entry that is NaN or +inf makes s NaN, also where the maximum passed over it and is -inf.
  float s = 0.f;
  double e_v = 0.0, e_z = 0.0;
  for (int k = lane; k < a.top; k += 32) {
    const float at = t.q[k], v = (at - m) * a.inv_temperature, e = at == -INFINITY ? 0.f : expf(v);
    t.q[k] = e;
    if (e != 0.f) {
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
    // Four ids a load. The last may have words of `z` in it; where one is taken for an id, the list
    // is looked at again all the same.
    const int4* four = reinterpret_cast<const int4*>(t.id);
    for (int k = lane; k < a.top; k += 32) {
      const int id = t.id[k];
      int same = 0;
#pragma unroll 4
      for (int o = 0; o < (a.top + 3) / 4; ++o) {
        const int4 v = four[o];
        same += (v.x == id) + (v.y == id) + (v.z == id) + (v.w == id);
      }
      twice |= id >= 0 && same > 1;
    }
  } else {
    for (int k = lane; k < hashed; k += 32) hash[k] = -1;
    __syncwarp();
    for (int k = lane; k < a.top; k += 32) {
      const int id = t.id[k];
      if (id < 0) continue;
      for (unsigned h = (unsigned)id * 2654435761u >> 7;; ++h) {  // ends: the table is twice the list
        const int was = atomicCAS(hash + (h & (hashed - 1)), -1, id);
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
    out.slope = bad || s != s ? NAN : m == -INFINITY ? 0.f : (float)-out.weight;
    out.q_logq = q_logq, out.q_z = q_z, out.q_sum = q_sum;
  }
  __syncwarp();
}

}  // namespace

// lz_losses_stream.cu: large vocabularies. The plan of a launch; clusters is 0
// where rows cannot be streamed or a row a team of threads does better.
struct LzStreamPlan {
  int clusters, ranks;
  int slots;    // of the ring, a chunk each
  int early;    // chunks of the next row taken before this one's gradient
  int ordered;  // rows by work_order; otherwise one row a cluster
  int hash;     // entries of a hash table of DISTILL, a power of two; 0 where the list is short
  int views;    // DISTILL: rows whose lists are kept, 2 or 4
  size_t smem;
  unsigned long long wait_ns;
};
int lz_stream_plan(const LzLossArgs* a, LzStreamPlan* plan);
int lz_stream_forward(const LzLossArgs* a, const LzStreamPlan* plan, cudaStream_t stream);
bool lz_stream_grad_fits(const LzLossArgs* a);
int lz_stream_grad(const LzLossArgs* a, cudaStream_t stream);
