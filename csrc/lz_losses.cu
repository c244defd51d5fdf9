// Vocabulary losses: entry points, and rows that a team of threads does alone
// (small vocabularies; rows that cannot be streamed, see lz_losses_stream.cu).
#include "lz_losses_dev.cuh"

namespace {

constexpr int kThreads = 512;  // of head_kernel and pair_kernel
constexpr int kWarps = kThreads / 32;
constexpr int kRowThreads = 128;
constexpr int kRowWarps = kRowThreads / 32;
// CTAs an SM: 64 registers a thread. With four blocks of 256 the sums of 8192 rows of
// 64 KB took 110 us, not 96.
constexpr int kRowCtas = 8;

template <typename V>
LZ_DEV V block_sum(V v, V* red, int warps) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  V s = red[0];
  for (int w = 1; w < warps; ++w) s += red[w];
  __syncthreads();
  return s;
}

// ---- rows that a team of TEAM threads does alone: a warp where a row is small
// (nothing waits for a barrier), a block otherwise. ----

// Thread `tid`'s share of a row's sum among TEAM.
template <typename T, int TEAM>
LZ_DEV LazySum row_sum(const T* x, long long n, float c, int tid) {
  constexpr int U = 4;
  LazySum s;
  s.init(c);
  const Split<T> sp(x, n);
  const uint4* v = reinterpret_cast<const uint4*>(x + sp.lead);
  int i = tid;
  for (; i + (U - 1) * TEAM < sp.vecs; i += U * TEAM) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = __ldg(v + i + u * TEAM);
    take_batch<T, U>(s, w, c, i == tid);
  }
  for (; i < sp.vecs; i += TEAM) {
    const uint4 w = __ldg(v + i);
    take_batch<T, 1>(s, &w, c, true);
  }
  const long long single = tid < 2 * Elem<T>::N ? single_of(sp.lead, sp.vecs, Elem<T>::N, tid, n) : -1;
  if (single >= 0) s.take_one(Elem<T>::get(x[single]), c);
  return s;
}

// Writes a row's dense gradient: zeros without a look at x where f is zero.
template <typename T, int TEAM>
LZ_DEV void row_dense(const T* x, T* out, long long n, const RowGrad& g, float c) {
  constexpr int N = Elem<T>::N, U = 4;
  const int tid = threadIdx.x % TEAM;
  // one element at a time where the two rows start at different offsets from a 16-byte border
  if (g.f != 0.f && (g.base != 0.f || ((uintptr_t)x ^ (uintptr_t)out) % 16)) {
    for (long long i = tid; i < n; i += TEAM) out[i] = Elem<T>::put(g.dense(Elem<T>::get(x[i]), c));
    return;
  }
  const Split<T> sp(out, n);
  const uint4* v = reinterpret_cast<const uint4*>(x + sp.lead);
  uint4* o = reinterpret_cast<uint4*>(out + sp.lead);
  const uint64_t c2 = pair(c, c), neg_ref = pair(-g.ref, -g.ref), f2 = pair(g.f, g.f);
  for (int i = tid; i < sp.vecs; i += U * TEAM) {
    uint4 w[U];
    if (g.f != 0.f)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * TEAM < sp.vecs) w[u] = __ldg(v + i + u * TEAM);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * TEAM < sp.vecs)
        st_cs_v4(o + i + u * TEAM, g.f == 0.f ? make_uint4(0, 0, 0, 0) : dense_vector<T>(w[u], c2, neg_ref, f2));
  }
  const long long single = tid < 2 * N ? single_of(sp.lead, sp.vecs, N, tid, n) : -1;
  if (single >= 0) out[single] = Elem<T>::put(g.f == 0.f ? 0.f : g.dense(Elem<T>::get(x[single]), c));
}

// The entries with t_j != 0, over what row_dense wrote (by all of the team, before). One warp.
template <typename T, int KIND>
LZ_DEV void row_sparse(const LzLossArgs& a, T* out, const RowParams& p, const TopView& t, const RowGrad& g, float c) {
  if (g.f == 0.f) return;
  const int lane = threadIdx.x % 32;
  if (KIND == LZ_LOSS_DISTILL) {
    for (int j = lane; j < a.top; j += 32)
      if (!(t.share[j] < 0.f)) out[t.id[j]] = Elem<T>::put(g.sparse(t.z[j], t.share[j], c));
  } else if (lane == 0 && p.token >= 0) {
    out[p.token] = Elem<T>::put(g.sparse(p.xy, 1.f, c));
  }
}

template <int TEAM>
LZ_DEV void team_sync() {
  if (TEAM == 32) __syncwarp();
  else __syncthreads();
}

// What a team keeps in shared memory; its list and hash table are in dynamic memory.
struct TeamShared {
  RowParams params;
  float2 part[kRowWarps];
};

template <int TEAM>
LZ_DEV TopView team_list(char* dynamic, int team, int top, int hash, int** table) {
  float* f = reinterpret_cast<float*>(dynamic) + (size_t)team * (4 * top + hash);
  *table = reinterpret_cast<int*>(f + 4 * top);
  return TopView{reinterpret_cast<int*>(f), f + top, f + 2 * top, f + 3 * top};
}

// The sum of a row, its scalars and outputs, then the gradient from a second look
// at the row, which the caches still hold.
template <typename T, int KIND, bool GRAD, int TEAM>
__global__ void __launch_bounds__(kRowThreads, kRowCtas) row_kernel(const __grid_constant__ LzLossArgs a, int hash) {
  constexpr int kTeams = kRowThreads / TEAM;
  __shared__ TeamShared teams[kTeams];
  __shared__ double red[kRowWarps];
  __shared__ bool last;
  extern __shared__ __align__(16) char dynamic[];
  const int team = threadIdx.x / TEAM, tid = threadIdx.x % TEAM, warp = tid / 32, lane = tid % 32;
  TeamShared& sh = teams[team];
  int* table = nullptr;
  const TopView list = team_list<TEAM>(dynamic, team, KIND == LZ_LOSS_DISTILL ? a.top : 0, hash, &table);
  const float c = (float)(kLog2e * (double)a.inv_temperature);
  for (long long r = (long long)blockIdx.x * kTeams + team; r < a.rows; r += (long long)gridDim.x * kTeams) {
    T* out = static_cast<T*>(a.grad) + (GRAD ? r * a.vocab : 0);
    const T* x = row_of<T>(a, r);
    if (!row_counts<KIND>(a, r)) {
      if (tid == 0) {
        no_outputs<KIND>(a, r);
        if (KIND != LZ_LOSS_LOGP) work_loss(a)[r] = 0.0;
      }
      if (GRAD) row_dense<T, TEAM>(x, out, a.vocab, RowGrad(0.f, 1.f, RowSum{0.f, 0.f, 1.f}), c);
      continue;
    }
    // A block's first warp has the teacher's list while the others have the row; a token's scalars are
    // fetched behind the row, when its logit is in the caches.
    constexpr int kSkip = KIND == LZ_LOSS_DISTILL && TEAM > 32 ? 32 : 0;
    LazySum s;
    s.init(c);
    if (KIND == LZ_LOSS_DISTILL && warp == 0) prepare_params<T, KIND>(a, x, r, sh.params, list, table, hash, c);
    if (tid >= kSkip) s = row_sum<T, TEAM - kSkip>(x, a.vocab, c, tid - kSkip);
    if (KIND != LZ_LOSS_DISTILL && warp == 0) prepare_params<T, KIND>(a, x, r, sh.params, list, table, hash, c);
    float m = s.ref, sum = s.total();
    lanes_join(m, sum, 32);
    if (TEAM > 32) {
      if (lane == 0) sh.part[warp] = make_float2(m, sum);
      __syncthreads();
      const float2 v = lane < kRowWarps ? sh.part[lane] : make_float2(-INFINITY, 0.f);
      m = v.x, sum = v.y;
      lanes_join(m, sum, kRowWarps);
    } else {
      __syncwarp();
    }
    RowSum n = {0.f, m, sum};
    if (!exact_ref(m)) n = slow_sum(x, a.vocab, c);
    const RowOut o = row_out<KIND>(a, sh.params, n.norm(), c);
    const RowGrad g(o.slope, a.inv_temperature, n);
    if (GRAD) {
      row_dense<T, TEAM>(x, out, a.vocab, g, c);
      team_sync<TEAM>();
      if (warp == 0) row_sparse<T, KIND>(a, out, sh.params, list, g, c);
    }
    if (warp == 0) {
      const double loss = row_outputs<KIND>(a, sh.params, o, n, list, r, c);
      if (KIND != LZ_LOSS_LOGP && lane == 0) work_loss(a)[r] = loss;
    }
    team_sync<TEAM>();  // the next row's scalars and list overwrite this one's
  }
  if (KIND == LZ_LOSS_LOGP) return;
  // The CTA that is done last adds the rows' losses up, in the rows' order.
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(work_ticket(a), 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
  for (long long r = threadIdx.x; r < a.rows; r += kRowThreads) s += __ldcg(work_loss(a) + r);
  s = block_sum(s, red, kRowWarps);
  if (threadIdx.x == 0) *a.loss = (float)s;
}

// The gradient from the rows' saved sums and slopes. POLICY and DISTILL: where
// `grad` holds the gradient for upstream 1 and the upstream is 1, it stands.
template <typename T, int KIND, int TEAM>
__global__ void __launch_bounds__(kRowThreads, kRowCtas) row_grad_kernel(const __grid_constant__ LzLossArgs a, int hash) {
  constexpr int kTeams = kRowThreads / TEAM;
  __shared__ TeamShared teams[kTeams];
  extern __shared__ __align__(16) char dynamic[];
  const float up = a.upstream ? *a.upstream : 1.f;
  if (!a.fresh && up == 1.f) return;
  const int team = threadIdx.x / TEAM, tid = threadIdx.x % TEAM, warp = tid / 32;
  TeamShared& sh = teams[team];
  int* table = nullptr;
  const TopView list = team_list<TEAM>(dynamic, team, KIND == LZ_LOSS_DISTILL ? a.top : 0, hash, &table);
  const float c = (float)(kLog2e * (double)a.inv_temperature);
  for (long long r = (long long)blockIdx.x * kTeams + team; r < a.rows; r += (long long)gridDim.x * kTeams) {
    const T* x = row_of<T>(a, r);
    T* out = static_cast<T*>(a.grad) + r * a.vocab;
    const float4 sum = work_sum(a)[r];
    const long long y = KIND == LZ_LOSS_DISTILL ? 0 : load_id(a.ids, a.ids64, r);
    const RowGrad g((float)row_slope_for<KIND>(a, r, y, up), a.inv_temperature, RowSum{sum.x, sum.y, sum.z});
    if (warp == 0 && g.f != 0.f) {
      if (KIND == LZ_LOSS_DISTILL) {
        prepare_params<T, KIND>(a, x, r, sh.params, list, table, hash, c);
      } else {
        if (tid == 0) sh.params.token = y < a.vocab ? (int)y : -1, sh.params.xy = y < a.vocab ? Elem<T>::get(x[y]) : 0.f;
        __syncwarp();
      }
    }
    row_dense<T, TEAM>(x, out, a.vocab, g, c);
    team_sync<TEAM>();
    if (warp == 0) row_sparse<T, KIND>(a, out, sh.params, list, g, c);
    team_sync<TEAM>();
  }
}

// 1 / denominator (0 where that is not positive: nothing counts), the ticket and,
// where `order` is set, the rows that count in front of those that do not, each
// in their order: taken in turns, every cluster of the streamed kernel gets as many.
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
      s = block_sum(s, red, kWarps);
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
    sum = block_sum(sum, red, kWarps);
    count = block_sum(count, red, kWarps);
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
  s = block_sum(s, red, kWarps);
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

// The rows' grid, a team a row at a time, and the team's lists. A warp where rows are
// very many and short, or tiny; in us, bf16, warp against block, policy with its
// gradient: 8192 rows of 8 KB 53 / 67, of 16 KB 90 / 91 (sums only 31 / 41), of 32 KB
// 161 / 140; 1024 rows of 8 KB 20 / 18, of 16 KB 25 / 21; 128 rows of 16 KB 26 / 17.
struct RowLaunch {
  int team, grid, hash;
  size_t smem;
};

int plan_rows(const LzLossArgs* a, RowLaunch* l) {
  int sms = 0;
  LZ_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, a->device));
  const bool distill = a->kind == LZ_LOSS_DISTILL;
  const long long row = a->vocab * (a->dtype == LZ_F32 ? 4 : 2);
  l->hash = 0;
  if (distill && a->top > kSmallList)
    for (l->hash = 32; l->hash < 2 * a->top;) l->hash *= 2;
  const bool warp = row <= 2048 || (row <= 16384 && a->rows >= 32ll * sms);
  l->team = warp && (!distill || a->top <= kSmallList) ? 32 : kRowThreads;
  const int teams = kRowThreads / l->team;
  const long long ctas = (a->rows + teams - 1) / teams, cap = (long long)sms * kRowCtas;
  l->grid = (int)(ctas < cap ? ctas : cap);
  l->smem = distill ? (size_t)teams * (4 * a->top + l->hash) * 4 : 0;
  return LZE_OK;
}

template <typename T, int KIND, bool GRAD>
void launch_rows(const LzLossArgs* a, const RowLaunch& l, cudaStream_t s) {
  if (l.team == 32) row_kernel<T, KIND, GRAD, 32><<<l.grid, kRowThreads, l.smem, s>>>(*a, l.hash);
  else row_kernel<T, KIND, GRAD, kRowThreads><<<l.grid, kRowThreads, l.smem, s>>>(*a, l.hash);
}

template <typename T, int KIND>
int forward_as(const LzLossArgs* a, cudaStream_t s) {
  LzStreamPlan stream;
  if (const int rc = lz_stream_plan(a, &stream)) return rc;
  if (KIND != LZ_LOSS_LOGP || stream.ordered) {
    head_kernel<KIND><<<1, kThreads, 0, s>>>(*a, stream.ordered);
    LZ_CUDA_TRY(cudaGetLastError());
  }
  if (!a->rows) return LZE_OK;
  if (stream.clusters) return lz_stream_forward(a, &stream, s);
  RowLaunch l;
  if (const int rc = plan_rows(a, &l)) return rc;
  if constexpr (KIND == LZ_LOSS_LOGP) launch_rows<T, KIND, false>(a, l, s);
  else if (a->grad) launch_rows<T, KIND, true>(a, l, s);
  else launch_rows<T, KIND, false>(a, l, s);
  LZ_CUDA_TRY(cudaGetLastError());
  return LZE_OK;
}

template <typename T, int KIND>
int backward_as(const LzLossArgs* a, cudaStream_t s) {
  if (!a->rows) return LZE_OK;
  if (lz_stream_grad_fits(a)) return lz_stream_grad(a, s);
  RowLaunch l;
  if (const int rc = plan_rows(a, &l)) return rc;
  if (l.team == 32) row_grad_kernel<T, KIND, 32><<<l.grid, kRowThreads, l.smem, s>>>(*a, l.hash);
  else row_grad_kernel<T, KIND, kRowThreads><<<l.grid, kRowThreads, l.smem, s>>>(*a, l.hash);
  LZ_CUDA_TRY(cudaGetLastError());
  return LZE_OK;
}

template <typename T>
int run_kind(const LzLossArgs* a, cudaStream_t s, bool forward) {
  switch (a->kind) {
    case LZ_LOSS_LOGP: return forward ? forward_as<T, LZ_LOSS_LOGP>(a, s) : backward_as<T, LZ_LOSS_LOGP>(a, s);
    case LZ_LOSS_POLICY: return forward ? forward_as<T, LZ_LOSS_POLICY>(a, s) : backward_as<T, LZ_LOSS_POLICY>(a, s);
    default: return forward ? forward_as<T, LZ_LOSS_DISTILL>(a, s) : backward_as<T, LZ_LOSS_DISTILL>(a, s);
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

extern "C" int lz_loss_backward(const LzLossArgs* a, cudaStream_t stream) {
  // What only the forward pass reads may be gone by now.
  LzLossArgs b = *a;
  b.old_logp = b.advantages = b.ref_logp = b.weights = b.denom_ptr = nullptr;
  b.loss = b.logp = b.kl = nullptr, b.clipped = nullptr;
  return run(&b, stream, false);
}

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
