// Vocabulary losses: entry points, and rows that a team of threads does alone
// (small vocabularies; rows that cannot be streamed, see lz_losses_stream.cu).
#include <algorithm>

#include "lz_losses_dev.cuh"

namespace {

constexpr int kThreads = 512;  // of head_kernel and pair_kernel
constexpr int kWarps = kThreads / 32;
constexpr int kRowThreads = 128;
constexpr int kRowWarps = kRowThreads / 32;
// CTAs an SM: 64 registers a thread. With four blocks of 256 the sums of 8192 rows of
// 64 KB took 110 us, not 96. Some kernels spill for it (policy's gradient by parts of a warp
// 208 bytes). Six CTAs need no spill: policy steps of 262144 x 256 took 100 us, not 109, of 8192 x
// 16384 128, not 133, but sums alone 62, not 59, and 72, not 68, and DISTILL's of 8192 x 4000 52, not 50.
constexpr int kRowCtas = 8;
constexpr long long kWarpBytes = 8192;  // of the rows that a warp has at a time
// More are the head's cluster's. A policy step of 24000 columns, one CTA against the cluster: 1024 rows
// 34.7 / 36.7 us, 2048 61.6 / 61.3, 3000 81.6 / 80.2, 8192 191.6 / 187.0.
constexpr long long kHeadRows = 2048;

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
#pragma unroll
  for (int t = tid; t < 2 * Elem<T>::N; t += TEAM) {
    const long long single = single_of(sp.lead, sp.vecs, Elem<T>::N, t, n);
    if (single >= 0) s.take_one(Elem<T>::get(x[single]), c);
  }
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
#pragma unroll
  for (int t = tid; t < 2 * N; t += TEAM) {
    const long long single = single_of(sp.lead, sp.vecs, N, t, n);
    if (single >= 0) out[single] = Elem<T>::put(g.f == 0.f ? 0.f : g.dense(Elem<T>::get(x[single]), c));
  }
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
  double loss;
};

template <int TEAM>
LZ_DEV TopView team_list(char* dynamic, int team, int top, int hash, int** table) {
  float* f = reinterpret_cast<float*>(dynamic) + (size_t)team * (4 * top + hash);
  *table = reinterpret_cast<int*>(f + 4 * top);
  return TopView{reinterpret_cast<int*>(f), f + top, f + 2 * top, f + 3 * top};
}

// The CTA that is done last adds the CTAs' losses (`loss`, in thread 0) up, in their order.
LZ_DEV void finish_loss(const LzLossArgs& a, double loss) {
  __shared__ double red[kRowWarps];
  __shared__ bool last;
  if (threadIdx.x == 0) {
    work_loss(a)[blockIdx.x] = loss;
    __threadfence();
    last = atomicAdd(work_ticket(a), 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
  for (unsigned k = threadIdx.x; k < gridDim.x; k += kRowThreads) s += __ldcg(work_loss(a) + k);
  s = block_sum(s, red, kRowWarps);
  if (threadIdx.x == 0) *a.loss = (float)s;
}

// The sum of a row, its scalars and outputs, then the gradient from a second look
// at the row, which the caches still hold.
template <typename T, int KIND, bool GRAD, int TEAM>
__global__ void __launch_bounds__(kRowThreads, kRowCtas) row_kernel(const __grid_constant__ LzLossArgs a, int hash) {
  constexpr int kTeams = kRowThreads / TEAM;
  __shared__ TeamShared teams[kTeams];
  extern __shared__ __align__(16) char dynamic[];
  const int team = threadIdx.x / TEAM, tid = threadIdx.x % TEAM, warp = tid / 32, lane = tid % 32;
  TeamShared& sh = teams[team];
  if (tid == 0) sh.loss = 0.0;
  int* table = nullptr;
  const TopView list = team_list<TEAM>(dynamic, team, KIND == LZ_LOSS_DISTILL ? a.top : 0, hash, &table);
  const float c = (float)(kLog2e * (double)a.inv_temperature);
  for (long long r = (long long)blockIdx.x * kTeams + team; r < a.rows; r += (long long)gridDim.x * kTeams) {
    T* out = static_cast<T*>(a.grad) + (GRAD ? r * a.vocab : 0);
    const T* x = row_of<T>(a, r);
    if (!row_counts<KIND>(a, r)) {
      if (tid == 0) no_outputs<KIND>(a, r);
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
      if (KIND != LZ_LOSS_LOGP && lane == 0) sh.loss += loss;
    }
    team_sync<TEAM>();  // the next row's scalars and list overwrite this one's
  }
  if (KIND == LZ_LOSS_LOGP) return;
  __syncthreads();
  double s = 0.0;
  for (int k = 0; k < kTeams; ++k) s += teams[k].loss;
  finish_loss(a, s);
}

// LOGP and POLICY, short rows where they are very many: `batch` of them a warp at a
// time, L lanes a row, and the scalars and outputs of each by a lane of its own. A warp
// a row spends more instructions on what is per row than on its elements.

// (reference, sum) over L lanes, as lanes_join.
template <int L>
LZ_DEV void group_join(float& m, float& s) {
  float top = m;
#pragma unroll
  for (int o = L / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  s *= m == -INFINITY ? 1.f : exp2_fast(m - top);  // a sum without a reference is 0 or NaN
#pragma unroll
  for (int o = L / 2; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  m = top;
}

// The gradients of the rows from `first` on; `g`, `token` and `xy` are those of the lane's row.
template <typename T, int L>
LZ_DEV void warp_gradients(const LzLossArgs& a, long long first, int rows, const RowGrad& g, int token, float xy, float c) {
  const int lane = threadIdx.x % 32;
  T* out = static_cast<T*>(a.grad) + first * a.vocab;
  for (int j = 0; j < rows; j += 32 / L) {
    const int i = j + lane / L;
    RowGrad d;
    d.f = __shfl_sync(~0u, g.f, i), d.base = __shfl_sync(~0u, g.base, i), d.ref = __shfl_sync(~0u, g.ref, i);
    if (i < rows) row_dense<T, L>(row_of<T>(a, first + i), out + i * a.vocab, a.vocab, d, c);
  }
  __syncwarp();
  if (lane < rows && g.f != 0.f && token >= 0) out[lane * a.vocab + token] = Elem<T>::put(g.sparse(xy, 1.f, c));
}

template <typename T, int KIND, bool GRAD, int L>
__global__ void __launch_bounds__(kRowThreads, kRowCtas) warp_kernel(const __grid_constant__ LzLossArgs a, int batch) {
  __shared__ double red[kRowWarps];
  const int lane = threadIdx.x % 32;
  const float c = (float)(kLog2e * (double)a.inv_temperature);
  const long long at = ((long long)blockIdx.x * kRowWarps + threadIdx.x / 32) * batch, step = (long long)gridDim.x * kRowWarps * batch;
  double loss = 0.0;
  for (long long first = at; first < a.rows; first += step) {
    const long long r = first + lane;
    const int rows = (int)min((long long)batch, a.rows - first);
    const bool counts = lane < rows && row_counts<KIND>(a, r);
    const unsigned counted = __ballot_sync(~0u, counts);
    RowSum n = {0.f, 0.f, 1.f};
    for (int j = 0; j < rows; j += 32 / L) {
      const int i = j + lane / L;
      LazySum s;
      s.init(c);
      if (counted >> i & 1) s = row_sum<T, L>(row_of<T>(a, first + i), a.vocab, c, lane % L);
      float m = s.ref, sum = s.total();
      group_join<L>(m, sum);
      m = __shfl_sync(~0u, m, lane % (32 / L) * L), sum = __shfl_sync(~0u, sum, lane % (32 / L) * L);
      if (lane / (32 / L) == j / (32 / L)) n.ref = m, n.sum = sum;
    }
    for (unsigned odd = __ballot_sync(~0u, counts && !exact_ref(n.ref)); odd; odd &= odd - 1) {
      const int i = __ffs(odd) - 1;
      const RowSum v = slow_sum(row_of<T>(a, first + i), a.vocab, c);
      if (lane == i) n = v;
    }
    RowParams p;
    p.token = -1, p.xy = 0.f;
    RowGrad g(0.f, 1.f, RowSum{0.f, 0.f, 1.f});
    if (counts) {
      token_params<T, KIND>(a, row_of<T>(a, r), r, p);
      const RowOut o = row_out<KIND>(a, p, n.norm(), c);
      g = RowGrad(o.slope, a.inv_temperature, n);
      loss += row_write<KIND>(a, p, o, n, 0.0, r, true);
    } else if (lane < rows) {
      no_outputs<KIND>(a, r);
    }
    if (GRAD) warp_gradients<T, L>(a, first, rows, g, p.token, p.xy, c);
  }
  if (KIND != LZ_LOSS_LOGP) finish_loss(a, block_sum(loss, red, kRowWarps));
}

template <typename T, int KIND, int L>
__global__ void __launch_bounds__(kRowThreads, kRowCtas) warp_grad_kernel(const __grid_constant__ LzLossArgs a, int batch) {
  const float up = a.upstream ? *a.upstream : 1.f;
  if (!a.fresh && up == 1.f) return;
  const int lane = threadIdx.x % 32;
  const float c = (float)(kLog2e * (double)a.inv_temperature);
  const long long at = ((long long)blockIdx.x * kRowWarps + threadIdx.x / 32) * batch, step = (long long)gridDim.x * kRowWarps * batch;
  for (long long first = at; first < a.rows; first += step) {
    const long long r = first + lane;
    const int rows = (int)min((long long)batch, a.rows - first);
    RowGrad g(0.f, 1.f, RowSum{0.f, 0.f, 1.f});
    int token = -1;
    float xy = 0.f;
    if (lane < rows) {
      const float4 sum = work_sum(a)[r];
      const long long y = load_id(a.ids, a.ids64, r);
      g = RowGrad((float)row_slope_for<KIND>(a, r, y, up), a.inv_temperature, RowSum{sum.x, sum.y, sum.z});
      if (g.f != 0.f && y < a.vocab) token = (int)y, xy = Elem<T>::get(row_of<T>(a, r)[y]);
    }
    warp_gradients<T, L>(a, first, rows, g, token, xy, c);
  }
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
// A cluster of CTAs where rows are many, each with a part of them: 8192 rows take 7 us, by
// one CTA 13, 262144 rows 19, by one CTA 80.
struct HeadPart {
  double weights;
  long long rows;  // that count
};

template <int KIND>
__global__ void __launch_bounds__(kThreads) head_kernel(const __grid_constant__ LzLossArgs a, bool order) {
  __shared__ double red[kWarps];
  __shared__ long long red_rows[kWarps];
  __shared__ int counts[2][kWarps];
  __shared__ alignas(16) HeadPart part;
  constexpr int U = 8;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const long long per = (a.rows + ranks - 1) / ranks, begin = min(rank * per, a.rows), end = min(begin + per, a.rows);
  const bool given = KIND == LZ_LOSS_LOGP || a.denom_ptr || a.denom >= 0.0;
  HeadPart all = {0.0, 0};
  long long before = 0;  // rows of the ranks before this that count
  if (!given || (order && ranks > 1)) {
    for (long long first = begin + threadIdx.x; first < end; first += U * kThreads) {
      long long id[U];
      float w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {  // no branch: the loads run together
        const long long r = min(first + u * kThreads, end - 1);
        id[u] = KIND == LZ_LOSS_DISTILL ? 0 : load_id(a.ids, a.ids64, r);
        w[u] = KIND != LZ_LOSS_LOGP && a.weights ? a.weights[r] : 1.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (id[u] >= 0 && first + u * kThreads < end) all.weights += (double)w[u], all.rows += w[u] != 0.f;
    }
    all.weights = block_sum(all.weights, red, kWarps);
    if (ranks > 1) {
      all.rows = block_sum(all.rows, red_rows, kWarps);
      if (threadIdx.x == 0) part = all;
      cluster_sync();
      all = {0.0, 0};
      for (uint32_t k = 0; k < ranks; ++k) {
        const HeadPart v = peer_value(&part, k);
        all.weights += v.weights, all.rows += v.rows;
        if (k < rank) before += v.rows;
      }
      cluster_sync();  // no CTA leaves while a peer reads its part
    }
  }
  if (rank == 0 && threadIdx.x == 0) {
    const double s = given ? (a.denom_ptr ? (double)*a.denom_ptr : a.denom) : all.weights;
    a.work[0] = s > 0.0 || s != s ? 1.0 / s : 0.0;
    *work_ticket(a) = 0u;
    if (KIND != LZ_LOSS_LOGP && a.rows == 0) *a.loss = 0.f;
  }
  if (!order) return;
  const int n = (int)a.rows;
  int front = (int)before, back = (int)(begin - before);  // rows placed at either end
  for (int first = (int)begin, k = 0; first < end; first += kThreads, k ^= 1) {
    const int r = first + threadIdx.x;
    const bool counts_ = r < end && row_counts<KIND>(a, r);
    const unsigned m = __ballot_sync(~0u, counts_);
    if (lane == 0) counts[k][warp] = __popc(m);
    __syncthreads();
    int ahead = 0, here = 0;
    for (int w = 0; w < kWarps; ++w) {
      ahead += w < warp ? counts[k][w] : 0;
      here += counts[k][w];
    }
    ahead += __popc(m & ((1u << lane) - 1));
    if (r < end) work_order(a)[counts_ ? front + ahead : n - 1 - (back + (int)threadIdx.x - ahead)] = r;
    front += here;
    back += min(kThreads, (int)end - first) - here;
  }
  if (rank == ranks - 1 && threadIdx.x == 0) *work_active(a) = front;
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
  // a term of weight zero is none, though an answer that cannot be makes it infinite
  if (threadIdx.x == 0) a.work[1 + pair] = (a.smoothing < 1.0 ? (1.0 - a.smoothing) * up : 0.0) + (a.smoothing > 0.0 ? a.smoothing * down : 0.0);
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

// The rows' grid, a team a row at a time, and the team's lists. A warp or a part of
// one where rows are very many and short, a warp where they are tiny. In us, bf16, a
// part against a warp, policy with its gradient: 262144 rows of 512 bytes 114 / 417 (sums
// only 37 / 116), 32768 rows of 2 KB 57 / 88, of 4 KB 93 / 111, 8192 rows of 4 KB 33 / 36. A
// warp against a block: 8192 rows of 8 KB 53 / 67, of 16 KB 90 / 91 (sums only 31 / 41), of
// 32 KB 161 / 140; 1024 rows of 8 KB 20 / 18, of 16 KB 25 / 21; 128 rows of 16 KB 26 / 17.
struct RowLaunch {
  int team, grid, hash;
  int batch;  // rows that a warp has at a time
  size_t smem;
};

int plan_rows(const LzLossArgs* a, RowLaunch* l) {
  int sms = 0;
  LZ_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, a->device));
  const bool distill = a->kind == LZ_LOSS_DISTILL;
  const long long row = a->vocab * (a->dtype == LZ_F32 ? 4 : 2);
  const long long cap = (long long)sms * kRowCtas, each = (a->rows + cap * kRowWarps - 1) / (cap * kRowWarps);  // rows a warp
  l->hash = 0;
  if (distill && a->top > kSmallList)
    for (l->hash = 32; l->hash < 2 * a->top;) l->hash *= 2;
  const bool warp = row <= 2048 || (row <= 16384 && a->rows >= 32ll * sms);
  l->team = warp && (!distill || a->top <= kSmallList) ? 32 : kRowThreads;
  if (!distill && row <= 2048 && each >= 4) l->team = 8;
  else if (!distill && row <= 4096 && each >= 2) l->team = 16;
  const int teams = kRowThreads / l->team, at_once = l->team < 32 ? 32 / l->team : 1;
  // All warps' batches together stay in L2 until their gradient.
  l->batch = l->team < 32 ? (int)std::max((long long)at_once, std::min({32ll, each, kWarpBytes / row})) : 1;
  l->smem = distill ? (size_t)teams * (4 * a->top + l->hash) * 4 : 0;
  const int of_cta = l->team < 32 ? kRowWarps * l->batch : teams;
  const long long ctas = (a->rows + of_cta - 1) / of_cta;
  l->grid = (int)(ctas < cap ? ctas : cap);
  return LZE_OK;
}

template <typename T, int KIND, bool GRAD>
void launch_rows(const LzLossArgs* a, const RowLaunch& l, cudaStream_t s) {
  if constexpr (KIND != LZ_LOSS_DISTILL)
    switch (l.team) {
      case 8: return warp_kernel<T, KIND, GRAD, 8><<<l.grid, kRowThreads, 0, s>>>(*a, l.batch);
      case 16: return warp_kernel<T, KIND, GRAD, 16><<<l.grid, kRowThreads, 0, s>>>(*a, l.batch);
    }
  if (l.team == 32) row_kernel<T, KIND, GRAD, 32><<<l.grid, kRowThreads, l.smem, s>>>(*a, l.hash);
  else row_kernel<T, KIND, GRAD, kRowThreads><<<l.grid, kRowThreads, l.smem, s>>>(*a, l.hash);
}

template <int KIND>
int launch_head(const LzLossArgs* a, bool order, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {a->rows > kHeadRows ? (unsigned)kMaxCluster : 1u, 1, 1};
  cfg.gridDim = dim3(at[0].val.clusterDim.x), cfg.blockDim = dim3(kThreads), cfg.stream = s, cfg.attrs = at, cfg.numAttrs = 1;
  LZ_CUDA_TRY(cudaLaunchKernelEx(&cfg, head_kernel<KIND>, *a, order));
  return LZE_OK;
}

template <typename T, int KIND>
int forward_as(const LzLossArgs* a, cudaStream_t s) {
  LzStreamPlan stream;
  if (const int rc = lz_stream_plan(a, &stream)) return rc;
  if (KIND != LZ_LOSS_LOGP || stream.ordered) {
    if (const int rc = launch_head<KIND>(a, stream.ordered, s)) return rc;
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
  if (KIND != LZ_LOSS_DISTILL && l.team == 8) warp_grad_kernel<T, KIND, 8><<<l.grid, kRowThreads, 0, s>>>(*a, l.batch);
  else if (KIND != LZ_LOSS_DISTILL && l.team == 16) warp_grad_kernel<T, KIND, 16><<<l.grid, kRowThreads, 0, s>>>(*a, l.batch);
  else if (l.team == 32) row_grad_kernel<T, KIND, 32><<<l.grid, kRowThreads, l.smem, s>>>(*a, l.hash);
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

// The id of the graph capture that the stream is in, 0 for none.
unsigned long long capture_of(cudaStream_t s) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(s, &status, &id) != cudaSuccess) {
    cudaGetLastError();  // the legacy stream while another one is captured: not in a capture itself
    return 0;
  }
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

int run(LzLossArgs* a, cudaStream_t s, bool forward) {
  if (a->kind < LZ_LOSS_LOGP || a->kind > LZ_LOSS_DISTILL || a->rows < 0 || a->vocab < 1 || a->vocab > INT32_MAX ||
      a->inner < 1 || a->inv_temperature <= 0.f ||
      (a->kind == LZ_LOSS_DISTILL && (a->top < 1 || a->top > LZ_LOSS_MAX_TOP))) {
    lz_set_error("loss: bad arguments (kind %d, rows %lld, vocabulary %lld, top %d)", a->kind, a->rows, a->vocab, a->top);
    return LZE_ARG;
  }
  const OnDevice on(a->device);
  LZ_CUDA_TRY(on.rc);
  if (forward && a->grad) a->capture = capture_of(s);
  if (!forward && !a->fresh && a->capture != capture_of(s)) return LZ_LOSS_APART;
  switch (a->dtype) {
    case LZ_F32: return run_kind<float>(a, s, forward);
    case LZ_F16: return run_kind<__half>(a, s, forward);
    case LZ_BF16: return run_kind<__nv_bfloat16>(a, s, forward);
  }
  lz_set_error("loss: dtype %d", a->dtype);
  return LZE_ARG;
}

}  // namespace

extern "C" int lz_loss_forward(LzLossArgs* a, cudaStream_t stream) { return run(a, stream, true); }

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
