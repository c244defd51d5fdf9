// Vocabulary losses on large vocabularies: a cluster of CTAs a row, each with a slice of it.
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
#include <algorithm>
#include <atomic>

#include "lz_losses_dev.cuh"

namespace {

constexpr int kMaxSlots = 64;
constexpr unsigned long long kWaitNs = 4000000000ull;  // bound of every wait where the caller gives none

// Which row, and this CTA's slice of it.
struct RowHead {
  long long row;  // -1: no more
  int lead, vecs, first, count, chunks;
};

constexpr int kListWarps = 2;

// The lists (id, z, q, share) of `views` rows, and each list warp's hash table.
__host__ __device__ inline int list_bytes(int kind, int top, int hash, int views) {
  return kind == LZ_LOSS_DISTILL ? (top * 16 * views + hash * 4 * kListWarps + 127) / 128 * 128 : 0;
}

// Every wait for a phase of a barrier is bounded. One that gives up marks its CTA. Nobody hands on
// what a marked CTA has of a row, so what others still receive is right; its warps leave their
// loops and tell all CTAs of the cluster, whose other waits then give up at once unless their
// phase is there. When all threads have left, every CTA of the cluster writes NaN over the
// outputs and gradients of the cluster's rows. In us, without and with the looks at the mark:
// 1024 rows of 608 KB with policy's gradient 221 / 223, 600 of 200 KB with DISTILL's 65.6 / 67.7,
// sums only 1 row of 300 KB 6.6 / 6.9, 4096 rows 191 / 195.
struct WaitState {
  unsigned long long limit;  // ns
  int failed;                // kFailed, or from the start kNoWait: what is not there at once is given up
};
constexpr int kFailed = 1, kNoWait = 2;

LZ_DEV void init_waits(WaitState* w, unsigned long long limit) {
  w->limit = limit;
  w->failed = limit == 1 ? kNoWait : 0;
}
LZ_DEV bool gave_up(const WaitState* w) { return *(const volatile int*)&w->failed == kFailed; }

struct alignas(128) StreamShared {
  uint64_t full[kMaxSlots], empty[kMaxSlots];
  uint64_t parts[2], peers[2], dense[2];  // of every other row
  uint64_t ready[4], used[4];             // of every row's scalars and list, in turn
  float2 warp_part[2][16];
  float2 peer_part[2][kMaxCluster];
  RowHead heads[4];
  RowGrad grad[2];
  RowParams params[4];
  WaitState waits;
};

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
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile WaitState* w) {
  unsigned long long began = 0;
  for (uint32_t it = 1; it; ++it) {
    if (try_wait<CLUSTER>(bar, parity)) return true;
    if (w->failed) break;
    if (it % 64 == 0) {
      const unsigned long long now = globaltimer();
      if (!began) began = now;
      if (now - began > w->limit) break;
    }
  }
  w->failed = kFailed;
  return false;
}

// Whether the phase came; lanes of a warp may differ.
template <bool CLUSTER>
LZ_DEV bool ring_wait(uint64_t* bar, uint32_t parity, WaitState* w) {
  return try_wait<CLUSTER>(smem_addr(bar), parity) || wait_on<CLUSTER>(smem_addr(bar), parity, w);
}

// One lane, when it or its warp has given up.
LZ_DEV void tell_cluster(const WaitState* w) {
  for (uint32_t rank = 0, ranks = cluster_size(); rank < ranks; ++rank)
    asm volatile(
        "{\n\t.reg .b32 p;\n\t"
        "mapa.shared::cluster.u32 p, %0, %1;\n\t"
        "st.shared::cluster.u32 [p], %2;\n\t}" ::"r"(smem_addr(&w->failed)),
        "r"(rank), "r"(kFailed)
        : "memory");
}

// After a wait that gave up: copies and peers' values still in flight land before the CTA ends.
LZ_DEV void drain_copies() {
  const unsigned long long began = globaltimer();
  for (uint32_t it = 0; it < 100000000u && globaltimer() - began < 20000000ull; ++it) {
  }
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

// Warps beside the W that take chunks: one feeds the ring, one has the rows'
// scalars; DISTILL's lists take two more (about 9000 cycles for 64 entries, of
// the 15000 that a slice of 150 KB takes), so that short rows need not wait for them.
template <int KIND>
constexpr int kHelpers = KIND == LZ_LOSS_DISTILL ? 2 + kListWarps : 2;

template <typename T, int KIND, bool GRAD, int W>
__global__ void __launch_bounds__((W + kHelpers<KIND>) * 32, 1) stream_kernel(const __grid_constant__ LzLossArgs a,
                                                                 const __grid_constant__ LzStreamPlan plan) {
  constexpr int N = Elem<T>::N, kTake = W * 32;
  constexpr int kChunkVecs = kBatch * kTake, kChunk = 16 * kChunkVecs;
  extern __shared__ __align__(128) char smem[];
  StreamShared& sh = *reinterpret_cast<StreamShared*>(smem);
  char* const lists = smem + sizeof(StreamShared);
  char* const ring = lists + list_bytes(KIND, a.top, plan.hash, plan.views);
  const uint32_t views = KIND == LZ_LOSS_DISTILL ? plan.views : 2, views_log2 = views == 4 ? 2 : 1;  // rows whose scalars are kept
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const long long cluster = blockIdx.x / ranks, clusters = gridDim.x / ranks;
  const float c = (float)(kLog2e * (double)a.inv_temperature);
  WaitState* const waits = &sh.waits;
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
    }
    for (int k = 0; k < 4; ++k) {
      mbar_init(&sh.ready[k], 1);
      mbar_init(&sh.used[k], 1);
    }
    fence_mbar_init();
    init_waits(waits, plan.wait_ns);
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
        for (int k = 0; k < h.chunks; ++k) {
          if (round && !ring_wait<false>(&sh.empty[slot], (round - 1) & 1, waits)) {
            tell_cluster(waits);
            goto fed;
          }
          const int vecs = min(kChunkVecs, h.count - k * kChunkVecs);
          bulk_g2s(ring + (size_t)slot * kChunk, from + (size_t)k * kChunk, vecs * 16, &sh.full[slot]);
          if (++slot == (uint32_t)plan.slots) slot = 0, ++round;
        }
        h = next;
      }
    fed:;
    }
    __syncwarp();
  } else if (warp < W) {  // ---- sums, then the dense gradient
    uint32_t slot = 0, round = 0;      // where the sums are
    uint32_t again = 0;                // where the gradient is
    LazySum sum;
    sum.init(c);
    int done = 0;  // chunks of the row that are in `sum`
    // Chunks [done, upto) of a row. Where one does not come its slot is read all the same, so that a warp
    // stays together, but not handed back to the ring.
    auto take = [&](const RowHead& h, int upto) {
      for (; done < upto; ++done) {
        const int vecs = h.count - done * kChunkVecs;
        const bool came = ring_wait<false>(&sh.full[slot], round & 1, waits);
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
          if (lane == 0 && came) mbar_arrive(&sh.empty[slot]);
        }
        if (++slot == (uint32_t)plan.slots) slot = 0, ++round;
      }
    };
    uint32_t turn = 0;
    for (;; ++turn) {
      // The row's head is there, and its place in `warp_part` free, when the row two before it is done with.
      const int k = turn & 1;
      if (!GRAD && turn >= 2) {
        ring_wait<false>(&sh.dense[k], ((turn - 2) >> 1) & 1, waits);
        __syncwarp();
        if (gave_up(waits)) break;  // a load of the whole warp: the same in every lane
      }
      const RowHead h = sh.heads[turn & 3];
      if (h.row < 0) break;
      const long long single = rank == 0 && tid < 2 * N ? single_of(h.lead, h.vecs, N, tid, a.vocab) : -1;
      float alone = 0.f;
      if (single >= 0) alone = Elem<T>::get(row_of<T>(a, h.row)[single]);
      take(h, h.chunks);
      if (single >= 0) sum.take_one(alone, c);
      float m = sum.ref, all = sum.total();
      lanes_join(m, all, 32);
      __syncwarp();
      if (lane == 0) {
        sh.warp_part[k][warp] = make_float2(m, all);
        mbar_arrive(&sh.parts[k]);
      }
      sum.init(c);
      done = 0;
      if (!GRAD) continue;
      const RowHead& next = sh.heads[(turn + 1) & 3];
      if (next.row >= 0) take(next, min(plan.early, next.chunks));
      ring_wait<false>(&sh.dense[k], (turn >> 1) & 1, waits);
      __syncwarp();
      if (gave_up(waits)) break;
      const RowGrad d = sh.grad[k];
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
            const uint4 e = dense_vector<T>(w[u], c2, off2, f2);
            if (tid + u * kTake < vecs) st_cs_v4(o + tid + u * kTake, e);
          }
        } else {
          for (int j = tid; j < min(vecs, kChunkVecs); j += kTake) {
            float e[N];
            Elem<T>::unpack(v[j], e);
#pragma unroll
            for (int q = 0; q < N; ++q) e[q] = d.dense(e[q], c);
            st_cs_v4(o + j, Elem<T>::pack(e));
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[again]);
        if (++again == (uint32_t)plan.slots) again = 0;
      }
      if (single >= 0)
        out[single] = Elem<T>::put(d.f == 0.f ? 0.f : d.dense(alone, c));
    }
    __syncwarp();
    const bool there = !gave_up(waits);
    if (!there && lane == 0) tell_cluster(waits);
    if (GRAD && there) {
      if (lane == 0) mbar_arrive(&sh.parts[turn & 1]);  // the last row is written
      for (long long i = (plan.ordered ? active : 0) + cluster; i < limit; i += clusters) {
        long long r;
        if (row_at(i, &r)) continue;
        T* out = static_cast<T*>(a.grad) + r * a.vocab;
        const RowHead h = slice_of(out, r, a.vocab, rank, ranks, kChunkVecs);
        uint4* o = reinterpret_cast<uint4*>(out + h.lead) + h.first;
        for (int j = tid; j < h.count; j += kTake) st_cs_v4(o + j, make_uint4(0, 0, 0, 0));
        const long long single = rank == 0 && tid < 2 * N ? single_of(h.lead, h.vecs, N, tid, a.vocab) : -1;
        if (single >= 0) out[single] = Elem<T>::put(0.f);
      }
    }
  } else if (KIND == LZ_LOSS_DISTILL && warp >= W + 2) {  // ---- the teacher's lists, by one warp or in turns
    const uint32_t mine = warp - (W + 2);
    int* const hash = reinterpret_cast<int*>(lists) + 4 * views * a.top + mine * plan.hash;
    long long r, to_come;
    for (uint32_t turn = mine; mine < views / 2 && row_at(cluster + (long long)turn * clusters, &r); turn += views / 2) {
      const int k = turn & (views - 1);
      if (row_at(cluster + (long long)(turn + views) * clusters, &to_come)) touch_list(a, to_come);
      if (turn >= views && !__all_sync(~0u, ring_wait<false>(&sh.used[k], ((turn >> views_log2) - 1) & 1, waits))) {
        if (lane == 0) tell_cluster(waits);
        break;
      }
      prepare_params<T, KIND>(a, row_of<T>(a, r), r, sh.params[k], view(k), hash, plan.hash, c);
      if (lane == 0) mbar_arrive(&sh.ready[k]);
      if (row_at(cluster + (long long)(turn + views / 2) * clusters, &to_come))
        touch_logits(a, row_of<T>(a, to_come), to_come);
    }
    __syncwarp();
  } else {  // ---- joins the sums; the rows' scalars, outputs and sparse entries
    double loss = 0.0;
    RowHead before = {-1};  // the row whose dense part is being written, its token and gradient
    RowGrad before_grad;
    float before_xy = 0.f;
    int before_token = -1;
    auto sparse = [&](int k) {
      if (!GRAD || before.row < 0 || before_grad.f == 0.f) return;
      T* out = static_cast<T*>(a.grad) + before.row * a.vocab;
      const long long lo = before.lead + (long long)before.first * N, hi = lo + (long long)before.count * N;
      const long long tail = before.lead + (long long)before.vecs * N;
      auto put = [&](int id, float x, float t) {
        if ((id >= lo && id < hi) || (rank == 0 && (id < before.lead || id >= tail)))
          out[id] = Elem<T>::put(before_grad.sparse(x, t, c));
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
        prepare_params<T, KIND>(a, row_of<T>(a, h.row), h.row, sh.params[k], TopView{}, nullptr, 0, c);
    };
    prepare(sh.heads[0], 0);
    uint32_t turn = 0;
    for (;; ++turn) {
      const RowHead h = sh.heads[turn & 3];
      if (h.row < 0) break;
      const int k = turn & 1, at = turn & (views - 1), last = (turn - 1) & (views - 1);
      const RowHead later = head_at(cluster + (long long)(turn + 2) * clusters);
      ring_wait<false>(&sh.parts[k], (turn >> 1) & 1, waits);
      float2 v = lane < W ? sh.warp_part[k][lane] : make_float2(-INFINITY, 0.f);
      lanes_join(v.x, v.y, W);
      if (ranks > 1) {
        __syncwarp();
        if (gave_up(waits)) break;
        if (lane == 0) mbar_expect(&sh.peers[k], ranks * (uint32_t)sizeof(float2));
        if (lane < ranks) send_to_peer(&sh.peer_part[k][rank], v, &sh.peers[k], lane);
        __syncwarp();
        ring_wait<true>(&sh.peers[k], (turn >> 1) & 1, waits);
        v = lane < ranks ? sh.peer_part[k][lane] : make_float2(-INFINITY, 0.f);
        lanes_join(v.x, v.y, kMaxCluster);
      }
      RowSum n = {0.f, v.x, v.y};
      if (KIND == LZ_LOSS_DISTILL) ring_wait<false>(&sh.ready[at], (turn >> views_log2) & 1, waits);
      __syncwarp();
      if (gave_up(waits)) break;
      if (!exact_ref(v.x)) n = slow_sum(row_of<T>(a, h.row), a.vocab, c);
      const RowParams& p = sh.params[at];
      const RowOut o = row_out<KIND>(a, p, n.norm(), c);
      const RowGrad g(o.slope, a.inv_temperature, n);
      if (lane == 0) {
        sh.grad[k] = g;
        sh.heads[(turn + 2) & 3] = later;
        mbar_arrive(&sh.dense[k]);
      }
      sparse(last);
      __syncwarp();
      if (KIND == LZ_LOSS_DISTILL && turn && lane == 0) mbar_arrive(&sh.used[last]);  // by the row before
      if (rank == 0) loss += row_outputs<KIND>(a, p, o, n, view(at), h.row, c);
      before = h, before_grad = g, before_xy = p.xy, before_token = p.token;
      __syncwarp();
      prepare(sh.heads[(turn + 1) & 3], k ^ 1);
    }
    if (GRAD && !gave_up(waits)) ring_wait<false>(&sh.parts[turn & 1], (turn >> 1) & 1, waits);
    __syncwarp();
    const bool there = !gave_up(waits);
    if (GRAD && there) sparse((turn - 1) & (views - 1));
    if (!there && lane == 0) tell_cluster(waits);
    if (rank == 0) {
      long long r;
      for (long long i = (plan.ordered ? active : 0) + cluster + lane * clusters; i < limit; i += 32 * clusters) {
        if (!row_at(i, &r)) no_outputs<KIND>(a, r);
      }
      if (!there) loss = NAN;
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
  if (!gave_up(waits)) return;
  drain_copies();
  for (long long i = cluster; i < limit; i += clusters) {
    long long r;
    row_at(i, &r);
    if (GRAD) {
      T* out = static_cast<T*>(a.grad) + r * a.vocab;
      const long long per = (a.vocab + ranks - 1) / ranks, end = min((rank + 1) * per, a.vocab);
      for (long long j = rank * per + tid; j < end; j += blockDim.x) out[j] = Elem<T>::put(NAN);
    }
    if (rank == 0 && tid == 0) {
      if (KIND != LZ_LOSS_DISTILL) a.logp[r] = NAN;
      if (KIND == LZ_LOSS_DISTILL || (KIND == LZ_LOSS_POLICY && a.ref_logp)) a.kl[r] = NAN;
      if (KIND == LZ_LOSS_POLICY) a.clipped[r] = 0;
      work_sum(a)[r] = make_float4(0.f, 0.f, NAN, 0.f);  // the backward pass's too
      work_slope(a)[r] = NAN;
    }
  }
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
  WaitState waits;
};

template <typename T, int KIND, int W>
__global__ void __launch_bounds__((W + 1) * 32, 1) stream_grad_kernel(const __grid_constant__ LzLossArgs a, int slots,
                                                                      unsigned long long limit_ns) {
  constexpr int N = Elem<T>::N, kTake = W * 32;
  constexpr int kChunkVecs = kBatch * kTake, kChunk = 16 * kChunkVecs;
  extern __shared__ __align__(128) char smem[];
  GradShared& sh = *reinterpret_cast<GradShared*>(smem);
  char* const ring = smem + sizeof(GradShared);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const float c = (float)(kLog2e * (double)a.inv_temperature);
  WaitState* const waits = &sh.waits;
  const float up = a.upstream ? *a.upstream : 1.f;
  if (!a.fresh && up == 1.f) return;
  if (tid == 0) {
    for (int s = 0; s < slots; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], W);
    }
    fence_mbar_init();
    init_waits(waits, limit_ns);
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
        const float4 sum = work_sum(a)[r];
        const long long y = load_id(a.ids, a.ids64, r);
        const double slope = row_slope_for<KIND>(a, r, y, up);
        const Split<T> sp(x, a.vocab);
        h.vecs = max(0, min(kChunkVecs, sp.vecs - piece * kChunkVecs));
        const long long at = sp.lead + (long long)piece * kChunkVecs * N;
        h.out = out + at;
        h.row = x, h.out_row = out;
        h.singles = piece == 0, h.lead = sp.lead, h.tail = (int)(a.vocab - sp.lead) % N;
        const RowGrad d((float)slope, a.inv_temperature, RowSum{sum.x, sum.y, sum.z});
        h.f = d.f, h.base = d.base, h.ref = d.ref;
        h.token = -1, h.token_vec = -1;
        if (y >= 0 && y < a.vocab && h.f != 0.f) {
          const long long in = y - at;
          if (in >= 0 && in < (long long)h.vecs * N) h.token_vec = (int)(in / N), h.token_at = (int)(in % N);
          else if (h.singles && (y < sp.lead || y >= a.vocab - h.tail)) h.token = (int)y;
          if (h.token_vec >= 0 || h.token >= 0) h.token_value = d.sparse(Elem<T>::get(x[y]), 1.f, c);
        }
        from = reinterpret_cast<const char*>(x + at);
      }
      bool free = true;
      for (int l = 0; l < 32 && first + (long long)l * gridDim.x < all; ++l) {
        if (lane == l) {
          free = !round || ring_wait<false>(&sh.empty[slot], (round - 1) & 1, waits);
          if (free) {
            sh.heads[slot] = h;
            if (h.f != 0.f && h.vecs > 0) bulk_g2s(ring + (size_t)slot * kChunk, from, h.vecs * 16, &sh.full[slot]);
            else mbar_arrive(&sh.full[slot]);  // nothing to read
          }
        }
        free = __shfl_sync(~0u, free, l);
        if (!free) break;
        if (++slot == (uint32_t)slots) slot = 0, ++round;
      }
      if (!free) break;
    }
  } else {
    uint32_t slot = 0, round = 0;
    for (long long g = blockIdx.x; g < all; g += gridDim.x) {
      if (!__all_sync(~0u, ring_wait<false>(&sh.full[slot], round & 1, waits))) break;
      const ChunkHead& h = sh.heads[slot];
      const uint4* v = reinterpret_cast<const uint4*>(ring + (size_t)slot * kChunk) + tid;
      uint4* o = static_cast<uint4*>(h.out) + tid;
      const int vecs = h.vecs;
      const float f = h.f, base = h.base, ref = h.ref;
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
          uint4 e;
          if (base == 0.f) {
            e = dense_vector<T>(w[u], c2, off2, f2);
          } else {
            float x[N];
            Elem<T>::unpack(w[u], x);
#pragma unroll
            for (int q = 0; q < N; ++q) x[q] = f * exp2_fast(fmaf(x[q] - base, c, -ref));
            e = Elem<T>::pack(x);
          }
          if (tid + u * kTake < vecs) st_cs_v4(o + u * kTake, e);
        }
        if (token_vec >= 0 && token_vec % kTake == tid)  // over its vector, by the thread that wrote it
          reinterpret_cast<T*>(static_cast<uint4*>(h.out) + token_vec)[h.token_at] = Elem<T>::put(h.token_value);
      }
      if (h.singles && tid < h.lead + h.tail) {
        const long long i = tid < h.lead ? tid : a.vocab - h.tail + tid - h.lead;
        float e = 0.f;
        if (f != 0.f) e = i == h.token ? h.token_value : f * exp2_fast(fmaf(Elem<T>::get(static_cast<const T*>(h.row)[i]) - base, c, -ref));
        static_cast<T*>(h.out_row)[i] = Elem<T>::put(e);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[slot]);
      if (++slot == (uint32_t)slots) slot = 0, ++round;
    }
  }
  __syncthreads();
  if (!gave_up(waits)) return;
  drain_copies();
  for (long long g = blockIdx.x; g < all; g += gridDim.x) {  // this CTA's chunks are NaN, not stale
    const long long r = g / per_row, piece = g % per_row;
    T* out = static_cast<T*>(a.grad) + r * a.vocab;
    const Split<T> sp(out, a.vocab);
    const long long at = sp.lead + piece * kChunkVecs * N, end = min(at + (long long)kChunkVecs * N, sp.lead + (long long)sp.vecs * N);
    for (long long j = at + tid; j < end; j += blockDim.x) out[j] = Elem<T>::put(NAN);
    if (piece == 0)
      for (long long t = tid; t < 2 * N; t += blockDim.x) {
        const long long single = single_of(sp.lead, sp.vecs, N, (int)t, a.vocab);
        if (single >= 0) out[single] = Elem<T>::put(NAN);
      }
  }
}

// Whether rows are streamed: not small, and each row and its gradient at the same
// offset from a 16-byte border. A row costs a cluster some 5000 cycles besides its
// bytes, which the many teams of row_kernel hide better while rows are short; it
// reads a row that outgrows the caches a second time. Few rows are streamed from
// 16 KB on, since a cluster splits them. In us, bf16, streamed against teams:
//   policy's gradient: 64 rows of 16 KB 15 / 14, of 32 KB 14 / 16, of 64 KB 16 / 21; 1024 of 48 KB 35 / 33, of
//     64 KB 42 / 43, of 80 KB 49 / 56; 8192 of 40 KB 180 / 162, of 48 KB 187 / 194, of 64 KB 208 / 266
//   DISTILL's, 64 entries: 64 rows of 32 KB 21 / 18, of 80 KB 21 / 23; 1024 of 72 KB 56 / 52, of 80 KB 57 / 60; 4096
//     of 40 KB 139 / 100, of 56 KB 139 / 138, of 64 KB 146 / 159. Long lists bound the streamed rows: 4096
//     of 64 KB with 128 entries 244 / 163
//   sums only: 64 rows of 64 KB 10 / 10, of 160 KB 10 / 14; LOGP 1024 of 128 KB 36 / 33, of 300 KB 62 / 62, of 600 KB
//     105 / 111, 4096 of 300 KB 220 / 211; policy 2048 of 128 KB 62 / 61, of 200 KB 80 / 82, of 400 KB 140 / 156
//   the gradient alone: 1024 rows of 64 KB 25 / 21, 8192 of 100 KB 256 / 266
// The borders are round numbers; next to them the other side is up to 10 % faster, for DISTILL of 4096
// rows and more from 40 to 52 KB up to 28 %.
template <typename T>
bool streams(const LzLossArgs* a, bool forward, bool grad) {
  const long long size = sizeof(T), row = a->vocab * size;
  const long long from = a->rows <= 64 && forward ? 16 : !forward ? 64 : !grad ? 128 : a->kind != LZ_LOSS_DISTILL || a->rows >= 4096 ? 40 : 80;
  if (row < from * 1024 || a->rows > INT32_MAX) return false;
  if (!grad) return true;
  return ((uintptr_t)a->logits ^ (uintptr_t)a->grad) % 16 == 0 &&
         (a->inner >= a->rows || (a->outer_stride * size - a->inner * row) % 16 == 0) &&
         (a->inner <= 1 || (a->inner_stride * size - row) % 16 == 0);
}

constexpr int kStreamWarps = 16;
constexpr int kChunk = 16 * kBatch * kStreamWarps * 32;  // bytes of a ring slot: a batch of every thread
constexpr int kSharedMax = 232448;

template <typename T, int KIND, bool GRAD>
int plan_as(const LzLossArgs* a, LzStreamPlan* l) {
  const long long row = a->vocab * (long long)sizeof(T);
  if (!streams<T>(a, true, GRAD)) return LZE_OK;
  int hash = 0;
  if (KIND == LZ_LOSS_DISTILL && a->top > kSmallList)
    for (hash = 32; hash < 2 * a->top;) hash *= 2;
  const int two = (int)sizeof(StreamShared) + list_bytes(KIND, a->top, hash, 2);
  const int four = (int)sizeof(StreamShared) + list_bytes(KIND, a->top, hash, 4);
  const int slots = std::min((kSharedMax - two) / kChunk, kMaxSlots);
  auto kernel = stream_kernel<T, KIND, GRAD, kStreamWarps>;
  static std::atomic<bool> known[kMaxDevices];
  static std::atomic<int> resident[kMaxDevices][kMaxCluster];
  if (!known[a->device].load(std::memory_order_acquire)) {
    LZ_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax));
    for (int k = 0; k < kMaxCluster; ++k) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute at[1] = {};
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim = {k + 1u, 1, 1};
      cfg.gridDim = dim3(840), cfg.blockDim = dim3((kStreamWarps + kHelpers<KIND>) * 32), cfg.dynamicSmemBytes = kSharedMax;
      cfg.attrs = at, cfg.numAttrs = 1;
      int g = 0;
      LZ_CUDA_TRY(cudaOccupancyMaxActiveClusters(&g, kernel, &cfg));
      resident[a->device][k].store(g, std::memory_order_relaxed);
    }
    known[a->device].store(true, std::memory_order_release);
  }
  // CTAs a row: the fewest bytes by the busiest cluster, a row's exchange counted as 50 KB. In us with 0 / 25 / 50 /
  // 200 KB, policy's gradient: 515 rows of 64 KB 38.4 / 32.8 / 32.8 / 32.7, 4000 of 200 KB 284 / 272 / 274 / 273, 300
  // of 120 KB 32.8 / 32.8 / 30.8 / 31.2.
  double best = 0.0;
  int chunks = 0;
  long long part = 0;
  for (int k = 0; k < kMaxCluster; ++k) {
    const int ranks = k + 1, g = resident[a->device][k].load(std::memory_order_relaxed);
    const long long slice = (row + ranks - 1) / ranks;
    if (g < 1 || (GRAD && (slice + 16 + kChunk - 1) / kChunk > slots)) continue;
    const double cost = (double)((a->rows + g - 1) / g) * ((double)slice * (GRAD ? 2 : 1) + 50e3);
    if (best != 0.0 && cost >= best) continue;
    best = cost;
    l->ranks = ranks;
    l->clusters = (int)(a->rows < g ? a->rows : g);
    chunks = (int)((slice + 16 + kChunk - 1) / kChunk), part = slice;
  }
  l->slots = slots, l->early = slots - chunks, l->ordered = a->rows > l->clusters, l->hash = hash;
  // Lists of four rows where a list takes longer than a row (8192 rows of 64 KB 371 us, 236 with
  // four) and the ring loses no slot. With two, a list's logits are read when its row is on the
  // way to L2 (4096 rows of 300 KB 425 us, with four 438).
  l->views = part <= 128 * 1024 && (kSharedMax - four) / kChunk >= slots ? 4 : 2;
  const int fixed = l->views == 4 ? four : two;
  l->smem = fixed + (size_t)slots * kChunk;
  l->wait_ns = a->wait_ns ? a->wait_ns : kWaitNs;
  return LZE_OK;
}

template <typename T, int KIND, bool GRAD>
int launch_as(const LzLossArgs* a, const LzStreamPlan& l, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)l.ranks, 1, 1};
  cfg.gridDim = dim3(l.clusters * l.ranks), cfg.blockDim = dim3((kStreamWarps + kHelpers<KIND>) * 32);
  cfg.dynamicSmemBytes = l.smem, cfg.stream = s, cfg.attrs = at, cfg.numAttrs = 1;
  LZ_CUDA_TRY(cudaLaunchKernelEx(&cfg, stream_kernel<T, KIND, GRAD, kStreamWarps>, *a, l));
  return LZE_OK;
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
  kernel<<<n, (kStreamWarps + 1) * 32, sizeof(GradShared) + (size_t)slots * kChunk, s>>>(*a, slots, a->wait_ns ? a->wait_ns : kWaitNs);
  LZ_CUDA_TRY(cudaGetLastError());
  return LZE_OK;
}

// Calls f<T, KIND, GRAD> for these arguments.
#define LZ_LOSS_CASES(F, ...)                                                                                       \
  do {                                                                                                              \
    switch (a->dtype) {                                                                                             \
      case LZ_F32: return F<float> __VA_ARGS__;                                                                     \
      case LZ_F16: return F<__half> __VA_ARGS__;                                                                    \
      default: return F<__nv_bfloat16> __VA_ARGS__;                                                                 \
    }                                                                                                               \
  } while (0)

template <typename T>
int plan_kind(const LzLossArgs* a, LzStreamPlan* l) {
  if (a->kind == LZ_LOSS_LOGP) return plan_as<T, LZ_LOSS_LOGP, false>(a, l);
  if (a->kind == LZ_LOSS_POLICY)
    return a->grad ? plan_as<T, LZ_LOSS_POLICY, true>(a, l) : plan_as<T, LZ_LOSS_POLICY, false>(a, l);
  return a->grad ? plan_as<T, LZ_LOSS_DISTILL, true>(a, l) : plan_as<T, LZ_LOSS_DISTILL, false>(a, l);
}

template <typename T>
int launch_kind(const LzLossArgs* a, const LzStreamPlan& l, cudaStream_t s) {
  if (a->kind == LZ_LOSS_LOGP) return launch_as<T, LZ_LOSS_LOGP, false>(a, l, s);
  if (a->kind == LZ_LOSS_POLICY)
    return a->grad ? launch_as<T, LZ_LOSS_POLICY, true>(a, l, s) : launch_as<T, LZ_LOSS_POLICY, false>(a, l, s);
  return a->grad ? launch_as<T, LZ_LOSS_DISTILL, true>(a, l, s) : launch_as<T, LZ_LOSS_DISTILL, false>(a, l, s);
}

template <typename T>
int grad_kind(const LzLossArgs* a, cudaStream_t s) {
  return a->kind == LZ_LOSS_LOGP ? launch_stream_grad<T, LZ_LOSS_LOGP>(a, s) : launch_stream_grad<T, LZ_LOSS_POLICY>(a, s);
}

}  // namespace

int lz_stream_plan(const LzLossArgs* a, LzStreamPlan* plan) {
  *plan = LzStreamPlan{};
  if (!a->rows || a->device < 0 || a->device >= kMaxDevices) return LZE_OK;
  LZ_LOSS_CASES(plan_kind, (a, plan));
}

int lz_stream_forward(const LzLossArgs* a, const LzStreamPlan* plan, cudaStream_t stream) {
  LZ_LOSS_CASES(launch_kind, (a, *plan, stream));
}

bool lz_stream_grad_fits(const LzLossArgs* a) {
  if (a->kind == LZ_LOSS_DISTILL || a->device < 0 || a->device >= kMaxDevices) return false;
  LZ_LOSS_CASES(streams, (a, false, true));
}

int lz_stream_grad(const LzLossArgs* a, cudaStream_t stream) { LZ_LOSS_CASES(grad_kind, (a, stream)); }
