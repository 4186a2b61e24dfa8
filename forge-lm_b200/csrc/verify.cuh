// verify.cuh — drafted tokens against the target's probabilities, and the token
// that follows the accepted ones (include/forge_b200.h, fb2_verify_drafts, has
// the rules).
//
// Two kernels.  k_verify_rows reads every row of logits once: its largest and
// sum of exp((l - largest) / T), or where it is largest for T <= 0.
// k_verify_walk takes a sequence: the drafts' probabilities are looked up at once
// and walked down by one thread; then the row at which the walk ended is weighed
// (without rejected tokens, or less the draft's probabilities), its sums over
// parts in the order of ids say in which part the draw falls, and that part is
// looked through.
//
// Which id a draw gives hangs on running sums over a whole row: in 32 bits they
// are off by some 1e-7 of the total, wider than most tokens of a large vocabulary,
// so exponentials and sums are in 64 bits here.
#pragma once
#include "kvq.cuh"
#include "pages.cuh"

namespace fb2 {

constexpr int VF_THREADS = 256, VF_WARPS = VF_THREADS / 32, VF_NODES = 1024, VF_RANKS = 8;

struct VerifyRow {
    double sum;  // of exp((l - top) / T); not positive and finite where the row has no probabilities
    float top;
    int best;  // the lowest id of the largest logit (T <= 0)
};
struct VerifyArgs {
    const void* logits;
    const float* probs;
    const int *drafts, *starts, *parents;
    const double* uniforms;
    const float* temperature;
    int *tokens, *nodes, *counts;
    VerifyRow* rows;
    long long logits_row, probs_row;
    int n_seqs, n_rows, vocab, max_nodes, ranks;  // ranks: CTAs of a cluster
    // the rows of sequence b
    FB2_DEV void rows_of(int b, int& first, int& last) const {
        if (!starts) {
            first = b, last = b + 1;
            return;
        }
        first = min(max(__ldg(starts + b), 0), n_rows);
        last = min(max(__ldg(starts + b + 1), first), n_rows);
        last = min(last, first + max_nodes);
    }
    FB2_DEV float heat(int b) const { return temperature ? __ldg(temperature + b) : 1.f; }
};

namespace vf {

FB2_DEV uint32_t cluster_map(uint32_t at, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    return r;
}
FB2_DEV double peek(const double* p, int rank) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(cluster_map((uint32_t)__cvta_generic_to_shared(p), rank)) : "memory");
    return v;
}
FB2_DEV int peek(const int* p, int rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_map((uint32_t)__cvta_generic_to_shared(p), rank)) : "memory");
    return v;
}
FB2_DEV float peek(const float* p, int rank) { return __int_as_float(peek(reinterpret_cast<const int*>(p), rank)); }
FB2_DEV double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// exp((l - top) / T) with cold = 1 / T; 0 for l = -inf, whatever T is
FB2_DEV double weight(float l, float top, double cold) {
    return l == -INFINITY ? 0.0 : exp(((double)l - (double)top) * cold);
}
// The sequence of a row: the last b with starts[b] <= row, by all lanes.
FB2_DEV int owner(const int* starts, int n, int row) {
    int lo = 0, hi = n;  // starts[lo] <= row (or lo = 0), starts[hi] > row (or hi = n)
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + (int)(threadIdx.x & 31) * step;
        const uint32_t le = __ballot_sync(0xffffffffu, at == lo || (at < hi && __ldg(starts + at) <= row));
        const int last = 31 - __clz(le);
        lo += last * step;
        hi = min(hi, lo + step);
    }
    return lo;
}
FB2_DEV bool proper(double sum) { return sum > 0.0 && sum < INFINITY; }

}  // namespace vf

// A cluster to a row; its CTAs each take a part of it.
template <class T>
__global__ void __launch_bounds__(VF_THREADS) k_verify_rows(VerifyArgs a) {
    __shared__ double s_sum[VF_WARPS], c_sum;
    __shared__ float s_top[VF_WARPS], c_top;
    __shared__ int s_best[VF_WARPS], c_best;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ranks = a.ranks, rank = blockIdx.x % ranks, row = blockIdx.x / ranks;
    const int b = a.starts ? vf::owner(a.starts, a.n_seqs, row) : row;
    int first, last;
    a.rows_of(b, first, last);
    if (row < first || row >= last) {  // the whole cluster
        if (rank == 0 && tid == 0) a.rows[row] = {0.0, -INFINITY, -1};
        return;
    }
    const float heat = a.heat(b);
    const bool greedy = !(heat > 0.f);
    const double cold = greedy ? 0.0 : 1.0 / (double)heat;
    const T* p = (const T*)a.logits + row * a.logits_row;
    constexpr int N = 16 / sizeof(T);
    // ids before the first 16-byte boundary, pieces of 16 bytes, the rest
    const int head = min(a.vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
    const int pieces = (a.vocab - head) / N, per = (pieces + ranks - 1) / ranks;
    const int p0 = min(rank * per, pieces), p1 = min(p0 + per, pieces);
    float top = -INFINITY;
    double sum = 0.0;
    int best = INT_MAX;
    auto take = [&](const float* v, int n, int id) {
        float most = v[0];
        for (int i = 1; i < n; i++) most = fmaxf(most, v[i]);
        if (greedy) {
            for (int i = 0; i < n; i++)
                if (v[i] > top) top = v[i], best = id + i;
        } else if (most > top) {
            sum *= vf::weight(top, most, cold);
            top = most;
        }
        for (int i = 0; i < n; i++) sum += vf::weight(v[i], top, cold);
    };
    if (rank == 0 && tid < head) {
        const float v = Dense<T>::get(p[tid]);
        take(&v, 1, tid);
    }
    for (int i = p0 + tid; i < p1; i += VF_THREADS) {
        float v[N];
        unpack16<T>(__ldg(reinterpret_cast<const uint4*>(p + head) + i), v);
        take(v, N, head + i * N);
    }
    if (rank == ranks - 1 && head + pieces * N + tid < a.vocab) {
        const int id = head + pieces * N + tid;
        const float v = Dense<T>::get(p[id]);
        take(&v, 1, id);
    }
    // (top, sum, best) of the warp, the CTA, the cluster
    auto join = [&](float t2, double s2, int b2) {
        const float t = fmaxf(top, t2);
        if (!greedy)
            sum = sum * vf::weight(top, t, cold) + s2 * vf::weight(t2, t, cold);
        else
            sum += s2;
        best = top > t2 ? best : t2 > top ? b2 : min(best, b2);
        top = t;
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float t2 = __shfl_xor_sync(0xffffffffu, top, o);
        const double s2 = __shfl_xor_sync(0xffffffffu, sum, o);
        join(t2, s2, __shfl_xor_sync(0xffffffffu, best, o));
    }
    if (lane == 0) s_top[warp] = top, s_sum[warp] = sum, s_best[warp] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < VF_WARPS; w++) join(s_top[w], s_sum[w], s_best[w]);
        c_top = top, c_sum = sum, c_best = best;
    }
    if (ranks > 1) pg::cluster_sync();
    if (rank == 0 && tid == 0) {
        for (int r = 1; r < ranks; r++) join(vf::peek(&c_top, r), vf::peek(&c_sum, r), vf::peek(&c_best, r));
        a.rows[row] = {sum, top, best};
    }
    if (ranks > 1) pg::cluster_sync();  // the others' shared memory stays until it is read
}

// A cluster to a sequence; its CTAs share the draw's row.
template <class T>
__global__ void __launch_bounds__(VF_THREADS) k_verify_walk(VerifyArgs a) {
    __shared__ double s_mass[VF_NODES], s_limit[VF_NODES], s_total[VF_NODES];
    __shared__ int s_parent[VF_NODES], s_token[VF_NODES], s_gone[VF_NODES];
    __shared__ double s_warp[VF_WARPS], c_sum;
    __shared__ int s_at, s_count, s_gone_n, s_rejected;
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ranks = a.ranks, rank = blockIdx.x % ranks, b = blockIdx.x / ranks;
    int first, last;
    a.rows_of(b, first, last);
    const int n = last - first;
    int* tokens = a.tokens + (long long)b * a.max_nodes;
    int* nodes = a.nodes + (long long)b * a.max_nodes;
    if (rank == 0)
        for (int i = tid; i < a.max_nodes; i += VF_THREADS) tokens[i] = nodes[i] = -1;
    if (n == 0) {  // the whole cluster
        if (rank == 0 && tid == 0) a.counts[b] = 0;
        return;
    }
    const float heat = a.heat(b);
    const bool greedy = !(heat > 0.f);
    const double cold = greedy ? 0.0 : 1.0 / (double)heat;
    const T* logits = (const T*)a.logits;
    // a draft's weight at its parent, and what it is held against
    for (int i = 1 + tid; i < n; i += VF_THREADS) {
        int parent = a.parents ? __ldg(a.parents + first + i) : i - 1;
        const int token = __ldg(a.drafts + first + i);
        double mass = 0.0, total = 1.0, limit = __ldg(a.uniforms + first + i);
        if (parent < 0 || parent >= i) {
            parent = -1;
        } else {
            const VerifyRow r = a.rows[first + parent];
            const bool known = (unsigned)token < (unsigned)a.vocab;
            if (!vf::proper(r.sum))
                mass = NAN;  // nothing is accepted
            else if (greedy)
                mass = token == r.best;
            else if (known)
                mass = vf::weight(Dense<T>::get(logits[(first + parent) * a.logits_row + token]), r.top, cold);
            if (!greedy) total = r.sum;
            if (a.probs) limit = known ? limit * (double)a.probs[(first + i) * a.probs_row + token] * total : NAN;
        }
        s_parent[i] = parent, s_token[i] = token;
        s_mass[i] = mass, s_limit[i] = limit, s_total[i] = total;
    }
    __syncthreads();
    if (tid == 0) {
        int at = 0, count = 1, gone_n = 0, rejected = -1;
        double gone = 0.0;
        if (rank == 0) nodes[0] = 0;
        for (int i = 1; i < n; i++) {
            if (s_parent[i] != at) continue;
            double mass = s_mass[i];
            for (int k = 0; k < gone_n; k++)
                if (s_gone[k] == s_token[i]) mass = 0.0;  // as a sibling that was rejected
            if ((a.probs ? s_limit[i] : s_limit[i] * (s_total[i] - gone)) < mass) {
                if (rank == 0) nodes[count] = i, tokens[count - 1] = s_token[i];
                at = i, count++;
                gone = 0.0, gone_n = 0, rejected = -1;
            } else {
                gone += mass;
                s_gone[gone_n++] = s_token[i];
                rejected = i;
            }
        }
        s_at = at, s_count = count, s_gone_n = gone_n, s_rejected = rejected;
    }
    __syncthreads();
    const int count = s_count, gone_n = a.probs ? 0 : s_gone_n;
    const VerifyRow r = a.rows[first + s_at];
    if (greedy || !vf::proper(r.sum)) {  // the whole cluster
        if (rank == 0 && tid == 0) {
            tokens[count - 1] = vf::proper(r.sum) ? r.best : -1;
            a.counts[b] = count;
        }
        return;
    }
    const T* p = logits + (first + s_at) * a.logits_row;
    const float* q = a.probs && s_rejected >= 0 ? a.probs + (first + s_rejected) * a.probs_row : nullptr;
    unsigned long long filter = 0;  // ids that may be among the rejected ones, by their low bits
    for (int k = 0; k < gone_n; k++) filter |= 1ull << (s_gone[k] & 63);
    bool all = false;  // no rejection counts
    auto mass = [&](int id) {
        const double e = vf::weight(Dense<T>::get(p[id]), r.top, cold);
        if (all) return e;
        if (q) return fmax(e / r.sum - (double)q[id], 0.0);
        if ((filter >> (id & 63)) & 1)
            for (int k = 0; k < gone_n; k++)
                if (s_gone[k] == id) return 0.0;
        return e;
    };
    // parts of the row, in order: a CTA's, a warp's
    const int share = ((a.vocab + ranks - 1) / ranks + VF_THREADS - 1) / VF_THREADS * VF_THREADS, each = share / VF_WARPS;
    const int w0 = min(a.vocab, rank * share + warp * each), w1 = min(a.vocab, w0 + each);
    double total;
    for (int turn = 0;; turn++) {
        double sum = 0.0;
        for (int id = w0 + lane; id < w1; id += 32) sum += mass(id);
        sum = vf::warp_sum(sum);
        if (lane == 0) s_warp[warp] = sum;
        __syncthreads();
        if (tid == 0) {
            sum = 0.0;
            for (int w = 0; w < VF_WARPS; w++) sum += s_warp[w];
            c_sum = sum;
        }
        pg::cluster_sync();
        total = 0.0;
        for (int k = 0; k < ranks; k++) total += vf::peek(&c_sum, k);
        if (total > 0.0 || turn) break;
        all = true;  // nothing is left: rounding alone leaves the draft's row there
        pg::cluster_sync();
    }
    const double target = __ldg(a.uniforms + first) * total;
    // the first part whose running sum passes the target, else the last that has any
    auto part_of = [&](auto part, int parts, double& passed) {
        double run = passed;
        int pick = 0;
        for (int k = 0; k < parts; k++) {
            const double v = part(k);
            if (!(v > 0.0)) continue;
            pick = k, passed = run;
            run += v;
            if (run > target) break;
        }
        return pick;
    };
    double passed = 0.0;
    const int cta = part_of([&](int k) { return vf::peek(&c_sum, k); }, ranks, passed);
    if (cta == rank) {
        const int w = part_of([&](int k) { return s_warp[k]; }, VF_WARPS, passed);
        if (w == warp) {
            // a lane's ids are neighbours: sums over the lanes, then through the lane's own
            const int run = (w1 - w0 + 31) / 32, l0 = min(w1, w0 + lane * run), l1 = min(w1, l0 + run);
            double sum = 0.0;
            int some = -1;  // the lane's last id that has any
            for (int id = l0; id < l1; id++) {
                const double v = mass(id);
                sum += v;
                if (v > 0.0) some = id;
            }
            double up = sum;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double v = __shfl_up_sync(0xffffffffu, up, o);
                if (lane >= o) up += v;
            }
            const uint32_t over = __ballot_sync(0xffffffffu, some >= 0 && passed + up > target);
            const uint32_t any = __ballot_sync(0xffffffffu, some >= 0);
            const int chosen = over ? __ffs(over) - 1 : any ? 31 - __clz(any) : -1;
            if (lane == chosen) {
                int token = some;
                if (over) {
                    double at = passed + up - sum;
                    for (int id = l0; id < l1; id++) {
                        const double v = mass(id);
                        if (!(v > 0.0)) continue;
                        at += v;
                        if (at > target) {
                            token = id;
                            break;
                        }
                    }
                }
                tokens[count - 1] = token;
            }
        }
    }
    if (rank == 0 && tid == 0) a.counts[b] = count;
    pg::cluster_sync();  // the others' sums stay until they are read
}

}  // namespace fb2
