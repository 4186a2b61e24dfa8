// verify.cuh — drafted tokens against the target's probabilities, and the token
// that follows the accepted ones (include/forge_b200.h, fb2_verify_drafts, has
// the rules).
//
// Two kernels.  k_verify_rows reads every row of logits once, some CTAs to a row:
// the largest and the sum of exp((l - largest) / T) of their parts, and where the
// largest is for T <= 0.  k_verify_walk takes a sequence: the drafts' probabilities
// are looked up at once and walked down by one warp; then the row at which the walk ended is weighed
// (without rejected tokens, or less the draft's probabilities), its sums over
// parts in the order of ids say in which part the draw falls, and that part is
// looked through.
//
// Which id a draw gives hangs on running sums over a whole row: in 32 bits they
// are off by some 1e-6 of the total, wider than most tokens of a large vocabulary,
// so the weights of the draw's row and their sums are in 64 bits.  Whether a draft is
// accepted hangs on one comparison, which a sum from 32-bit exponentials decides
// but for one uniform in some 2^16; where it does not, that row is summed in 64 bits
// first.  So every decision is that of fp64, and all rows but one of a sequence are
// read at the cost of 32-bit exponentials.
//
// 161 rows x 131071, bf16, of 32 sequences with draft probabilities: 47 us, 16 of them for
// the rows (2.6 TB/s; 10 instructions a logit and the waits between them), the rest for the draws: two
// passes of some 35 instructions a logit where a draft was rejected (fp64 arithmetic
// itself goes at 64 lanes a cycle and is a quarter of them).  Exponentials of CUDA's exp()
// in fp64 for all rows: 184.  289 rows x 50257, fp16, 8 trees: 22 us (89); 5 rows x 16384: 12
// (25), a chain of two launches, eight dependent loads and four cluster barriers.
#pragma once
#include "kvq.cuh"
#include "pages.cuh"

namespace fb2 {

constexpr int VF_THREADS = 256, VF_WARPS = VF_THREADS / 32, VF_NODES = 1024, VF_RANKS = 8;
constexpr int VW_THREADS = 512, VW_WARPS = VW_THREADS / 32;
constexpr int VW_BATCH = 4;                 // loads of a lane that are in flight at once
constexpr int VW_RUN = 32 * VW_BATCH;       // ids of a warp's batch
constexpr int VW_PARTS = 16;                // of a warp's ids, each with its own sum
constexpr int VW_NODE = 44;                 // bytes of shared memory for a node
// How far a sum of k_verify_rows may be off, relative.  An exponent (l - top) * log2(e) / T
// has three roundings, and the exponents' mean under p is at most log2(vocab) <= 31: 31 *
// 3 * 2^-24 * ln 2; ex2.approx 2^-22; a sum of 8 in fp32, the rest in fp64: 2^-21.
// Together below 2^-17.  Twice that, for the products it enters.
constexpr double VF_OFF = 1.0 / 65536;
constexpr float VF_COLD = 1e-30f;  // a T below is not divided by in 32 bits: all its tests go by 64

struct VerifyRow {
    double sum;  // of exp((l - top) / T), to VF_OFF; not positive and finite where the row has no probabilities
    float top;
    int best;  // the lowest id of the largest logit (T <= 0; -1: none)
};
struct VerifyArgs {
    const void* logits;
    const float* probs;
    const int *drafts, *starts, *parents;
    const double* uniforms;
    const float* temperature;
    int *tokens, *nodes, *counts;
    VerifyRow* rows;  // [n_rows][parts]: of a part of a row each
    long long logits_row, probs_row;
    int n_seqs, n_rows, vocab, max_nodes;
    int parts, ranks;  // CTAs of a row, and of a sequence's cluster: at most VF_RANKS
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
FB2_DEV double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
FB2_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
FB2_DEV float2 add2(float2 a, float2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return reinterpret_cast<float2&>(r);
}
FB2_DEV float2 mul2(float2 a, float2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return reinterpret_cast<float2&>(r);
}
// 2^(i / 1024), i = 0..1023: what the exponentials in 64 bits are looked up in;
// products of two factors, so that a thread calls exp2 once or not at all.
FB2_DEV void fill_powers(double* powers, double* factors) {
    const int i = threadIdx.x;
    if (i < 64) factors[i] = exp2(i < 32 ? (double)i / 1024 : (double)(i - 32) / 32);
    __syncthreads();
    for (int k = i; k < 1024; k += blockDim.x) powers[k] = factors[k & 31] * factors[32 + (k >> 5)];
}
// fp32 as fp64, without a conversion (which go at the rate of fp64 arithmetic): 0 and
// what is smaller than 2^-126 become some 2^-127, infinities 2^128.
FB2_DEV double widen(float v) {
    const int bits = __float_as_int(v);
    return __hiloint2double(((bits >> 3) & 0x8fffffff) + 0x38000000, bits << 29);
}
// exp((l - top) / T), l <= top, by a table and a polynomial (P. T. P. Tang,
// Table-driven implementation of the exponential function, ACM TOMS 15, 1989):
// 2^(n / 1024) from the table and the exponent, exp(t), |t| <= ln 2 / 2048, from its
// series to t^3 (t^4 / 24 < 2^-50).  0 where it falls below 2^-1000: the first logit that does
// not is found in 64 bits and rounded up (a limit rounded to nearest lets in logits whose
// exponent is far below where T is less than the step between logits).
struct Heat {
    double cold;  // 1024 log2(e) / T, of logits as `weight` takes them
    double top;
    float cut;   // below: 0
    bool small;  // logits are taken 2^100 times as large
    FB2_DEV void at(float t, float heat) {
        // T below 2^-70 and a top as small as what `widen` is off by may be next to it: logits go
        // up, those that overflow are far below.  (Below a larger top every other logit is.)
        small = heat < 0x1p-70f && fabsf(t) < 0x1p-20f;
        const double by = small ? heat * 0x1p100 : (double)heat;
        cold = 1024 * 1.4426950408889634074 / by;
        t = scaled(t);
        top = widen(t);
        cut = fmaxf(__double2float_ru((double)t - 1000 * 0.69314718055994530942 * by), -3.402823466e38f);  // (-inf is below)
    }
    FB2_DEV float scaled(float l) const { return small ? l * 0x1p100f : l; }
    // l: scaled; BITS: of a logit's type; 16-bit ones leave the low half of a double 0
    template <int BITS>
    FB2_DEV double weight(float l, const double* powers) const {
        const bool none = l < cut;
        const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the nearest whole number
        const double wide = widen(l), d = (BITS == 32 ? wide : __hiloint2double(__double2hiint(wide), 0)) - top, high = fma(d, cold, magic), t = fma(d, cold, magic - high);
        const int n = __double2loint(high);
        constexpr double u = 6.7690154351557159e-4;  // ln 2 / 1024
        double e = fma(t, u * u * u / 6, u * u / 2);
        e = fma(e, t, u);
        double p = powers[n & 1023];
        p = __hiloint2double(__double2hiint(p) + ((n >> 10) << 20), __double2loint(p));
        e = fma(e * t, p, p);
        return none ? 0.0 : e;  // (no branch: weights of neighbours overlap)
    }
};
// v where it is positive, else 0
FB2_DEV double positive(double v) { return __double2hiint(v) < 0 ? 0.0 : v; }
// The first k in 0..n-1 whose running sum over `part`, from `passed` on, passes the
// target, else the last with a positive part (-1: none); `passed` becomes the sum
// before it.  By the lanes of a warp.
template <class F>
FB2_DEV int pick(F part, int n, double target, double& passed) {
    const int lane = threadIdx.x & 31, per = (n + 31) / 32, k0 = min(lane * per, n), k1 = min(k0 + per, n);
    double sum = 0.0;
    for (int k = k0; k < k1; k++) sum += fmax(part(k), 0.0);
    double up = sum;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const double v = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += v;
    }
    const uint32_t over = __ballot_sync(0xffffffffu, sum > 0.0 && passed + up > target), any = __ballot_sync(0xffffffffu, sum > 0.0);
    if (!any) return -1;
    const int chosen = over ? __ffs(over) - 1 : 31 - __clz(any);
    int at = -1;
    double before = passed + (up - sum), run = before;
    if (lane == chosen)
        for (int k = k0; k < k1; k++) {
            const double v = part(k);
            if (!(v > 0.0)) continue;
            at = k, before = run;
            run += v;
            if (run > target) break;
        }
    passed = __shfl_sync(0xffffffffu, before, chosen);
    return __shfl_sync(0xffffffffu, at, chosen);
}
// log2(e) / T, T > 0; not 0 for T = inf, as -inf times it has to be -inf
FB2_DEV float near_of(float heat) { return fmaxf(1.44269504088896341f / fmaxf(heat, VF_COLD), 1e-44f); }
// The whole row's of its parts, which VF_RANKS neighbouring lanes have one each of
FB2_DEV VerifyRow joined(VerifyRow r, float near) {
#pragma unroll
    for (int o = 1; o < VF_RANKS; o *= 2) {
        const VerifyRow s{__shfl_xor_sync(0xffffffffu, r.sum, o), __shfl_xor_sync(0xffffffffu, r.top, o), __shfl_xor_sync(0xffffffffu, r.best, o)};
        if (s.best >= 0 && (r.best < 0 || s.top > r.top || (s.top == r.top && s.best < r.best))) r.best = s.best;
        const float top = fmaxf(r.top, s.top);
        r.sum = r.sum * (double)ex2((r.top - top) * near) + s.sum * (double)ex2((s.top - top) * near);
        r.top = top;
    }
    return r;
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

// a.parts CTAs to a row.
template <class T>
__global__ void __launch_bounds__(VF_THREADS) k_verify_rows(VerifyArgs a) {
    __shared__ double s_sum[VF_WARPS];
    __shared__ float s_top[VF_WARPS];
    __shared__ int s_best[VF_WARPS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the walk's launch; it waits for this grid's end
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int part = blockIdx.x % a.parts, row = blockIdx.x / a.parts;
    const int b = a.starts ? vf::owner(a.starts, a.n_seqs, row) : row;
    int first, last;
    a.rows_of(b, first, last);
    if (row < first || row >= last) {
        if (tid == 0) a.rows[blockIdx.x] = {0.0, -INFINITY, -1};
        return;
    }
    const float heat = a.heat(b);
    const bool greedy = !(heat > 0.f);
    const float cold = vf::near_of(greedy ? 1.f : heat);
    const T* p = (const T*)a.logits + row * a.logits_row;
    constexpr int N = 16 / sizeof(T);
    // ids before the first 16-byte boundary, pieces of 16 bytes, the rest
    const int head = min(a.vocab, (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
    const int pieces = (a.vocab - head) / N, per = (pieces + a.parts - 1) / a.parts;
    const int p0 = min(part * per, pieces), p1 = min(p0 + per, pieces);
    // The terms are relative to `base`, which follows the largest logit when that is 2^8
    // of a term away: a sum that was rescaled weighs a 256th, and its roundings with it.
    float top = -3.402823466e38f, base = top;  // (finite: -inf less this is -inf)
    double sum = 0.0;
    int best = -1;
    auto raise = [&](float most) {
        top = fmaxf(top, most);
        if ((most - base) * cold > 8.f) {
            sum *= (double)vf::ex2((base - most) * cold);
            base = most;
        }
    };
    // sum of exp2((v - base) * cold) of a piece (NaN for NaN, and for all where one is inf), two values to an instruction
    auto terms = [&](const float (&v)[N]) {
        const float2 up = make_float2(-base, -base), by = make_float2(cold, cold);
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const float2 x = vf::mul2(vf::add2(make_float2(v[j], v[j + 1]), up), by);
            s = vf::add2(s, make_float2(vf::ex2(x.x), vf::ex2(x.y)));
        }
        return s.x + s.y;
    };
    const uint4* body = reinterpret_cast<const uint4*>(p + head);
    constexpr int M = 2;  // loads in flight (4: 2 us more for 289 rows x 50257, fp16)
    for (int i0 = p0 + tid; i0 < p1; i0 += M * VF_THREADS) {
        uint4 w[M];
#pragma unroll
        for (int m = 0; m < M; m++) w[m] = i0 + m * VF_THREADS < p1 ? __ldg(body + i0 + m * VF_THREADS) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < M; m++) {
            const int i = i0 + m * VF_THREADS;
            if (i >= p1) break;
            float v[N];
            unpack16<T>(w[m], v);
            float most = v[0];
#pragma unroll
            for (int j = 1; j < N; j++) most = fmaxf(most, v[j]);
            if (greedy && (most > top || (most == top && best < 0)))
#pragma unroll
                for (int j = N - 1; j >= 0; j--)
                    if (v[j] == most) best = head + i * N + j;
            raise(most);
            sum += (double)terms(v);
        }
    }
    auto edge = [&](int id) {
        const float v = Dense<T>::get(p[id]);
        if (v > top || (v == top && (best < 0 || id < best))) best = id;
        raise(v);
        sum += (double)vf::ex2((v - base) * cold);
    };
    if (part == 0 && tid < head) edge(tid);
    if (part == a.parts - 1 && head + pieces * N + tid < a.vocab) edge(head + pieces * N + tid);
    // in every lane the lanes' largest, the sum below it, the first id that has it
    auto join = [&]() {
        const float most = warp_max(top);
        if (greedy) best = (int)__reduce_min_sync(0xffffffffu, top == most ? (uint32_t)best : 0xffffffffu);  // -1: none
        sum = vf::warp_sum(sum * (double)vf::ex2((base - most) * cold));
        top = base = most;
    };
    join();
    if (lane == 0) s_top[warp] = top, s_sum[warp] = sum, s_best[warp] = best;
    __syncthreads();
    if (warp == 0) {
        const bool one = lane < VF_WARPS;
        top = base = one ? s_top[lane] : -3.402823466e38f, sum = one ? s_sum[lane] : 0.0, best = one ? s_best[lane] : -1;
        join();
        if (lane == 0) a.rows[blockIdx.x] = {sum, top, best};
    }
}

// A cluster to a sequence; its CTAs share the draw's row.
template <class T>
__global__ void __launch_bounds__(VW_THREADS, 2) k_verify_walk(VerifyArgs a) {
    // of the nodes: their rows' sums; the drafts' weights at their parents, what they are held
    // against, their parents, their tokens; the tokens of rejected ones
    extern __shared__ __align__(16) unsigned char vw_smem[];
    VerifyRow* s_row = reinterpret_cast<VerifyRow*>(vw_smem);
    double *s_mass = reinterpret_cast<double*>(s_row + a.max_nodes), *s_limit = s_mass + a.max_nodes;
    int *s_parent = reinterpret_cast<int*>(s_limit + a.max_nodes), *s_token = s_parent + a.max_nodes, *s_gone = s_token + a.max_nodes;
    __shared__ double s_powers[1024], s_factors[64], s_part[VW_WARPS * VW_PARTS], s_warp[VW_WARPS], c_sum[2];
    __shared__ double s_lost;
    __shared__ unsigned char s_hit[VW_WARPS * VW_PARTS];  // parts that have a rejected token
    __shared__ int s_at, s_count, s_gone_n, s_rejected, s_next, s_ask;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ranks = a.ranks, rank = blockIdx.x % ranks, b = blockIdx.x / ranks;
    vf::fill_powers(s_powers, s_factors);
    int first, last;
    a.rows_of(b, first, last);
    const int n = last - first;
    int* tokens = a.tokens + (long long)b * a.max_nodes;
    int* nodes = a.nodes + (long long)b * a.max_nodes;
    const float heat = a.heat(b);
    const bool greedy = !(heat > 0.f);
    vf::Heat at_heat;
    const float near = vf::near_of(greedy ? 1.f : heat);
    const T* logits = (const T*)a.logits;
    pdl_wait();  // the rows' sums, and the outputs' memory
    if (rank == 0)
        for (int i = tid; i < a.max_nodes; i += VW_THREADS) tokens[i] = nodes[i] = -1;
    if (n == 0) {  // the whole cluster
        if (rank == 0 && tid == 0) a.counts[b] = 0;
        return;
    }
    for (int i0 = 0; i0 < n; i0 += VW_THREADS / VF_RANKS) {
        const int i = i0 + tid / VF_RANKS, k = tid % VF_RANKS;
        VerifyRow r{0.0, -3.402823466e38f, -1};
        if (i < n && k < a.parts) r = a.rows[(long long)(first + i) * a.parts + k];
        r = vf::joined(r, near);
        if (i < n && k == 0) s_row[i] = r;
    }
    __syncthreads();  // they and the table
    // a draft's weight at its parent, and what it is held against
    for (int i = 1 + tid; i < n; i += VW_THREADS) {
        int parent = a.parents ? __ldg(a.parents + first + i) : i - 1;
        const int token = __ldg(a.drafts + first + i);
        double mass = 0.0, limit = __ldg(a.uniforms + first + i);
        if (parent < 0 || parent >= i) {
            parent = -1;
        } else {
            const bool known = (unsigned)token < (unsigned)a.vocab;
            const float l = known ? Dense<T>::get(logits[(first + parent) * a.logits_row + token]) : -INFINITY;
            const double q = a.probs && known ? (double)a.probs[(first + i) * a.probs_row + token] : NAN;
            const VerifyRow r = s_row[parent];
            if (!vf::proper(r.sum))
                mass = NAN;  // nothing is accepted
            else if (greedy)
                mass = token == r.best;
            else {
                vf::Heat h;
                h.at(r.top, heat);
                mass = h.template weight<8 * sizeof(T)>(h.scaled(l), s_powers);
            }
            if (a.probs) limit *= q;
        }
        s_parent[i] = parent, s_token[i] = token;
        s_mass[i] = mass, s_limit[i] = limit;
    }
    if (tid == 0) s_at = 0, s_count = 1, s_gone_n = 0, s_rejected = -1, s_next = 1, s_lost = 0.0;
    if (tid == 0 && rank == 0) nodes[0] = 0;
    for (int i = tid; i < VW_WARPS * VW_PARTS; i += VW_THREADS) s_part[i] = 0.0, s_hit[i] = 0;  // parts behind the row's end stay so
    __syncthreads();

    // ---- sums over a row, in parts in the order of ids: a CTA's, a warp's, a batch's
    const int share = ((a.vocab + ranks - 1) / ranks + VW_THREADS - 1) / VW_THREADS * VW_THREADS, each = share / VW_WARPS;
    const int w0 = min(a.vocab, rank * share + warp * each), w1 = min(a.vocab, w0 + each);
    const int run = ((each + VW_PARTS - 1) / VW_PARTS + VW_RUN - 1) / VW_RUN * VW_RUN;  // ids of a part
    const T* p = nullptr;
    const float* q = nullptr;  // the rejected draft's probabilities
    double scale = 1.0;                  // with q: 1 / the row's sum
    const double* sums = nullptr;        // of the CTAs
    int gone_n = 0;                      // rejected tokens that count as nothing
    // weights of VW_BATCH ids from `id` on, STEP apart, up to `end`
    auto batch = [&](int id, int end, double (&m)[VW_BATCH], auto step, bool hit) {
        constexpr int N = VW_BATCH, STEP = decltype(step)::value;
        float l[N], qv[N];
#pragma unroll
        for (int j = 0; j < N; j++) l[j] = id + STEP * j < end ? Dense<T>::get(p[id + STEP * j]) : -INFINITY;
        if (q) {
#pragma unroll
            for (int j = 0; j < N; j++) qv[j] = id + STEP * j < end ? __ldg(q + id + STEP * j) : 0.f;
        }
        if (at_heat.small) {
#pragma unroll
            for (int j = 0; j < N; j++) l[j] = at_heat.scaled(l[j]);
        }
#pragma unroll
        for (int j = 0; j < N; j++) m[j] = at_heat.template weight<8 * sizeof(T)>(l[j], s_powers);
        if (q) {
#pragma unroll
            for (int j = 0; j < N; j++) m[j] = vf::positive(fma(m[j], scale, -vf::widen(qv[j])));
        }
        if (hit)
            for (int k = 0; k < gone_n; k++)
#pragma unroll
                for (int j = 0; j < N; j++)
                    if (s_gone[k] == id + STEP * j) m[j] = 0.0;
    };

    // ---- the walk by one warp, until it ends or a test needs its row's sum in 64 bits;
    // that sum; the draw's.  One loop, so that the sums' code is there (and fetched) once.
    enum { WALK, DRAW, DRAW_ALL } state = WALK;
    int known = -1;  // the node whose sum is known
    double exact = 0.0, total = 0.0;
    for (int turn = 0;; turn++) {
        if (state == WALK) {
            if (warp == 0) {
                int at = s_at, count = s_count, gn = s_gone_n, rejected = s_rejected, ask = -1;
                double gone = s_lost;  // the rejected siblings' weight
                for (int i = s_next;;) {
                    // the node's next child
                    uint32_t kids = 0;
                    int i0 = i;
                    for (; i0 < n; i0 += 32) {
                        kids = __ballot_sync(0xffffffffu, i0 + lane < n && s_parent[i0 + lane] == at);
                        if (kids) break;
                    }
                    if (!kids) {
                        s_next = n;
                        break;
                    }
                    i = i0 + __ffs(kids) - 1;
                    const int token = s_token[i];
                    double mass = s_mass[i];
                    bool again = false;  // a sibling with this token was rejected
                    for (int k = lane; k < gn; k += 32) again |= s_gone[k] == token;
                    again = __any_sync(0xffffffffu, again);
                    if (again) mass = 0.0;
                    const double sum = greedy ? 1.0 : known == at ? exact : s_row[at].sum, weighed = a.probs ? sum : sum - gone;
                    const double held = s_limit[i] * weighed;
                    if (!greedy && known != at && mass > 0.0 && (fabs(held - mass) <= VF_OFF * fabs(s_limit[i]) * sum || heat < VF_COLD)) {
                        ask = at;
                        s_next = i;
                        break;
                    }
                    if (held < mass) {
                        if (rank == 0 && lane == 0) nodes[count] = i, tokens[count - 1] = token;
                        at = i, count++;
                        gone = 0.0, gn = 0, rejected = -1;
                    } else {
                        if (!again) {
                            gone += mass;
                            if (lane == 0) s_gone[gn] = token;
                            gn++;
                        }
                        rejected = i;
                    }
                    __syncwarp();
                    i++;
                }
                if (lane == 0) s_at = at, s_count = count, s_gone_n = gn, s_rejected = rejected, s_lost = gone, s_ask = ask;
            }
            __syncthreads();
        }
        // (here, behind the barrier: warp 0 writes them again in its next turn)
        const int node = s_at, rejected = s_rejected, ask = s_ask;
        const VerifyRow r = s_row[node];
        p = logits + (first + node) * a.logits_row;
        at_heat.at(r.top, heat);
        if (state == WALK && ask < 0) {
            if (greedy || !vf::proper(r.sum)) {  // the whole cluster
                if (rank == 0 && tid == 0) {
                    tokens[s_count - 1] = vf::proper(r.sum) ? r.best : -1;
                    a.counts[b] = s_count;
                }
                if (turn) pg::cluster_sync();  // this CTA's sums have been read
                return;
            }
            if (!a.probs || rejected < 0 || known == node) state = DRAW;
        }
        if (state == DRAW) {
            if (a.probs) {
                if (rejected >= 0) q = a.probs + (first + rejected) * a.probs_row, scale = 1.0 / exact;
            } else {
                gone_n = s_gone_n;
                for (int k = tid; k < gone_n; k += VW_THREADS) {
                    const int at = s_gone[k] - rank * share;
                    if (at >= 0 && at < share) s_hit[at / each * VW_PARTS + at % each / run] = 1;
                }
                __syncthreads();
            }
        }
        // the row's sums
        double all = 0.0;
        for (int k = 0, p0 = w0; k < VW_PARTS && p0 < w1; k++, p0 += run) {
            double sum = 0.0;
            const int p1 = min(w1, p0 + run);
            const bool hit = gone_n && s_hit[warp * VW_PARTS + k];
            for (int id = p0; id < p1; id += VW_RUN) {
                double m[VW_BATCH];
                batch(id + lane, p1, m, std::integral_constant<int, 32>{}, hit);
#pragma unroll
                for (int j = 0; j < VW_BATCH; j++) sum += m[j];
            }
            sum = vf::warp_sum(sum);
            if (lane == 0) s_part[warp * VW_PARTS + k] = sum;
            all += sum;
        }
        if (lane == 0) s_warp[warp] = all;
        __syncthreads();
        sums = &c_sum[turn & 1];  // the other one may still be read
        if (warp == 0) {
            const double s = vf::warp_sum(lane < VW_WARPS ? s_warp[lane] : 0.0);
            if (lane == 0) c_sum[turn & 1] = s;
        }
        pg::cluster_sync();
        total = vf::warp_sum(lane < ranks ? vf::peek(sums, lane) : 0.0);
        if (state == WALK) {
            exact = total, known = node;
            if (ask < 0) state = DRAW;
        } else if (total > 0.0 || state == DRAW_ALL) {
            break;
        } else {  // nothing is left: the row as if nothing had been rejected
            q = nullptr, gone_n = 0;
            state = DRAW_ALL;
        }
    }
    const int count = s_count;
    const double target = __ldg(a.uniforms + first) * total;
    if (warp == 0) {
        double passed = 0.0;
        const double mine = lane < ranks ? vf::peek(sums, lane) : 0.0;
        const int cta = vf::pick([&](int) { return mine; }, ranks, target, passed);  // lane k has CTA k's
        if (cta == rank) {
            const int part = vf::pick([&](int k) { return s_part[k]; }, VW_WARPS * VW_PARTS, target, passed);
            // through the part's ids, of which a lane has neighbours
            const int c0 = rank * share + part / VW_PARTS * each;
            const int p0 = c0 + part % VW_PARTS * run, p1 = min(min(a.vocab, c0 + each), p0 + run);
            int token = -1;
#pragma unroll 1
            for (int id = p0 + lane * VW_BATCH; id - lane * VW_BATCH < p1; id += VW_RUN) {
                double m[VW_BATCH], sum = 0.0;
                batch(id, p1, m, std::integral_constant<int, 1>{}, gone_n && s_hit[part]);
#pragma unroll
                for (int j = 0; j < VW_BATCH; j++) sum += m[j];
                double up = sum;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const double v = __shfl_up_sync(0xffffffffu, up, o);
                    if (lane >= o) up += v;
                }
                const uint32_t any = __ballot_sync(0xffffffffu, sum > 0.0), over = __ballot_sync(0xffffffffu, passed + up > target) & any;
                // the first of the lane's ids that passes the target, or its last with a weight
                int found = -1;
                double at = passed + (up - sum);
#pragma unroll
                for (int j = 0; j < VW_BATCH; j++)
                    if (m[j] > 0.0 && (found < 0 || !(at > target))) found = id + j, at += m[j];
                if (any) token = __shfl_sync(0xffffffffu, found, over ? __ffs(over) - 1 : 31 - __clz(any));
                if (over) break;
                passed += __shfl_sync(0xffffffffu, up, 31);
            }
            if (lane == 0) {
                tokens[count - 1] = token;
                a.counts[b] = count;
            }
        }
    }
    pg::cluster_sync();  // the others' sums stay until they are read
}

}  // namespace fb2
