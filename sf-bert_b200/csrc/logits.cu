// Operators on rows of logits: log probabilities of given tokens with entropy and top alternatives, distillation from a
// teacher's top tokens, and their gradients.
//
// With m = max_j x_j, S = sum_j exp(s (x_j - m)), l = ln S and p_j = exp(s (x_j - m) - l):
//   log probability    s (x_t - m) - l
//   entropy            l - sum_j p_j s (x_j - m)
//   distillation       sum_k q_k (ln q_k - ln p_k) over the teacher's list, with or without one more class for what it leaves
//   gradients          s g (d_jt - p_j) - s h p_j (ln p_j + H)      and      s w (Q p_j - q_j)
// All of it is bound by the one pass over the logits (and the one over their gradient); the kernels are built so that
// each element is read once, whole windows of 16 bytes at a time, several on their way per thread.
#include "logits.cuh"
#include <cooperative_groups.h>
#include <cfloat>

namespace cg = cooperative_groups;

namespace sfb {
// A counter is cleared by a kernel and not by a memset, which nothing overlaps: the launch behind it sets itself up meanwhile.
__global__ void zero_kernel(uint32_t *counter)
{
    grid_dependency_wait();
    grid_launch_dependents();
    *counter = 0;
}
static int set_zero(const char *who, uint32_t *counter, cudaStream_t s)
{
    if (counter) launch_overlapped(zero_kernel, dim3(1), dim3(1), 0, s, counter);
    return check_launch(who);
}

namespace lg {

constexpr uint32_t kThreads = 256;
constexpr int kU = 4;                     // windows that a thread has on their way at a time
constexpr int kG = 4;                     // the same for gradients
constexpr uint32_t kCap = 1024;           // candidates for a row's alternatives
constexpr uint32_t kMaxList = 128;        // alternatives, entries of a teacher's list (four per lane)
constexpr uint32_t kMaxCluster = 8;
// A remainder whose logarithm is below this is summed again for the gradient (sum_unlisted): an unlisted token's share of it is the power of a
// difference from that logarithm, of which fp32 loses 2^-24 of its size -- 2^-17 of the share here, all of it at ten million.
constexpr float kFarRest = -64.f;
constexpr uint32_t kShort = 1024;         // windows of a row that a warp takes by itself where there are many

struct StatParams {
    const void *x;
    uint64_t pitch;                       // elements from row to row
    uint32_t rows, vocab;
    float scale, s2;                      // s2 = scale * log2(e)
    const int32_t *targets;
    float *logp, *stats, *entropy, *top_logp;
    int32_t *top_ids;
    uint32_t k;                           // alternatives, or entries of the lists
    const int32_t *ids;                   // the lists [rows][k]
    const float *teacher;
    float *loss;
    uint32_t *missed;
    uint32_t count_here;                  // targets (entries) counted by one CTA behind the rows'; 0: each row adds its own
};

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}

// bits in the order of the values (-0 is 0)
__device__ __forceinline__ uint32_t ordered(float v)
{
    const uint32_t u = __float_as_uint(v + 0.f);
    return u ^ (uint32_t)((int32_t)u >> 31 | (int32_t)0x80000000);
}
__device__ __forceinline__ float from_ordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }
// larger for larger values, and among equal ones for the lower index
__device__ __forceinline__ unsigned long long rank_key(float v, uint32_t index) { return (unsigned long long)ordered(v) << 32 | (0xffffffffu - index); }

__device__ __forceinline__ float warp_max_nan(float v)
{
    float y;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(v));
    return y;
}

// the sums of a warp's threads, beside the largest of their maxima
template <bool ENT> __device__ __forceinline__ void warp_sums(Sums &a, float &mx, float s2)
{
    mx = warp_max_nan(mx);
    a.move_to(mx, s2);
    a.s = warp_sum(a.s);
    if (ENT) a.e = warp_sum(a.e);
}

// N windows into the sums
template <int DT, bool ENT, int N> __device__ __forceinline__ void add_windows(Sums &a, const uint4 (&v)[N], float s2)
{
    const Pair minus_r = pair(-a.r, -a.r), factor = pair(s2, s2);
    Pair s = pair(a.s, 0.f), e = pair(a.e, 0.f);
#pragma unroll
    for (int u = 0; u < N; u++) {
        float x[Win<DT>::kElems];
        unpack<DT>(v[u], x);
#pragma unroll
        for (uint32_t j = 0; j < Win<DT>::kElems; j += 2) {
            const Pair t = mul2(factor, add2(pair(x[j], x[j + 1]), minus_r));
            float t0, t1;
            halves(t, t0, t1);
            const Pair y = pair(ex2(t0), ex2(t1));
            s = add2(s, y);
            if (ENT) e = fma2(y, pair(fmaxf(t0, kFar), fmaxf(t1, kFar)), e);
        }
    }
    float s0, s1;
    halves(s, s0, s1);
    a.s = s0 + s1;
    if (ENT) {
        halves(e, s0, s1);
        a.e = s0 + s1;
    }
}

// listed tokens of a window (bit j: element j) become -inf
template <int DT> __device__ __forceinline__ void drop_listed(uint4 &v, uint32_t bits)
{
    uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (DT == SFB_F32) {
            if (bits >> j & 1) u[j] = Win<DT>::kInf;
        } else {
            if (bits >> (2 * j) & 1) u[j] = (u[j] & 0xffff0000u) | Win<DT>::kInf;
            if (bits >> (2 * j + 1) & 1) u[j] = (u[j] & 0xffffu) | Win<DT>::kInf << 16;
        }
    }
    v = make_uint4(u[0], u[1], u[2], u[3]);
}

struct Part { float m, s, e; };

// ids outside [0, vocab), counted by one CTA
__device__ __forceinline__ void count_missed(const int32_t *ids, uint32_t n, uint32_t vocab, uint32_t *missed, uint32_t *part)
{
    uint32_t bad = 0;
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x * 8) {
        int32_t v[8];
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = i + u * blockDim.x < n ? ids[i + u * blockDim.x] : 0;
#pragma unroll
        for (int u = 0; u < 8; u++) bad += (uint32_t)v[u] >= vocab;
    }
    bad = __reduce_add_sync(0xffffffffu, bad);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = bad;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < blockDim.x / 32; w++) bad += part[w];
        *missed = bad;
    }
}

struct TopShared {
    uint32_t gm[kThreads];                // largest values of the groups of threads: 24 bits in their order, then 255 - group
    unsigned long long cand[kCap];        // candidates (in CTA 0)
    uint32_t hits[kCap];
    float best[kMaxList];
    uint32_t cnt, n_hits, tau, part[8];
    float m, l;
};

// sum over the CTA's threads
__device__ __forceinline__ uint32_t block_sum(uint32_t v, uint32_t *part)
{
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (uint32_t w = 0; w < blockDim.x / 32; w++) v += part[w];
    return v;
}

// The candidates when too many values reach the bound, by one CTA from the whole row (by now in L2); they are then sh->cnt from the
// first place on.
// Mostly it is one value that many have: a constant row, or one whose banned tokens hold the type's lowest value and too few
// others are left.  Then what is above it is collected, and of the ties the first ones, which are the ones that count: a pass or two.
__device__ __forceinline__ void push_candidate(TopShared *sh, float v, uint32_t index)
{
    const uint32_t at = atomicAdd(&sh->cnt, 1u);
    if (at < kCap) sh->cand[at] = rank_key(v, index);
}
template <int DT> __device__ __noinline__ bool collect_ties(const Row<DT> row, uint32_t k, TopShared *sh)
{
    constexpr uint32_t E = Win<DT>::kElems;
    const uint32_t windows = row.windows(), tau = sh->tau, top = tau | 0xffu;       // the bound is 24 bits of a value
    uint32_t above = 0, least = 0xffffffffu, most = 0;
    for (uint32_t w = threadIdx.x; w < windows; w += blockDim.x) {
        float v[E];
        unpack<DT>(load_window(row, w), v);
#pragma unroll
        for (uint32_t j = 0; j < E; j++) {
            const uint32_t o = ordered(v[j]);
            if (!(v[j] > neg_inf()) || o < tau) continue;
            above += o > top;
            if (o <= top) { least = min(least, o); most = max(most, o); }
        }
    }
    above = block_sum(above, sh->part);
    __syncthreads();
    if (threadIdx.x == 0) { sh->cnt = 0; sh->part[0] = 0xffffffffu; sh->part[1] = 0; }
    __syncthreads();
    atomicMin(&sh->part[0], least);
    atomicMax(&sh->part[1], most);
    __syncthreads();
    least = sh->part[0];
    if (above >= k || least != sh->part[1]) return false;
    for (uint32_t w = threadIdx.x; w < windows && above; w += blockDim.x) {
        float v[E];
        unpack<DT>(load_window(row, w), v);
#pragma unroll
        for (uint32_t j = 0; j < E; j++)
            if (v[j] > neg_inf() && ordered(v[j]) > top) push_candidate(sh, v[j], w * E + j - row.head);
    }
    for (uint32_t w0 = 0; w0 < windows; w0 += 64) {                // at most 64 windows' ties beyond those that are needed
        if (threadIdx.x < 64 && w0 + threadIdx.x < windows) {
            float v[E];
            unpack<DT>(load_window(row, w0 + threadIdx.x), v);
#pragma unroll
            for (uint32_t j = 0; j < E; j++)
                if (v[j] > neg_inf() && ordered(v[j]) == least) push_candidate(sh, v[j], (w0 + threadIdx.x) * E + j - row.head);
        }
        __syncthreads();
        const bool enough = sh->cnt >= k;
        __syncthreads();
        if (enough) break;
    }
    return true;
}
// Otherwise (most of the large values went to a few threads) the bound is bisected over the values and their indices, a pass for each
// step.
template <int DT> __device__ __noinline__ void bisect_candidates(const Row<DT> row, uint32_t k, TopShared *sh)
{
    unsigned long long lo = (unsigned long long)sh->tau << 32, hi = ~0ull, x = lo;      // at least k reach lo (or all there are), fewer than k hi
    const uint32_t windows = row.windows();
    for (;;) {
        const unsigned long long mid = lo + (hi - lo) / 2;
        if (mid == lo) { x = hi; break; }
        uint32_t c = 0;
        for (uint32_t w = threadIdx.x; w < windows; w += blockDim.x) {
            float v[Win<DT>::kElems];
            unpack<DT>(load_window(row, w), v);
#pragma unroll
            for (uint32_t j = 0; j < Win<DT>::kElems; j++) c += v[j] > neg_inf() && rank_key(v[j], w * Win<DT>::kElems + j - row.head) >= mid;
        }
        c = block_sum(c, sh->part);
        if (c < k) hi = mid;
        else if (c > kCap) lo = mid;
        else { x = mid; break; }
    }
    __syncthreads();
    if (threadIdx.x == 0) sh->cnt = 0;
    __syncthreads();
    for (uint32_t w = threadIdx.x; w < windows; w += blockDim.x) {
        float v[Win<DT>::kElems];
        unpack<DT>(load_window(row, w), v);
#pragma unroll
        for (uint32_t j = 0; j < Win<DT>::kElems; j++) {
            const unsigned long long key = rank_key(v[j], w * Win<DT>::kElems + j - row.head);
            if (v[j] > neg_inf() && key >= x) {
                const uint32_t at = atomicAdd(&sh->cnt, 1u);
                if (at < kCap) sh->cand[at] = key;
            }
        }
    }
    __syncthreads();
}

template <int DT> __device__ __forceinline__ uint32_t listed_bits(const uint8_t *bits, uint32_t w)
{
    return DT == SFB_F32 ? bits[w >> 1] >> ((w & 1) * 4) & 15u : bits[w];
}
// The elements of a row that are not in a whole window, one per thread of its first 2 * kElems: the window at its front, then
// the one at its back.  Their position, kNoWindow for threads (and windows) without one.
template <int DT> __device__ __forceinline__ uint32_t edge_position(const Row<DT> &row, uint32_t i)
{
    constexpr uint32_t E = Win<DT>::kElems;
    if (i >= 2 * E) return kNoWindow;
    const uint32_t w = i < E ? row.front() : row.back();
    if (w == kNoWindow) return kNoWindow;
    const uint32_t pos = w * E + i % E;
    return pos >= row.head && pos < row.end ? pos : kNoWindow;
}
template <bool ENT> __device__ __forceinline__ void add_element(Sums &a, float x, float s2, float gap)
{
    if (!a.prepare(x, s2, gap)) return;
    const float t = s2 * (x - a.r), y = ex2(t);
    a.s += y;
    if (ENT) a.e = fmaf(y, fmaxf(t, kFar), a.e);
}

// a row of tokens, its sums known beside m
template <bool ENT> __device__ __forceinline__ void finish_tokens(const StatParams &p, uint32_t r, int32_t target, float x_target, float m, float s, float e)
{
    const bool empty = m == neg_inf();
    const float l = empty ? neg_inf() : logf(s);
    p.stats[2 * (size_t)r] = m;
    p.stats[2 * (size_t)r + 1] = l;
    if (p.logp) p.logp[r] = target < 0 ? 0.f : empty ? neg_inf() : p.scale * (x_target - m) - l;
    if (ENT) p.entropy[r] = empty ? 0.f : l - kLn2 * (e / s);
}

// What a warp's entries of a row's list come to before the row's sums are known.  A divergence is small beside the logarithms that it
// is made of, so those are subtracted entry by entry, d_k = (lq_k - mq) - s (x_k - x_r) with x_r the largest listed logit, and what
// is left of the sums' logarithms is taken from their quotient: with q_k = e^(lq_k - mq) / Z
//   loss = sum_k q_k d_k - s (x_r - m) + ln (S / Z).
struct ListPart {
    float mq, z, w, x_r, listed;          // max lq, sum e = e^(lq - mq), sum e d, max x, sum over distinct of 2^(s2 (x - x_r))
};

// One warp: its entries, one per lane.  again: the lane's token stands earlier in the list.
template <int KD> __device__ __forceinline__ void sum_entries(float lq, float x, bool again, float scale, float s2, ListPart *out)
{
    const float mq = KD == 1 ? warp_max_nan(lq) : 0.f, x_r = warp_max_nan(x), base = x_r == neg_inf() ? 0.f : x_r;
    const float e = lq == neg_inf() ? 0.f : ex2(kLog2e * (lq - mq));
    const float z = warp_sum(e), w = warp_sum(e > 0.f || e != e ? e * fmaf(-scale, x - base, lq - mq) : 0.f);
    const float listed = KD == 2 ? warp_sum(again ? 0.f : ex2(s2 * (x - base))) : 0.f;
    if ((threadIdx.x & 31) == 0) *out = {mq, z, w, x_r, x_r == neg_inf() ? 0.f : listed};
}

// One thread: the row's results, m and s known.  KD 2: those of the tokens that are not listed.  Their sum stands beside their own
// largest logit: beside the row's, which a list that holds nearly all of the mass leaves far behind, it would be lost.
template <int KD> __device__ __forceinline__ void finish_lists(const StatParams &p, uint32_t r, const ListPart *part, float m, float s)
{
    const uint32_t n = (p.k + 31) / 32;
    float mq = KD == 1 ? neg_inf() : 0.f, z = 0.f, w = 0.f, listed = 0.f;
    const float m_rest = m, s_rest = s;
    if (KD == 2)
        for (uint32_t i = 0; i < n; i++) m = max_nan(m, part[i].x_r);
    const bool empty = m == neg_inf();
    if (KD == 1)
        for (uint32_t i = 0; i < n; i++) mq = max_nan(mq, part[i].mq);
    for (uint32_t i = 0; i < n; i++) {
        const ListPart g = part[i];
        const float f = KD == 2 ? 1.f : g.mq == neg_inf() ? 0.f : ex2(kLog2e * (g.mq - mq)), base = g.x_r == neg_inf() ? 0.f : g.x_r;
        z += f * g.z;
        if (!(f * g.z <= 0.f)) w += f * (g.w + g.z * fmaf(-p.scale, base - m, KD == 2 ? 0.f : g.mq - mq));     // sum of e ((lq - mq) - s (x - m))
        if (KD == 2 && g.x_r != neg_inf()) listed += g.listed * ex2(p.s2 * (base - m));
    }
    const float rest = KD == 2 && !(m_rest == neg_inf()) ? s_rest * ex2(fmaxf(p.s2 * (m_rest - m), kFar)) : 0.f;
    if (KD == 2) s = rest + listed;
    const float l = empty ? neg_inf() : logf(s);
    float loss = 0.f;
    if (!(z <= 0.f)) loss = empty ? -neg_inf() : KD == 1 ? w / z + logf(s / z) : fmaf(z, l, w);
    float *st = p.stats + (KD == 2 ? 3 : 2) * (size_t)r;
    st[0] = m;
    st[1] = l;
    if (KD == 2) {
        const float left = fmaxf(0.f, 1.f - z);
        float lr = neg_inf();
        if (!(m_rest == neg_inf())) {
            // ln p_r and ln q_r, which are small where most is left, without the sums' own logarithms; a product with the distance to the
            // largest logit stays finite where the distance times the scale may not
            const float ls = logf(s_rest);
            if (left > 0.f) loss += rest > listed ? left * (log1pf(-z) - log1pf(-listed / s)) : fmaf(left * p.scale, m - m_rest, left * (log1pf(-z) + (l - ls)));
            lr = l != l ? l : fmaxf(fmaf(p.scale, m_rest - m, ls), -FLT_MAX);      // -inf is what has no token left
        }
        st[2] = lr;
    }
    p.loss[r] = loss;
}

// A row's statistics, and what is made of them.  One CTA per row, or a cluster of CTAs where there are few rows: each
// takes every C-th piece, and CTA 0 joins the parts.  KD: 0 tokens, 1 lists, 2 lists with the remainder as one more class.
// Many rows are bound by the pass: 9 instructions and an exponential per element with entropy and alternatives, the issue slots
// 72 % and the exponential unit 66 % busy beside 5.2 TB/s from memory (2048 rows of 131072 bf16, 103 us).  8192 such rows take 355 us in a short
// burst and 421 under the power cap, when passes follow each other: 93 and 78 % of what a copy's rate allows; 4096 of 30522
// (without entropy) 46, 83 %.  Fewer rows are bound by what comes one after another:
// launch, the first loads, the join of a cluster's CTAs over their barrier (about 1000 cycles), and for alternatives their bound, the
// second look and the ranks: one row of 30522 bf16 takes 2.6 us, with entropy and 20 alternatives 5.3, 64 rows of 100003 fp16 with 5 8.1; a
// call from the host 6.7 and 10.1 of the last two.
// Rows streamed through a ring of bulk copies by CTAs that stay were built, too: the loads then never pause, but
// the warps that add up waited at every row's end for the one that finishes it, and the same rows took 59 us instead of 44.
template <int DT, bool ENT, bool TOP, int KD>
__global__ void __launch_bounds__(kThreads, 4) row_stats_kernel(const StatParams p)
{
    extern __shared__ __align__(16) uint8_t dyn[];       // TOP: the largest value of each group of windows; KD 2: a bit per position
    __shared__ Part parts[kMaxCluster * 8];
    __shared__ __align__(16) uint8_t top_raw[TOP ? sizeof(TopShared) : 16];
    TopShared *const top_s = (TopShared *)top_raw;
    __shared__ int32_t l_id[KD == 2 ? kMaxList : 1];
    __shared__ ListPart list[kMaxList / 32];
    __shared__ uint32_t l_twice;
    constexpr bool kMaySkip = KD == 0 && !ENT && !TOP;   // a row without a target has nothing to give

    const uint32_t T = blockDim.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t C = cluster_size(), rank = cluster_rank();
    const uint32_t r = blockIdx.x / C;
    // Every CTA of the cluster waits for this arrival before its first word into another CTA.  CTA 0 has to be there by then, and, with
    // alternatives, its counter of candidates, to which all of them add, has to be 0: the arrival releases that store, the wait acquires it.
    if (TOP && tid == 0) { top_s->cnt = 0; top_s->n_hits = 0; }
    if (C > 1) {
        if (TOP) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        else asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    }
    if (KD == 2)
        for (uint32_t i = tid; i < (p.vocab + 2 * Win<DT>::kElems + 31) / 32; i += T) ((uint32_t *)dyn)[i] = 0;
    grid_dependency_wait();
    grid_launch_dependents();

    bool skip = r >= p.rows;
    int32_t target = -1;
    if (skip) {
        if (rank == 0) count_missed(KD ? p.ids : p.targets, p.count_here, p.vocab, p.missed, (uint32_t *)parts);
    } else if (kMaySkip && p.targets) {
        target = p.targets[r];
        if ((uint32_t)target >= p.vocab) {
            if (rank == 0 && tid == 0) {
                if (p.missed && !p.count_here) atomicAdd(p.missed, 1u);
                p.logp[r] = 0.f;
                p.stats[2 * (size_t)r] = p.stats[2 * (size_t)r + 1] = 0.f;
            }
            skip = true;
        }
    }
    if (skip) {
        __syncwarp();
        if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        return;
    }

    // The pass goes by groups of kU windows per thread, the next group on its way while one is added up; the first sets out here.
    const void *x = (const char *)p.x + (size_t)r * p.pitch * Win<DT>::kSize;
    const Row<DT> row(x, p.vocab);
    const float gap = 40.f / p.s2;
    const uint32_t n_whole = row.whole_count(), step = C * kU * T, first = rank * kU * T;
    const uint4 *src = row.base + row.first_whole() + tid;
    float *keys = (float *)dyn;
    auto load = [&](uint4 (&v)[kU], uint32_t i0) {
        if (i0 + kU * T <= n_whole) {
#pragma unroll
            for (int u = 0; u < kU; u++) v[u] = load16(src + i0 + u * T);
        } else {
#pragma unroll
            for (int u = 0; u < kU; u++) v[u] = i0 + u * T + tid < n_whole ? load16(src + i0 + u * T) : no_elements<DT>();
        }
    };
    uint4 v[kU], next[kU];
    const uint32_t groups = first < n_whole ? (n_whole - first + step - 1) / step : 0;
    if (groups) load(next, first);
    const uint32_t edge = rank == 0 ? edge_position<DT>(row, tid) : kNoWindow;       // what is not in a whole window: an element each
    float x_edge = edge != kNoWindow ? load_element<DT>(x, edge - row.head) : neg_inf();
    const bool merges = rank == 0 && warp == (TOP ? T / 32 - 1 : 0);      // with alternatives, others look for their bound meanwhile
    float x_target = 0.f;
    if (KD == 0 && merges && p.targets) {
        if (!kMaySkip) {
            target = p.targets[r];
            if ((uint32_t)target >= p.vocab) {
                target = -1;
                if (lane == 0 && p.missed && !p.count_here) atomicAdd(p.missed, 1u);
            }
        }
        if (target >= 0) x_target = load_element<DT>(x, (uint32_t)target);
    }
    if (KD) {
        // an entry of the list per thread
        int32_t id = -1;
        float lq = neg_inf(), xl = neg_inf();
        if (tid < p.k) {
            id = p.ids[(size_t)r * p.k + tid];
            lq = p.teacher[(size_t)r * p.k + tid];
        }
        const bool ok = (uint32_t)id < p.vocab;
        if (!ok) lq = neg_inf();
        if (ok && rank == 0) xl = load_element<DT>(x, (uint32_t)id);
        bool again = false;
        if (KD == 2) {
            if (tid == 0) l_twice = 0;
            if (tid < p.k) l_id[tid] = ok ? id : -1;
            __syncthreads();                              // the bits are clear
            if (ok) {
                const uint32_t pos = row.head + (uint32_t)id, bit = 1u << (pos & 31);
                if (atomicOr((uint32_t *)dyn + (pos >> 5), bit) & bit) l_twice = 1;
            }
            __syncthreads();
            if (l_twice && ok)                            // a token that is listed twice counts once in the sum of the listed
                for (uint32_t j = 0; j < tid; j++) again |= l_id[j] == id;
        }
        if (rank == 0 && warp < (p.k + 31) / 32) {
            if (p.missed && !p.count_here) {
                const uint32_t bad = __popc(__ballot_sync(0xffffffffu, tid < p.k && !ok));
                if (lane == 0 && bad) atomicAdd(p.missed, bad);
            }
            sum_entries<KD>(lq, xl, again, p.scale, p.s2, &list[warp]);
        }
    }

    // ---- the pass ----
    Sums a;
    float mx = neg_inf();
    for (uint32_t g = 0; g < groups; g++) {
        const uint32_t i0 = first + g * step;
#pragma unroll
        for (int u = 0; u < kU; u++) v[u] = next[u];
        if (g + 1 < groups) load(next, i0 + step);
        if (KD == 2) {
#pragma unroll
            for (int u = 0; u < kU; u++) {
                const uint32_t i = i0 + u * T + tid;
                const uint32_t b = i < n_whole ? listed_bits<DT>(dyn, row.first_whole() + i) : 0;
                if (b) drop_listed<DT>(v[u], b);
            }
        }
        const float m = max_windows<DT, kU>(v);
        if (TOP) keys[g * T + tid] = m;
        mx = max_nan(mx, m);
        if (a.prepare(m, p.s2, gap)) add_windows<DT, ENT, kU>(a, v, p.s2);
    }
    if (edge != kNoWindow) {
        if (KD == 2 && ((const uint32_t *)dyn)[edge >> 5] >> (edge & 31) & 1) x_edge = neg_inf();
        mx = max_nan(mx, x_edge);
        add_element<ENT>(a, x_edge, p.s2, gap);
    }

    // ---- the parts of the warps (and CTAs) meet in CTA 0 ----
    uint32_t n_groups = 0;
    if (TOP) {
        // groups of neighbouring threads, as large as leaves 2 k of them (32 at least)
        uint32_t g = 1;
        while (g < 32 && T / (2 * g) >= max(32u, 2 * p.k)) g *= 2;
        n_groups = T / g;
        float gm = mx;
        for (uint32_t o = 1; o < g; o <<= 1) gm = max_nan(gm, __shfl_xor_sync(0xffffffffu, gm, o));
        if ((tid & (g - 1)) == 0) top_s->gm[tid / g] = (ordered(gm) & ~0xffu) | (255 - tid / g);
    }
    warp_sums<ENT>(a, mx, p.s2);
    if (C > 1) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (lane == 0) cg::this_cluster().map_shared_rank(parts, 0)[rank * 8 + warp] = Part{mx, a.s, a.e};
        if (!TOP) {
            cg::this_cluster().sync();
            if (rank) return;
        }
    } else if (lane == 0) {
        parts[warp] = Part{mx, a.s, a.e};
    }
    if (TOP || C == 1) __syncthreads();

    auto merge = [&]() {
        const uint32_t warps = T / 32;
        Sums b;
        float bm = neg_inf();
        for (uint32_t i = lane; i < C * warps; i += 32) {
            const Part q = parts[i / warps * 8 + i % warps];
            Sums c;
            c.r = q.m; c.s = q.s; c.e = q.e;
            const float m2 = max_nan(bm, q.m);
            b.move_to(m2, p.s2);
            c.move_to(m2, p.s2);
            b.s += c.s; b.e += c.e;
            bm = m2;
        }
        warp_sums<ENT>(b, bm, p.s2);
        if (lane == 0) {
            if (KD) finish_lists<KD>(p, r, list, bm, b.s);
            else finish_tokens<ENT>(p, r, target, x_target, bm, b.s, b.e);
            if (TOP) { top_s->m = bm; top_s->l = bm == neg_inf() ? neg_inf() : logf(b.s); }
        }
    };
    if (!TOP) {
        if (merges) merge();
        return;
    }

    // ---- alternatives ----
    // At least k groups of threads of a CTA have a value at or above the k-th largest of the groups' maxima, so every one of the k
    // largest values that the CTA has seen is: only windows whose maximum reaches that bound are looked at again.  CTA 0 ranks
    // what all of them find.
    if (tid < n_groups) {
        const uint32_t own = top_s->gm[tid];
        uint32_t above = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < n_groups; j += 4) {
            const uint4 o = *(const uint4 *)&top_s->gm[j];
            above += (o.x > own) + (o.y > own) + (o.z > own) + (o.w > own);
        }
        if (above == min(p.k, n_groups) - 1) top_s->tau = n_groups < p.k ? 0 : own & ~0xffu;
    }
    if (C == 1 && merges) merge();
    __syncthreads();
    const uint32_t tau = top_s->tau;
    TopShared *const join = C > 1 ? cg::this_cluster().map_shared_rank(top_s, 0) : top_s;
    auto candidate = [&](float v, uint32_t index) {
        if (v > neg_inf() && ordered(v) >= tau) {
            const uint32_t at = C > 1 ? atomicAdd(&join->cnt, 1u) : atomicAdd(&top_s->cnt, 1u);
            if (at < kCap) join->cand[at] = rank_key(v, index);
        }
    };
    if (edge != kNoWindow) candidate(x_edge, edge - row.head);
    for (uint32_t g = 0; g < groups; g++) {
        const float m = keys[g * T + tid];
        if (m > neg_inf() && ordered(m) >= tau) {
            const uint32_t at = atomicAdd(&top_s->n_hits, 1u);
            if (at < kCap) top_s->hits[at] = first + g * step + tid;
        }
    }
    __syncthreads();
    const uint32_t n_hits = top_s->n_hits;
    if (n_hits > kCap) {
        if (tid == 0) atomicAdd(&join->cnt, kCap + 1);
    } else {
        constexpr uint32_t E = Win<DT>::kElems;
        const uint32_t n = n_hits * kU * E;
        if (n <= 4 * T) {
            // few: an element each for the CTA's threads, four on their way (the shortest path of a row by itself)
            float e[4];
            uint32_t index[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const uint32_t i = tid + j * T, at = (i < n ? top_s->hits[i / (kU * E)] : 0) + i / E % kU * T;
                index[j] = (row.first_whole() + at) * E + i % E - row.head;
                e[j] = i < n && at < n_whole ? load_element<DT>(x, index[j]) : neg_inf();
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) candidate(e[j], index[j]);
        } else {
            // a window each, most of which hold nothing (64 alternatives of 4096 rows of 30522 bf16: 98 -> 87 us)
            for (uint32_t i = tid; i < n_hits * kU; i += T) {
                const uint32_t at = top_s->hits[i / kU] + i % kU * T;
                const uint4 one[1] = {at < n_whole ? load16(row.base + row.first_whole() + at) : no_elements<DT>()};
                if (!(ordered(max_windows<DT, 1>(one)) >= tau)) continue;
                float e[E];
                unpack<DT>(one[0], e);
#pragma unroll
                for (uint32_t j = 0; j < E; j++) candidate(e[j], (row.first_whole() + at) * E + j - row.head);
            }
        }
    }
    if (C > 1) {
        cg::this_cluster().sync();
        if (rank) return;
        if (merges) merge();
    } else {
        __syncthreads();
    }
    if (top_s->cnt > kCap && !collect_ties<DT>(row, p.k, top_s)) bisect_candidates<DT>(row, p.k, top_s);
    const uint32_t total = top_s->cnt;
    int32_t *out_ids = p.top_ids + (size_t)r * p.k;
    for (uint32_t i = tid; i < total; i += T) {
        const unsigned long long key = top_s->cand[i];
        uint32_t above = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < total; j++) above += top_s->cand[j] > key;
        if (above < p.k) {
            top_s->best[above] = from_ordered((uint32_t)(key >> 32));
            out_ids[above] = (int32_t)(0xffffffffu - (uint32_t)key);
        }
    }
    __syncthreads();
    const float m = top_s->m, l = top_s->l;
    const bool sound = l == l;                  // no NaN in the row
    for (uint32_t i = tid; i < p.k; i += T) {
        p.top_logp[(size_t)r * p.k + i] = !sound ? l : i < total ? p.scale * (top_s->best[i] - m) - l : neg_inf();
        if (!sound || i >= total) out_ids[i] = -1;
    }
}

// Many rows: a warp each, eight to a CTA, with nothing to wait for.  Four warps that share a row wait for its end, and the SM for
// their successors: 8192 rows of 4000 bf16 with entropy take 14 us so, 24 with a CTA per row; of 30522 83 and 91.  KD 0 or 1.
template <int DT, bool ENT, int KD>
__global__ void __launch_bounds__(kThreads, 4) short_rows_kernel(const StatParams p)
{
    constexpr uint32_t kWarps = kThreads / 32, T = 32;
    constexpr bool kMaySkip = KD == 0 && !ENT;
    __shared__ ListPart list[kWarps][kMaxList / 32];
    __shared__ uint32_t part[kWarps];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = blockIdx.x * kWarps + warp;
    grid_dependency_wait();
    grid_launch_dependents();
    if (blockIdx.x * kWarps >= p.rows) {
        count_missed(KD ? p.ids : p.targets, p.count_here, p.vocab, p.missed, part);
        return;
    }
    if (r >= p.rows) return;
    const void *x = (const char *)p.x + (size_t)r * p.pitch * Win<DT>::kSize;
    int32_t target = KD == 0 && p.targets ? p.targets[r] : -1;
    if (KD == 0 && p.targets && (uint32_t)target >= p.vocab) {
        target = -1;
        if (lane == 0 && p.missed && !p.count_here) atomicAdd(p.missed, 1u);
        if (kMaySkip) {
            if (lane == 0) { p.logp[r] = 0.f; p.stats[2 * (size_t)r] = p.stats[2 * (size_t)r + 1] = 0.f; }
            return;
        }
    }
    const Row<DT> row(x, p.vocab);
    const float gap = 40.f / p.s2;
    const uint32_t n_whole = row.whole_count();
    const uint4 *src = row.base + row.first_whole() + lane;
    auto load = [&](uint4 (&v)[kU], uint32_t i0) {
#pragma unroll
        for (int u = 0; u < kU; u++) v[u] = i0 + u * T + lane < n_whole ? load16(src + i0 + u * T) : no_elements<DT>();
    };
    uint4 v[kU], next[kU];
    if (n_whole) load(next, 0);
    const uint32_t edge = edge_position<DT>(row, lane);
    const float x_edge = edge != kNoWindow ? load_element<DT>(x, edge - row.head) : neg_inf();
    const float x_target = KD == 0 && target >= 0 ? load_element<DT>(x, (uint32_t)target) : 0.f;
    if (KD) {
        uint32_t bad = 0;
        for (uint32_t i0 = 0; i0 < p.k; i0 += 32) {
            const uint32_t i = i0 + lane;
            const int32_t id = i < p.k ? p.ids[(size_t)r * p.k + i] : -1;
            const bool ok = (uint32_t)id < p.vocab;
            bad += __popc(__ballot_sync(0xffffffffu, i < p.k && !ok));
            const float lq = ok ? p.teacher[(size_t)r * p.k + i] : neg_inf(), xl = ok ? load_element<DT>(x, (uint32_t)id) : neg_inf();
            sum_entries<KD>(lq, xl, false, p.scale, p.s2, &list[warp][i0 / 32]);
        }
        if (lane == 0 && bad && p.missed && !p.count_here) atomicAdd(p.missed, bad);
    }
    Sums a;
    float mx = neg_inf();
    for (uint32_t i0 = 0; i0 < n_whole; i0 += kU * T) {
#pragma unroll
        for (int u = 0; u < kU; u++) v[u] = next[u];
        if (i0 + kU * T < n_whole) load(next, i0 + kU * T);
        const float m = max_windows<DT, kU>(v);
        mx = max_nan(mx, m);
        if (a.prepare(m, p.s2, gap)) add_windows<DT, ENT, kU>(a, v, p.s2);
    }
    if (edge != kNoWindow) {
        mx = max_nan(mx, x_edge);
        add_element<ENT>(a, x_edge, p.s2, gap);
    }
    __syncwarp();
    warp_sums<ENT>(a, mx, p.s2);
    if (lane == 0) {
        if (KD) finish_lists<KD>(p, r, list[warp], mx, a.s);
        else finish_tokens<ENT>(p, r, target, x_target, mx, a.s, a.e);
    }
}

// ---- gradients --------------------------------------------------------------------------------------------------------
struct GradParams {
    const void *x;
    void *out;
    uint64_t pitch, out_pitch;
    uint32_t rows, vocab, width;
    uint32_t parts, per;                  // CTAs per row, windows of each
    float scale, s2;
    const int32_t *targets;
    const float *stats, *dlogp, *entropy, *dentropy;
    const int32_t *ids;
    const float *teacher, *dloss, *token_stats;
    uint32_t k;
};

// windows of x that start where those of out do not
template <int DT> __device__ __forceinline__ uint4 load_shifted(const void *x, uint32_t head, uint32_t n, uint32_t w)
{
    uint32_t v[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
        const uint32_t i = w * Win<DT>::kElems + j * (Win<DT>::kElems / 4) - head;       // below the row's start: wraps, and is no index
        if (DT == SFB_F32) {
            v[j] = i < n ? ((const uint32_t *)x)[i] : Win<DT>::kInf;
        } else {
            const uint32_t lo = i < n ? ((const uint16_t *)x)[i] : Win<DT>::kInf, hi = i + 1 < n ? ((const uint16_t *)x)[i + 1] : Win<DT>::kInf;
            v[j] = lo | hi << 16;
        }
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// One CTA of at least kMaxList threads: the list names every token of the vocabulary.
__device__ __noinline__ bool lists_all(const int32_t *ids, uint32_t vocab)
{
    bool first = threadIdx.x < kMaxList && ids[threadIdx.x] >= 0;
    for (uint32_t j = 0; j < threadIdx.x && first; j++) first = ids[j] != ids[threadIdx.x];
    return (uint32_t)__syncthreads_count(first) == vocab;
}
// One CTA: the tokens of a row that are not listed, the largest and the base-2 logarithm of their sum beside it.  ids: kMaxList of them, -1
// for none.  seen: a bit for each remainder modulo kSeen that a window with a listed token has; a warp looks at such a window together,
// four entries of the list per lane.  part: one per warp.
// With L2 flushed, 257 rows of 50021 fp32 and lists of 128 take 70 us where all remainders are far away, 29 where none is; 4096 of 30522 bf16 and
// lists of 64 182 and 102.
constexpr uint32_t kSeen = 8192;
template <int DT> __device__ __noinline__ float2 sum_unlisted(const Row<DT> row, float s2, const int32_t *ids, const uint32_t *seen, Part *part)
{
    constexpr uint32_t E = Win<DT>::kElems;
    const uint32_t windows = row.windows(), T = blockDim.x, lane = threadIdx.x % 32;
    const float gap = 40.f / s2;
    const int4 o = ((const int4 *)ids)[lane];
    Sums a;
    float mx = neg_inf();
    for (uint32_t w0 = threadIdx.x - lane; w0 < windows; w0 += T) {
        uint4 v[1] = {load_window(row, w0 + lane)};
        for (uint32_t hits = __ballot_sync(0xffffffffu, seen[(w0 + lane) % kSeen / 32] >> ((w0 + lane) % 32) & 1); hits; hits &= hits - 1) {
            const uint32_t at = __ffs(hits) - 1, first = (w0 + at) * E - row.head;     // (-1 is a position in front of the row, which holds -inf)
            auto bit = [&](int32_t id) { return (uint32_t)id - first < E ? 1u << ((uint32_t)id - first) : 0u; };
            const uint32_t bits = __reduce_or_sync(0xffffffffu, bit(o.x) | bit(o.y) | bit(o.z) | bit(o.w));
            if (lane == at) drop_listed<DT>(v[0], bits);
        }
        const float m = max_windows<DT, 1>(v);
        mx = max_nan(mx, m);
        if (a.prepare(m, s2, gap)) add_windows<DT, false, 1>(a, v, s2);
        __syncwarp();
    }
    warp_sums<false>(a, mx, s2);
    if (lane == 0) part[threadIdx.x / 32] = {mx, a.s, 0.f};
    __syncthreads();
    mx = neg_inf();
    for (uint32_t w = 0; w < T / 32; w++) mx = max_nan(mx, part[w].m);
    float s = 0.f;
    for (uint32_t w = 0; w < T / 32; w++) s += part[w].s * ex2(fmaxf(s2 * (part[w].m - mx), kFar));
    return make_float2(mx, log2f(s));
}

// A row (or a part of it) per CTA, a round of kG windows per thread at a time: loaded, turned into the gradient and stored.  Bound by
// memory: 8192 rows of 30522 bf16 156 us in a short burst, 162 when passes follow each other, 98 and 95 % of a copy's rate; lists and hard
// labels add a prologue to each row (4096 rows: 94 and 100 us, 82 and 77 %).
// dx = p (c0 + c1 t) with t the base-2 logarithm of p, plus the given target's share (KD 0, ENT: c1 is not 0);
// dx = c0 2^t + c2 2^t2, what is listed made again by itself (KD 1, and 2 with the remainder; HARD 1: c2 is not 0).  HARD 2: at temperature 2 the
// second power, the softmax's at temperature 1, is the first one's square times a constant of the row (which goes to c2), and an
// exponential per element less: 4096 rows of 30522 bf16 with lists of 64 take 104.5 us at scale 0.5, 108.5 at any other (L2 flushed).
template <int DT, bool ENT, int KD, int HARD, bool SAME>
__global__ void __launch_bounds__(kThreads, KD ? 5 : 6) row_grad_kernel(const GradParams p)
{
    __shared__ __align__(16) int32_t l_id[KD ? kMaxList : 4];
    __shared__ __align__(16) float l_q[KD ? kMaxList : 4];
    __shared__ float l_x[KD ? kMaxList + 1 : 1];              // the logits of the list's tokens, and of the target; each is its thread's own
    __shared__ uint32_t l_seen[KD == 2 ? kSeen / 32 : 1];
    __shared__ Part l_sum[KD == 2 ? kThreads / 32 : 1];
    __shared__ float2 l_part[kMaxList / 32];                  // a warp's entries: the largest teacher value, the sum of the powers beside it
    constexpr uint32_t E = Win<DT>::kElems;
    constexpr bool kMaySkip = !KD && !ENT;                    // a row without a target is zeros
    const uint32_t T = blockDim.x, tid = threadIdx.x, lane = tid & 31;
    const uint32_t r = blockIdx.x / p.parts, part = blockIdx.x - r * p.parts;
    grid_dependency_wait();
    grid_launch_dependents();

    const void *x = (const char *)p.x + (size_t)r * p.pitch * Win<DT>::kSize;
    void *out = (char *)p.out + (size_t)r * p.out_pitch * Win<DT>::kSize;
    const Row<DT> orow(out, p.width), row(x, p.vocab);        // SAME: both start at the same place of their windows
    uint32_t w_begin = part * p.per, w_end = min(orow.windows(), w_begin + p.per);
    int32_t i_begin = (int32_t)(w_begin * E) - (int32_t)orow.head, i_end = (int32_t)(w_end * E) - (int32_t)orow.head;

    int32_t target = p.targets ? p.targets[r] : -1;
    if ((uint32_t)target >= p.vocab) target = -1;
    const float *st = p.stats + (KD == 2 ? 3 : 2) * (size_t)r;
    const float m = st[0];
    const bool zero = m == neg_inf() || (kMaySkip && target < 0);       // no token is left (every probability is 0), or nothing is asked for
    // the windows [a_begin, a_end) are whole ones of x and out (none if theirs start at different places); the few others come after them
    uint32_t a_begin, a_end, rounds, first_round;
    auto set_rounds = [&]() {
        a_begin = SAME ? max(w_begin, row.first_whole()) : w_begin;
        a_end = SAME ? max(a_begin, min(w_end, row.first_whole() + row.whole_count())) : w_begin;
        rounds = (a_end - a_begin + kG * T - 1) / (kG * T);
        first_round = rounds ? r % rounds : 0;
    };
    set_rounds();
    uint4 v[kG];
    auto load_round = [&](uint32_t round) {
        const uint32_t w0 = a_begin + round * (kG * T) + tid;
#pragma unroll
        for (int u = 0; u < kG; u++)
            if (w0 + u * T < a_end) v[u] = __ldcs(row.base + w0 + u * T);
    };
    if (!zero && rounds) load_round(first_round);

    float c0, c1 = 0.f, c2 = 0.f, l2, l2b = 0.f, target_share = 0.f;
    float ref = m;                                            // what the exponents of the pass are taken beside
    float listed_c = 0.f;
    if (!KD) {
        const float g = target >= 0 ? p.dlogp[r] : 0.f;
        l2 = st[1] * kLog2e;
        c0 = -p.scale * g;
        if (ENT) {
            const float h = p.dentropy[r];
            c0 = -p.scale * (g + h * p.entropy[r]);
            c1 = -p.scale * h * kLn2;
        }
        target_share = p.scale * g;
    } else {
        int32_t id = -1;                                      // this thread's entry of the list
        float lq = neg_inf();
        if (tid < p.k) {
            id = p.ids[(size_t)r * p.k + tid];
            lq = p.teacher[(size_t)r * p.k + tid];
            if ((uint32_t)id >= p.vocab) { id = -1; lq = neg_inf(); }
            l_id[tid] = id;
        } else if (tid < kMaxList) {
            l_id[tid] = -1;
        }
        const uint32_t n = (p.k + 31) / 32;
        if (tid / 32 < n) {
            const float mq = KD == 2 ? 0.f : warp_max_nan(lq), z = warp_sum(lq == neg_inf() ? 0.f : ex2(kLog2e * (lq - mq)));
            if (lane == 0) l_part[tid / 32] = make_float2(mq, z);
        }
        // out may be x: what is listed (and the target) is read before anything is written
        auto load_listed = [&]() {
            if (id >= i_begin && id < i_end && id >= 0) l_x[tid] = load_element<DT>(x, (uint32_t)id);
            if (HARD && tid == 0 && target >= 0 && target >= i_begin && target < i_end) l_x[kMaxList] = load_element<DT>(x, (uint32_t)target);
        };
        load_listed();
        const float sw = p.scale * p.dloss[r], l = st[1], lr = KD == 2 ? st[2] : 0.f;
        if (HARD) {
            const float g = target >= 0 ? p.dlogp[r] : 0.f;
            c2 = -g;
            l2b = p.token_stats[2 * (size_t)r + 1] * kLog2e;
        }
        __syncthreads();
        float mq = KD == 2 ? 0.f : neg_inf(), z = 0.f;
        if (KD == 1)
            for (uint32_t w = 0; w < n; w++) mq = max_nan(mq, l_part[w].x);
        for (uint32_t w = 0; w < n; w++) z += l_part[w].x == neg_inf() ? 0.f : l_part[w].y * (KD == 2 ? 1.f : ex2(kLog2e * (l_part[w].x - mq)));
        const bool none = mq == neg_inf();
        if (tid < kMaxList) l_q[tid] = lq == neg_inf() || none ? 0.f : ex2(kLog2e * (lq - mq)) * (KD == 2 ? 1.f : 1.f / z);
        const float left = KD == 2 ? fmaxf(0.f, 1.f - z) : 0.f, all = KD == 2 ? z + left : none ? 0.f : 1.f;
        listed_c = sw * all;
        l2 = l * kLog2e;
        c0 = sw * all;
        if (KD == 2) {
            // unlisted tokens: all * p - left * p / p_rest, as a multiple of their share of the remainder
            if (lr == neg_inf()) {
                // Every unlisted one has a probability of 0, the loss has no term for the remainder, and neither has its gradient.  (A list that
                // holds the whole vocabulary keeps q_r in Q: no token is there to take it, and nothing goes to one.)
                if (!(p.k >= p.vocab && lists_all(l_id, p.vocab))) listed_c = sw * z;
                c0 = 0.f;
            } else {
                c0 = sw * (all * expf(lr - l) - left);
                l2 = lr * kLog2e;
            }
            if (lr < kFarRest && lr > neg_inf() && left > 0.f) {
                // One CTA for the whole row, the others are done: out may be x, and the row is read before any of it is written.
                if (part) return;
                w_end = orow.windows();
                i_end = (int32_t)(w_end * E) - (int32_t)orow.head;
                set_rounds();
                load_listed();
                for (uint32_t i = tid; i < kSeen / 32; i += T) l_seen[i] = 0;
                __syncthreads();
                const uint32_t w_id = ((uint32_t)id + row.head) / E;
                if (id >= 0) atomicOr(&l_seen[w_id % kSeen / 32], 1u << (w_id % 32));
                __syncthreads();
                const float2 rest = sum_unlisted<DT>(row, p.s2, l_id, l_seen, l_sum);
                ref = rest.x;
                l2 = rest.y;
#pragma unroll
                for (int u = 0; u < kG; u++) v[u] = no_elements<DT>();
                if (!zero && rounds) load_round(first_round);
            }
        }
    }

    const uint32_t w_target = !KD && target >= 0 ? ((uint32_t)target + orow.head) / E : kNoWindow;
    const Pair minus_r = pair(-ref, -ref), s2 = pair(p.s2, p.s2), minus_l = pair(-l2, -l2), k0 = pair(c0, c0), k1 = pair(c1, c1);
    // HARD 2: 2^t2 = (2^t)^2 * 2^(2 l2 - l2b)
    const float c2s = HARD == 2 ? c2 * ex2(fmaf(2.f, l2, -l2b)) : c2;
    const float l2r = HARD == 1 ? fmaf(kLog2e, m - ref, l2b) : l2b;
    const Pair log2e = pair(kLog2e, kLog2e), minus_lb = pair(-l2r, -l2r), k2 = pair(c2s, c2s);
    auto turn = [&](float (&y)[E]) {
#pragma unroll
        for (uint32_t j = 0; j < E; j += 2) {
            const Pair d = add2(pair(y[j], y[j + 1]), minus_r), t = fma2(s2, d, minus_l);
            float t0, t1;
            halves(t, t0, t1);
            const Pair e = pair(ex2(t0), ex2(t1));
            Pair g = mul2(e, ENT ? fma2(k1, pair(fmaxf(t0, kFar), fmaxf(t1, kFar)), k0) : k0);
            if (HARD == 1) {
                halves(fma2(log2e, d, minus_lb), t0, t1);
                g = fma2(k2, pair(ex2(t0), ex2(t1)), g);
            } else if (HARD == 2) {
                g = fma2(mul2(k2, e), e, g);
            }
            halves(g, y[j], y[j + 1]);
        }
    };
    auto add_target = [&](float (&y)[E]) {
        const uint32_t at = ((uint32_t)target + orow.head) % E;
#pragma unroll
        for (uint32_t j = 0; j < E; j++)
            if (j == at) y[j] += target_share;
    };
    if (zero) {
        for (uint32_t w = a_begin + tid; w < a_end; w += T) {
            float y[E] = {};
            if (w == w_target) add_target(y);
            __stcs((uint4 *)orow.base + w, pack<DT>(y));
        }
    } else {
        // Rows start at different rounds: with all of them at the same column, reads and writes crowded the same memory channels
        // (8192 rows of 30522 bf16: 195 us so, 158 with it).
        for (uint32_t i = 0, round = first_round; i < rounds; i++) {
            const uint32_t w0 = a_begin + round * (kG * T) + tid;
            round = round + 1 == rounds ? 0 : round + 1;
#pragma unroll
            for (int u = 0; u < kG; u++) {
                const uint32_t w = w0 + u * T;
                if (w >= a_end) break;
                float y[E];
                unpack<DT>(v[u], y);
                turn(y);
                if (w == w_target) add_target(y);
                __stcs((uint4 *)orow.base + w, pack<DT>(y));
            }
            // all of a round's loads after all of the last one's stores: taking turns window by window cost 20 % of the bandwidth
            asm volatile("" ::: "memory");
            if (i + 1 < rounds) load_round(round);
        }
    }
    // the windows before and behind those, element by element where they are not whole
    for (uint32_t n = tid;; n += T) {
        const uint32_t before = a_begin - w_begin, w = n < before ? w_begin + n : max(a_end, w_begin) + (n - before);
        if (w >= w_end) break;
        float y[E];
        unpack<DT>(SAME ? load_window(row, w) : load_shifted<DT>(x, orow.head, p.vocab, w), y);
        if (zero) {
#pragma unroll
            for (uint32_t j = 0; j < E; j++) y[j] = 0.f;
        } else {
            turn(y);
        }
        if (w == w_target) add_target(y);
#pragma unroll
        for (uint32_t j = 0; j < E; j++) {
            const uint32_t pos = w * E + j;
            // behind the vocabulary it is 0 whatever the row's factors are (times which a probability of 0 may be NaN)
            if (pos >= orow.head && pos < orow.end) store_element<DT>(out, pos - orow.head, pos - orow.head < p.vocab ? y[j] : 0.f);
        }
    }
    if (!KD) return;
    // What is listed, and the target: made again from all the shares it has.  A token that stands in the list twice is
    // written twice, with the same value.
    __syncthreads();
    const float listed_w = p.scale * p.dloss[r], l2_listed = st[1] * kLog2e, l2_hard = HARD ? p.token_stats[2 * (size_t)r + 1] * kLog2e : 0.f;
    auto again = [&](int32_t token, float xl) {
        float q = 0.f;
        bool listed = false;
        for (uint32_t j = 0; j < p.k; j += 4) {
            const int4 o = *(const int4 *)&l_id[j];
            const float4 w = *(const float4 *)&l_q[j];
            if (o.x == token) { q += w.x; listed = true; }
            if (o.y == token) { q += w.y; listed = true; }
            if (o.z == token) { q += w.z; listed = true; }
            if (o.w == token) { q += w.w; listed = true; }
        }
        const float d = xl - m;
        float y = 0.f;
        if (!zero) y = listed ? listed_c * ex2(fmaf(p.s2, d, -l2_listed)) : c0 * ex2(fmaf(p.s2, xl - ref, -l2));
        y -= listed_w * q;
        if (HARD) {
            if (!zero) y = fmaf(c2, ex2(fmaf(kLog2e, d, -l2_hard)), y);
            if (token == target) y -= c2;
        }
        store_element<DT>(out, (uint32_t)token, y);
    };
    const int32_t id = tid < kMaxList ? l_id[tid] : -1;
    if (id >= 0 && id >= i_begin && id < i_end) again(id, l_x[tid]);
    if (HARD && tid == 0 && target >= 0 && target >= i_begin && target < i_end) again(target, l_x[kMaxList]);
}

// ---- launches -----------------------------------------------------------------------------------------------------------
template <int DT, bool ENT, bool TOP, int KD> static int launch_stats(cudaStream_t s, StatParams &p, const char *who)
{
    const int dev = current_device(), sms = device_sm_count(dev);
    SFB_REQUIRE(sms > 0, "%s: cannot query the device", who);
    const uint32_t windows = p.vocab / Win<DT>::kElems + 2;      // at most, wherever a row starts
    const uint64_t entries = p.missed ? KD ? (uint64_t)p.rows * p.k : p.targets ? p.rows : 0 : 0;
    if constexpr (!TOP && KD != 2) {
        constexpr bool kMaySkip = KD == 0 && !ENT;
        // A warp per row: short rows, and rows up to four times as long where there is one for every warp that the SMs hold, unless they may
        // have nothing to do.  (Of longer ones the last to be dealt take too long by themselves: 5000 rows of 50021 fp32 190 us, 153 else.)
        if (p.rows >= (uint32_t)sms * 8 && (windows <= kShort || (windows <= 4 * kShort && p.rows >= (uint32_t)sms * 32 && !(kMaySkip && p.targets)))) {
            p.count_here = entries <= kThreads * 32 ? (uint32_t)entries : 0;
            if (!p.count_here && set_zero(who, p.missed, s)) return 1;
            const uint32_t rows_per = kThreads / 32;
            launch_overlapped(short_rows_kernel<DT, ENT, KD>, dim3((p.rows + rows_per - 1) / rows_per + (p.count_here ? 1 : 0)), dim3(kThreads), 0, s, p);
            return check_launch(who);
        }
    }
    // What a row's end costs is paid by each of its warps, so many rows have four of them each (4096 rows of 30522 bf16: 44 us, with
    // eight 50), few rows eight (257 of 50021 fp32: 19 us, with four 25), and so have long rows with alternatives, whose bound is the
    // tighter the more threads it comes from (4096 rows of 100003 bf16, 20 alternatives: 162 us, with four 180).  Many short rows
    // with few alternatives, or short lists and their remainder, have two (8192 of 1000 fp32, one alternative: 20 us, with four 32; 8192
    // of 1000 bf16, lists of 64: 22 and 32).
    uint32_t T = windows > 256 || TOP || KD ? 128 : 64;
    if (windows > 512 && (p.rows < (uint32_t)sms * 8 || (TOP && (p.k > 32 || windows > 8192)))) T = 256;
    if (((TOP && p.k <= 32) || (KD == 2 && p.k <= 64)) && windows <= 1024 && p.rows >= (uint32_t)sms * 8) T = 64;
    uint32_t C = 1;
    // CTAs per row, while each has more than a group of windows: as many as there are SMs without one, and a few for every SM where
    // each has two groups.  With alternatives CTA 0 ranks what all of them find, at least k from each, in time that grows as the square: from
    // 40 on that costs more than a shorter pass gives (rows of 131072: one row with 20 in four CTAs 7.8 us, in eight 7.7; 40 in two 10.5, in eight
    // 12.9; 64 in one 14.1, in eight 25.3; 64 rows with 20 in four 9.6, in eight 12.8).
    while (C < kMaxCluster && windows > C * kU * T && (!TOP || C * p.k <= 40)) {
        const uint64_t ctas = (uint64_t)p.rows * C * 2;
        if (ctas > (uint64_t)sms && (2 * ctas > 7 * (uint64_t)sms || windows < 2 * C * 2 * kU * T)) break;
        C *= 2;
    }
    p.count_here = entries <= T * 32u ? (uint32_t)entries : 0;
    if (!p.count_here && set_zero(who, p.missed, s)) return 1;
    for (;; C = 1) {
        const uint32_t groups = (windows + C * kU * T - 1) / (C * kU * T);
        const size_t smem = TOP ? (size_t)groups * T * sizeof(float) : KD == 2 ? ((size_t)p.vocab + 2 * Win<DT>::kElems + 31) / 32 * 4 : 0;
        SFB_REQUIRE(smem <= 200 * 1024, "%s: vocab=%u is too large", who, p.vocab);
        static DeviceOnce once;
        if (!once.done(dev)) {
            SFB_REQUIRE(cudaFuncSetAttribute(row_stats_kernel<DT, ENT, TOP, KD>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) == cudaSuccess,
                        "%s: cannot reserve shared memory", who);
            once.mark(dev);
        }
        const uint32_t grid = (p.rows + (p.count_here ? 1 : 0)) * C;
        const cudaError_t e = launch_overlapped_cluster(row_stats_kernel<DT, ENT, TOP, KD>, dim3(grid), dim3(T), smem, s, C, p);
        if (e == cudaSuccess || C == 1) break;
        (void)cudaGetLastError();                // a device or a partition that cannot place clusters
    }
    return check_launch(who);
}

template <int DT, bool ENT, int KD, int HARD> static int launch_grad(cudaStream_t s, GradParams &p, const char *who)
{
    const int sms = device_sm_count(current_device());
    SFB_REQUIRE(sms > 0, "%s: cannot query the device", who);
    const uint32_t windows = p.width / Win<DT>::kElems + 2;
    const uint32_t T = windows > 512 ? 256 : windows > 256 || KD ? 128 : 64;
    const uint32_t round = T * kG;
    uint32_t rounds = (windows + round - 1) / round;
    // A CTA takes several rounds of windows where enough CTAs are left for every SM: lists cost each CTA a few thousand cycles.
    uint32_t per = 1;
    while (per < rounds && (uint64_t)p.rows * ((rounds + per * 2 - 1) / (per * 2)) >= (uint64_t)sms * (KD ? 4 : 32)) per *= 2;
    p.per = per * round;
    p.parts = (windows + p.per - 1) / p.per;
    SFB_REQUIRE((uint64_t)p.rows * p.parts < (1ull << 31), "%s: too many rows", who);
    const uint64_t size = Win<DT>::kSize;
    const bool same = ((uintptr_t)p.x & 15) == ((uintptr_t)p.out & 15) && (p.pitch * size & 15) == (p.out_pitch * size & 15);
    const dim3 grid(p.rows * p.parts);
    if (same) launch_overlapped(row_grad_kernel<DT, ENT, KD, HARD, true>, grid, dim3(T), 0, s, p);
    else launch_overlapped(row_grad_kernel<DT, ENT, KD, HARD, false>, grid, dim3(T), 0, s, p);
    return check_launch(who);
}

}  // namespace lg

#define BY_TYPE(dtype, f, ...)                                                                         \
    ((dtype) == SFB_F32 ? f<SFB_F32, __VA_ARGS__> : (dtype) == SFB_BF16 ? f<SFB_BF16, __VA_ARGS__> : f<SFB_F16, __VA_ARGS__>)

static int check_rows(const char *who, const void *x, uint64_t pitch, uint32_t rows, uint32_t vocab, uint32_t width, int dtype, float scale)
{
    SFB_REQUIRE(valid_dtype(dtype), "%s: unknown dtype %d", who, dtype);
    SFB_REQUIRE(x && ((uintptr_t)x & (elem_size(dtype) - 1)) == 0, "%s: logits are NULL or not aligned to their elements", who);
    SFB_REQUIRE(vocab >= 1 && vocab <= width && width <= (1u << 30), "%s: vocab=%u of width=%u out of range", who, vocab, width);
    SFB_REQUIRE(pitch >= width || rows <= 1, "%s: a row pitch smaller than the rows", who);
    SFB_REQUIRE(rows < (1u << 27), "%s: too many rows", who);
    SFB_REQUIRE(scale > 0.f && scale <= 1e6f, "%s: scale must be positive (and at most 1e6)", who);
    return 0;
}

}  // namespace sfb

using namespace sfb;

extern "C" int sfb_token_logprobs(sfb_stream_t stream, const void *logits, uint64_t pitch, const int32_t *targets, uint32_t rows, uint32_t vocab,
                                  int dtype, float scale, float *logp, float *stats, float *entropy, float *top_logp, int32_t *top_ids,
                                  uint32_t top_k, uint32_t *missed)
{
    const char *who = "sfb_token_logprobs";
    if (rows == 0) return set_zero(who, missed, as_stream(stream));
    if (check_rows(who, logits, pitch, rows, vocab, vocab, dtype, scale)) return 1;
    SFB_REQUIRE(stats, "%s: NULL pointer", who);
    SFB_REQUIRE(!targets == !logp, "%s: targets and logp go together", who);
    SFB_REQUIRE(top_k <= lg::kMaxList && top_k <= vocab, "%s: top_k=%u must be at most %u and vocab=%u", who, top_k, lg::kMaxList, vocab);
    SFB_REQUIRE(top_k == 0 || (top_logp && top_ids), "%s: NULL pointer", who);
    SFB_REQUIRE(top_k == 0 || vocab <= (1u << 19), "%s: vocab=%u is too large for alternatives (%u)", who, vocab, 1u << 19);
    lg::StatParams p = {logits, pitch, rows, vocab, scale, scale * lg::kLog2e, targets, logp, stats, entropy, top_logp, top_ids, top_k,
                        nullptr, nullptr, nullptr, targets ? missed : nullptr, 0};
    cudaStream_t s = as_stream(stream);
    if (!targets && set_zero(who, missed, s)) return 1;
    if (top_k) return entropy ? BY_TYPE(dtype, lg::launch_stats, true, true, 0)(s, p, who) : BY_TYPE(dtype, lg::launch_stats, false, true, 0)(s, p, who);
    return entropy ? BY_TYPE(dtype, lg::launch_stats, true, false, 0)(s, p, who) : BY_TYPE(dtype, lg::launch_stats, false, false, 0)(s, p, who);
}

extern "C" int sfb_token_logprobs_grad(sfb_stream_t stream, const void *logits, uint64_t pitch, const int32_t *targets, const float *stats,
                                       const float *dlogp, const float *entropy, const float *dentropy, void *out, uint64_t out_pitch, uint32_t rows,
                                       uint32_t vocab, uint32_t width, int dtype, float scale)
{
    const char *who = "sfb_token_logprobs_grad";
    if (rows == 0) { clear_error(); return 0; }
    if (check_rows(who, logits, pitch, rows, vocab, width, dtype, scale)) return 1;
    SFB_REQUIRE(targets && stats && dlogp && out, "%s: NULL pointer", who);
    SFB_REQUIRE(!entropy == !dentropy, "%s: entropy and dentropy go together", who);
    SFB_REQUIRE(((uintptr_t)out & (elem_size(dtype) - 1)) == 0 && (out_pitch >= width || rows <= 1), "%s: out is misaligned or its rows overlap", who);
    lg::GradParams p = {logits, out, pitch, out_pitch, rows, vocab, width, 0, 0, scale, scale * lg::kLog2e, targets, stats, dlogp, entropy, dentropy,
                        nullptr, nullptr, nullptr, nullptr, 0};
    cudaStream_t s = as_stream(stream);
    return dentropy ? BY_TYPE(dtype, lg::launch_grad, true, 0, 0)(s, p, who) : BY_TYPE(dtype, lg::launch_grad, false, 0, 0)(s, p, who);
}

extern "C" int sfb_distill_topk(sfb_stream_t stream, const void *logits, uint64_t pitch, const int32_t *ids, const float *teacher, uint32_t rows,
                                uint32_t vocab, uint32_t k, int dtype, float scale, int tail, float *loss, float *stats, uint32_t *missed)
{
    const char *who = "sfb_distill_topk";
    if (rows == 0) return set_zero(who, missed, as_stream(stream));
    if (check_rows(who, logits, pitch, rows, vocab, vocab, dtype, scale)) return 1;
    SFB_REQUIRE(ids && teacher && loss && stats, "%s: NULL pointer", who);
    SFB_REQUIRE(k >= 1 && k <= lg::kMaxList, "%s: %u entries per list (1 to %u)", who, k, lg::kMaxList);
    SFB_REQUIRE(!tail || vocab <= (1u << 20), "%s: vocab=%u is too large for the remainder (%u)", who, vocab, 1u << 20);
    lg::StatParams p = {logits, pitch, rows, vocab, scale, scale * lg::kLog2e, nullptr, nullptr, stats, nullptr, nullptr, nullptr, k,
                        ids, teacher, loss, missed, 0};
    cudaStream_t s = as_stream(stream);
    return tail ? BY_TYPE(dtype, lg::launch_stats, false, false, 2)(s, p, who) : BY_TYPE(dtype, lg::launch_stats, false, false, 1)(s, p, who);
}

extern "C" int sfb_distill_topk_grad(sfb_stream_t stream, const void *logits, uint64_t pitch, const int32_t *ids, const float *teacher,
                                     const float *stats, const float *dloss, const int32_t *targets, const float *token_stats, const float *dlogp,
                                     void *out, uint64_t out_pitch, uint32_t rows, uint32_t vocab, uint32_t width, uint32_t k, int dtype, float scale,
                                     int tail)
{
    const char *who = "sfb_distill_topk_grad";
    if (rows == 0) { clear_error(); return 0; }
    if (check_rows(who, logits, pitch, rows, vocab, width, dtype, scale)) return 1;
    SFB_REQUIRE(ids && teacher && stats && dloss && out, "%s: NULL pointer", who);
    SFB_REQUIRE(!targets == !token_stats && !targets == !dlogp, "%s: targets, token_stats and dlogp go together", who);
    SFB_REQUIRE(k >= 1 && k <= lg::kMaxList, "%s: %u entries per list (1 to %u)", who, k, lg::kMaxList);
    SFB_REQUIRE(((uintptr_t)out & (elem_size(dtype) - 1)) == 0 && (out_pitch >= width || rows <= 1), "%s: out is misaligned or its rows overlap", who);
    lg::GradParams p = {logits, out, pitch, out_pitch, rows, vocab, width, 0, 0, scale, scale * lg::kLog2e, targets, stats, dlogp, nullptr, nullptr,
                        ids, teacher, dloss, token_stats, k};
    cudaStream_t s = as_stream(stream);
    if (tail) return targets ? BY_TYPE(dtype, lg::launch_grad, false, 2, 1)(s, p, who) : BY_TYPE(dtype, lg::launch_grad, false, 2, 0)(s, p, who);
    if (!targets) return BY_TYPE(dtype, lg::launch_grad, false, 1, 0)(s, p, who);
    return scale == 0.5f ? BY_TYPE(dtype, lg::launch_grad, false, 1, 2)(s, p, who) : BY_TYPE(dtype, lg::launch_grad, false, 1, 1)(s, p, who);
}

extern "C" uint64_t sfb_linear_logprobs_workspace(uint32_t m, uint32_t vocab) { return tc_linear_logprobs_workspace(m, vocab); }

extern "C" int sfb_linear_logprobs(sfb_stream_t stream, const void *x, const void *table, const float *bias, const int32_t *targets, uint32_t m,
                                   uint32_t vocab, uint32_t k, int dtype, float scale, float *logp, float *stats, float *entropy, uint32_t *missed,
                                   void *workspace)
{
    const char *who = "sfb_linear_logprobs";
    if (m == 0) return set_zero(who, missed, as_stream(stream));
    SFB_REQUIRE(x && table && targets && logp && stats && workspace, "%s: NULL pointer", who);
    SFB_REQUIRE(dtype == SFB_BF16 || dtype == SFB_F16, "%s: x and table must be bf16 or fp16", who);
    SFB_REQUIRE(vocab >= 1 && vocab <= (1u << 30) && k >= 8 && k % 8 == 0 && k <= (1u << 30), "%s: vocab=%u must be at least 1, k=%u a multiple of 8", who, vocab, k);
    SFB_REQUIRE(m < (1u << 27), "%s: too many rows", who);
    SFB_REQUIRE((((uintptr_t)x | (uintptr_t)table | (uintptr_t)workspace) & 15) == 0, "%s: x, table and workspace must be 16-byte aligned", who);
    SFB_REQUIRE(scale > 0.f && scale <= 1e6f, "%s: scale must be positive (and at most 1e6)", who);
    return tc_linear_logprobs(as_stream(stream), x, table, bias, targets, m, vocab, k, dtype, scale, logp, stats, entropy, missed, workspace);
}
