// Gradients of the embedding lookup out[b, l] = scale table[ids[b, l]] + pos[l]:
//   dtable[v] = scale sum over the tokens with id v of dout,     dpos[l] = sum over the batch of dout[., l].
// No atomics on floating-point numbers: every sum has a fixed order, so that the same inputs give the same bits.
//
// Three launches.  (1) sort_and_positions_kernel: some CTAs bring the tokens into the order of their ids, equal ids by position, while the others
// add up the batch, reading dout in order.  (2) table_grad_kernel walks the sorted tokens in pieces of equal length, so that a word that
// is a tenth of the text does not hang on one CTA; a run of equal ids that lies in one piece is written at once, the parts of
// one that does not go to the workspace.  The rows of tokens that do not occur are zeros from the first launch.
// (3) join_kernel adds up the parts.  Bound by memory: dout is read by (1) and gathered by (2), from L2 where it fits, and the table's
// gradient is written once.  Few tokens: one launch (few_tokens_kernel).
#include "common.cuh"

namespace sfb {
namespace emb {

constexpr uint32_t kSortThreads = 512, kSortWarps = kSortThreads / 32;
constexpr uint32_t kStride = kSortWarps + 1;         // counters per id: neighbouring ids in different banks
constexpr uint32_t kNear = 2048;                     // tokens of a CTA that it keeps in shared memory
constexpr uint32_t kFill = 8192;                     // 16-byte pieces of zeros per CTA
constexpr uint32_t kFew = 2048, kFewCtas = 2560;     // tokens, and CTAs for them, up to which one launch makes everything
constexpr uint32_t kMaxRange = 1024;                 // ids that one CTA sorts

struct GradArgs {
    const void *dout;
    const int32_t *ids;
    void *dtable, *dpos;
    uint32_t n, batch, len, hidden, vocab, range, sorters, pos_ctas, fillers, ways, piece, pieces;      // fillers: CTAs that write the table's zeros ahead
    float scale;
    int accumulate;
    uint32_t *bad;
    // workspace
    int2 *sorted, *unsorted;                         // (position, id), in the order of the ids; one CTA's in the order of the positions
    uint32_t *starts;                                // [vocab + 1]
    float *parts;                                    // [pieces][2][hidden]
};

__device__ __forceinline__ uint32_t warp_scan(uint32_t v, uint32_t lane)      // inclusive
{
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= (uint32_t)o) v += u;
    }
    return v;
}

// A CTA owns `range` consecutive ids and looks at all tokens: it counts those below its range, which is where its part of the sorted
// list begins, and collects its own in order, a share of the tokens per warp.  These are then sorted by counting, per warp and id, so
// that equal ids stay in order.  No CTA waits for another.  The ids come from L2 (4 bytes per token and CTA).
__device__ __forceinline__ void sort_ids(const GradArgs &a, uint32_t *count)      // count: [range][kStride]
{
    __shared__ int2 near_list[kNear];
    __shared__ uint32_t s_below[kSortWarps], s_mine[kSortWarps], s_bad[kSortWarps], s_sum[kSortWarps];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t lo = blockIdx.x * a.range, width = min(a.range, a.vocab - lo);
    // a warp's share of the tokens, 128 at a time: four neighbours per lane, four such loads on their way
    const uint32_t share = ((a.n + kSortWarps - 1) / kSortWarps + 127) / 128 * 128, t0 = min(a.n, warp * share), t1 = min(a.n, t0 + share);
    const bool wide = ((uintptr_t)a.ids & 15) == 0;
    auto fetch = [&](uint32_t t, uint32_t (&id)[4]) {          // tokens t to t + 3; beyond the share: no id
        if (wide && t + 4 <= t1) {
            const uint4 u = __ldg((const uint4 *)(a.ids + t));
            id[0] = u.x; id[1] = u.y; id[2] = u.z; id[3] = u.w;
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) id[j] = t + j < t1 ? (uint32_t)__ldg(a.ids + t + j) : 0xffffffffu;
        }
    };
    uint32_t below = 0, mine = 0, bad = 0;
    for (uint32_t t = t0; t < t1; t += 512) {
        uint32_t id[4][4];
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) fetch(t + 128 * k + 4 * lane, id[k]);
#pragma unroll
        for (uint32_t k = 0; k < 4; k++)
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {                 // a negative id is a large one
                below += id[k][j] < lo;
                mine += id[k][j] - lo < width;
                bad += t + 128 * k + 4 * lane + j < t1 && id[k][j] >= a.vocab;
            }
    }
    below = __reduce_add_sync(0xffffffffu, below);
    mine = __reduce_add_sync(0xffffffffu, mine);
    bad = __reduce_add_sync(0xffffffffu, bad);
    if (lane == 0) {
        s_below[warp] = below;
        s_mine[warp] = mine;
        s_bad[warp] = bad;
    }
    for (uint32_t i = threadIdx.x; i < width * kStride; i += kSortThreads) count[i] = 0;
    __syncthreads();
    uint32_t base = 0, total = 0, before = 0, bad_all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSortWarps; w++) {
        base += s_below[w];
        if (w < warp) before += s_mine[w];
        total += s_mine[w];
        bad_all += s_bad[w];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.bad) *a.bad = bad_all;
    // own tokens, in order of position
    int2 *list = total <= kNear ? near_list : a.unsorted + base;
    if (total) {
        uint32_t at = before;
        for (uint32_t t = t0; t < t1; t += 512) {
            uint32_t id[4][4];
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) fetch(t + 128 * k + 4 * lane, id[k]);
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) {
                uint32_t lower = 0, all = 0;                   // of the lanes below; of all
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {
                    const uint32_t votes = __ballot_sync(0xffffffffu, id[k][j] - lo < width);
                    lower += __popc(votes & ((1u << lane) - 1u));
                    all += __popc(votes);
                }
#pragma unroll
                for (uint32_t j = 0; j < 4; j++)
                    if (id[k][j] - lo < width) list[at + lower++] = make_int2((int)(t + 128 * k + 4 * lane + j), (int)id[k][j]);
                at += all;
            }
        }
    }
    __syncthreads();
    // how often each warp's share of them has each id
    const uint32_t part = ((total + kSortWarps - 1) / kSortWarps + 31) / 32 * 32, i0 = min(total, warp * part), i1 = min(total, i0 + part);
    for (uint32_t i = i0 + lane; i < i1; i += 32) atomicAdd(&count[((uint32_t)list[i].y - lo) * kStride + warp], 1u);
    __syncthreads();
    // where each (id, warp) begins: an exclusive scan, ids outermost; a thread takes neighbouring ids
    const uint32_t per = (width + kSortThreads - 1) / kSortThreads, v0 = min(width, threadIdx.x * per), v1 = min(width, v0 + per);
    uint32_t sum = 0;
    for (uint32_t v = v0; v < v1; v++)
        for (uint32_t w = 0; w < kSortWarps; w++) sum += count[v * kStride + w];
    const uint32_t upto = warp_scan(sum, lane);
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    uint32_t off = upto - sum;
#pragma unroll
    for (uint32_t w = 0; w < kSortWarps; w++)
        if (w < warp) off += s_sum[w];
    for (uint32_t v = v0; v < v1; v++) {
        a.starts[lo + v] = base + off;
        for (uint32_t w = 0; w < kSortWarps; w++) {
            const uint32_t c = count[v * kStride + w];
            count[v * kStride + w] = off;
            off += c;
        }
    }
    if (lo + width == a.vocab && threadIdx.x == 0) a.starts[a.vocab] = base + total;
    __syncthreads();
    for (uint32_t i = i0; i < i1; i += 32) {
        const bool in = i + lane < i1;
        const int2 e = in ? list[i + lane] : make_int2(0, -1);
        const uint32_t same = __match_any_sync(0xffffffffu, e.y), rank = __popc(same & ((1u << lane) - 1u));
        uint32_t *c = &count[(in ? (uint32_t)e.y - lo : 0u) * kStride + warp];
        const uint32_t at = in ? *c + rank : 0u;
        __syncwarp();
        if (in && rank == 0) *c += __popc(same);
        __syncwarp();
        if (in) a.sorted[base + at] = e;
    }
}

// ---- sums of rows --------------------------------------------------------------------------------------------------------------
template <int DT> struct Piece;                      // what a lane has of a row: 16 bytes
template <> struct Piece<SFB_F32> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void add(float (&s)[N], const uint4 &u)
    {
        s[0] += __uint_as_float(u.x); s[1] += __uint_as_float(u.y); s[2] += __uint_as_float(u.z); s[3] += __uint_as_float(u.w);
    }
};
template <> struct Piece<SFB_BF16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void add(float (&s)[N], const uint4 &u)
    {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            s[2 * i] += __uint_as_float(w[i] << 16);
            s[2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};
template <> struct Piece<SFB_F16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void add(float (&s)[N], const uint4 &u)
    {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            s[2 * i] += f.x;
            s[2 * i + 1] += f.y;
        }
    }
};
template <int N> struct Words { typedef uint4 type; };
template <> struct Words<2> { typedef uint2 type; };
// N neighbouring results, times scale, rounded once; add: onto what is there
template <int GT, int N>
__device__ __forceinline__ void write_sums(void *out, size_t at, const float (&s)[N], float scale, bool add)
{
    float v[N];
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = s[i] * scale;
    if constexpr (GT == SFB_F32) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            float4 *p = (float4 *)((float *)out + at + i);
            float4 o = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            if (add) {
                const float4 u = *p;
                o.x += u.x; o.y += u.y; o.z += u.z; o.w += u.w;
            }
            __stcs(p, o);
        }
    } else {
        typedef typename Words<N / 2>::type W;
        W *p = (W *)((uint16_t *)out + at);
        __align__(16) uint32_t w[N / 2];
        if (add) *(W *)w = *p;
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            float x = v[2 * i], y = v[2 * i + 1];
            if constexpr (GT == SFB_BF16) {
                if (add) {
                    x += __uint_as_float(w[i] << 16);
                    y += __uint_as_float(w[i] & 0xffff0000u);
                }
                const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                if (add) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                    x += f.x;
                    y += f.y;
                }
                const __half2 h = __floats2half2_rn(x, y);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        __stcs(p, *(const W *)w);
    }
}

// A warp takes `piece` sorted tokens and 32 lanes' columns.  Four tokens' loads are on their way together: what ends a run stands there as
// often, and with eight of them registers and code made the whole call slower (32768 x 1024 fp16 58 -> 45 us).  fp32: five CTAs per
// SM (32768 x 768 76 -> 65; 16-bit types spill then, 53 -> 62).
template <int DT, int GT>
__global__ void __launch_bounds__(256, DT == SFB_F32 ? 5 : 1) table_grad_kernel(const GradArgs a)
{
    constexpr int N = Piece<DT>::N, U = 4;
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t groups = (a.hidden / N + 31) / 32, y = blockIdx.x / groups, col = ((blockIdx.x - y * groups) * 32 + lane) * N;
    const bool live = col < a.hidden;
    const uint32_t c = y * 8 + warp, total = a.starts[a.vocab];
    const uint32_t i0 = c * a.piece, i1 = min(total, i0 + a.piece);
    if (i0 >= total) return;
    const int before = i0 ? a.sorted[i0 - 1].y : -1, after = i1 < total ? a.sorted[i1].y : -1;
    float s[N] = {};
    int cur = -1;
    bool opened = false;                             // the current run began before this piece
    auto flush = [&](bool goes_on) {
        if (cur < 0 || !live) return;
        if (!opened && !goes_on) {
            write_sums<GT, N>(a.dtable, (size_t)cur * a.hidden + col, s, a.scale, a.accumulate);
        } else {
            float *p = a.parts + ((size_t)c * 2 + (opened ? 0 : 1)) * a.hidden + col;
#pragma unroll
            for (int i = 0; i < N; i += 4) *(float4 *)(p + i) = make_float4(s[i], s[i + 1], s[i + 2], s[i + 3]);
        }
    };
    for (uint32_t g = i0; g < i1; g += 32) {
        const int2 e = g + lane < i1 ? a.sorted[g + lane] : make_int2(0, -1);
        const uint32_t here = min(32u, i1 - g);
        for (uint32_t j = 0; j < here; j += U) {
            uint4 u[U];
#pragma unroll
            for (int k = 0; k < U; k++) {
                const uint32_t pos = (uint32_t)__shfl_sync(0xffffffffu, e.x, (j + k) & 31);
                u[k] = make_uint4(0u, 0u, 0u, 0u);
                if (live && j + k < here) u[k] = __ldg((const uint4 *)((const typename Elem<DT>::type *)a.dout + (size_t)pos * a.hidden + col));
            }
#pragma unroll
            for (int k = 0; k < U; k++) {
                const int id = __shfl_sync(0xffffffffu, e.y, (j + k) & 31);
                if (j + k < here) {
                    if (id != cur) {
                        flush(false);
                        opened = cur < 0 && id == before;
                        cur = id;
#pragma unroll
                        for (int i = 0; i < N; i++) s[i] = 0.f;
                    }
                    Piece<DT>::add(s, u[k]);
                }
            }
        }
    }
    flush(cur == after);
}

// The runs that more than one piece has.  A warp looks at the end of a piece for a run that begins in it and goes on, and adds up its parts; those
// of a long one are shared by the CTA's warps.
constexpr uint32_t kAlone = 16;                      // parts that a warp adds up by itself
template <int GT>
__global__ void __launch_bounds__(256) join_kernel(const GradArgs a)
{
    __shared__ float4 share[8][32];
    __shared__ uint32_t long_id[8], long_parts[8];
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t groups = (a.hidden / 4 + 31) / 32, y = blockIdx.x / groups, col = ((blockIdx.x - y * groups) * 32 + lane) * 4;
    const bool live = col < a.hidden;
    const uint32_t c = y * 8 + warp, total = a.starts[a.vocab];
    const uint64_t end = (uint64_t)(c + 1) * a.piece;
    // part 0 is this piece's second slot, part k the first slot of piece c + k
    auto sum = [&](uint32_t c0, uint32_t k0, uint32_t k1) {
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live) {
#pragma unroll 8
            for (uint32_t k = k0; k < k1; k++) {
                const float4 u = *(const float4 *)(a.parts + ((size_t)(c0 + k) * 2 + (k ? 0 : 1)) * a.hidden + col);
                s.x += u.x; s.y += u.y; s.z += u.z; s.w += u.w;
            }
        }
        return s;
    };
    auto write = [&](uint32_t id, const float4 &s) {
        const float v[4] = {s.x, s.y, s.z, s.w};
        if (live) write_sums<GT, 4>(a.dtable, (size_t)id * a.hidden + col, v, a.scale, a.accumulate);
    };
    uint32_t parts = 0, id = 0;
    if (end < total) {
        id = (uint32_t)a.sorted[end - 1].y;
        const uint32_t next = (uint32_t)a.sorted[end].y, first = a.starts[id], last = a.starts[id + 1];
        if (next == id && first >= c * a.piece) parts = 1 + (uint32_t)((last - end + a.piece - 1) / a.piece);
    }
    if (parts && parts <= kAlone) write(id, sum(c, 0, parts));
    if (lane == 0) {
        long_id[warp] = id;
        long_parts[warp] = parts > kAlone ? parts : 0;
    }
    __syncthreads();
    for (uint32_t w = 0; w < 8; w++) {
        const uint32_t n = long_parts[w];
        if (!n) continue;
        const uint32_t per = (n + 7) / 8, k0 = min(n, warp * per);
        float4 s = sum(y * 8 + w, k0, min(n, k0 + per));
        share[warp][lane] = s;
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (int k = 1; k < 8; k++) {
                const float4 u = share[k][lane];
                s.x += u.x; s.y += u.y; s.z += u.z; s.w += u.w;
            }
            write(long_id[w], s);
        }
        __syncthreads();
    }
}

// dpos: a warp has 32 lanes' columns of one position and a share of the batch (`ways` warps per position, whose shares meet in shared memory)
template <int DT, int GT>
__device__ __forceinline__ void add_positions(const GradArgs &a, uint32_t cta, float *share)      // share: [kSortWarps][N][33]
{
    constexpr int N = Piece<DT>::N;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ways = a.ways, part = warp % ways;
    const uint32_t groups = (a.hidden / N + 31) / 32, y = cta / groups, col = ((cta - y * groups) * 32 + lane) * N, l = y * (kSortWarps / ways) + warp / ways;
    const bool live = col < a.hidden && l < a.len;
    const uint32_t per = (a.batch + ways - 1) / ways, b0 = min(a.batch, part * per), b1 = min(a.batch, b0 + per);
    float s[N] = {};
    if (live) {
        const typename Elem<DT>::type *src = (const typename Elem<DT>::type *)a.dout + (size_t)l * a.hidden + col;
        const size_t step = (size_t)a.len * a.hidden;
        uint32_t b = b0;
        for (; b + 8 <= b1; b += 8) {
            uint4 u[8];
#pragma unroll
            for (int k = 0; k < 8; k++) u[k] = __ldg((const uint4 *)(src + (b + k) * step));
#pragma unroll
            for (int k = 0; k < 8; k++) Piece<DT>::add(s, u[k]);
        }
        for (; b < b1; b++) Piece<DT>::add(s, __ldg((const uint4 *)(src + b * step)));
    }
    if (ways > 1) {
#pragma unroll
        for (int i = 0; i < N; i++) share[(warp * N + i) * 33 + lane] = s[i];
        __syncthreads();
        if (part) return;
        for (uint32_t w = 1; w < ways; w++)
#pragma unroll
            for (int i = 0; i < N; i++) s[i] += share[((warp + w) * N + i) * 33 + lane];
    }
    if (live) write_sums<GT, N>(a.dpos, (size_t)l * a.hidden + col, s, 1.f, a.accumulate);
}

// The first CTAs sort, the others add up positions or write zeros: one waits for latencies while the others move data.
template <int DT, int GT>
__global__ void __launch_bounds__(kSortThreads) sort_and_positions_kernel(const GradArgs a)
{
    extern __shared__ __align__(16) uint32_t dynamic[];
    grid_dependency_wait();
    grid_launch_dependents();
    if (blockIdx.x < a.sorters) {
        sort_ids(a, dynamic);
        return;
    }
    const uint32_t y = blockIdx.x - a.sorters, both = 2 * min(a.pos_ctas, a.fillers), at = y < both ? y >> 1 : y - both / 2;
    if (y < both ? y & 1 : a.fillers > a.pos_ctas) {
        const size_t pieces = (size_t)a.vocab * a.hidden * sizeof(typename Elem<GT>::type) / 16, i0 = (size_t)at * kFill;
        uint4 *out = (uint4 *)a.dtable + i0;
        const uint32_t n = (uint32_t)(pieces - i0 < kFill ? pieces - i0 : kFill);
#pragma unroll 8
        for (uint32_t i = threadIdx.x; i < n; i += kSortThreads) __stcs(out + i, make_uint4(0u, 0u, 0u, 0u));
    } else {
        add_positions<DT, GT>(a, at, (float *)dynamic);
    }
}

// ---- few tokens: one launch ------------------------------------------------------------------------------------------------------------
// A CTA per token and 32 lanes' columns: where an earlier token has the same id there is nothing to do, otherwise its warps look for the id among
// shares of the tokens from there on and add up what they find, and their sums meet in shared memory.  Beside them the positions' sums, and CTAs that
// write zeros to ranges of rows, all but those whose id they find among the tokens.  Every CTA reads all ids, 4 bytes each from L2.  Most CTAs only find
// that they have nothing to do, so as many as possible are on an SM: 32 registers and two tokens' loads at once (us, 52 registers and eight / 32 and four
// / 32 and two: 320 tokens x 768 fp32 22.6 / 19.4 / 19.2, 320 x 2048 fp16 9.5 / 7.1 / 6.6; 320 times the same id 6.4 / 7.1 / 7.7).  Zeros and tokens
// in turn instead of the tokens first: 24.7.
template <int DT, int GT>
__global__ void __launch_bounds__(kSortThreads, 4) few_tokens_kernel(const GradArgs a, uint32_t token_ctas, uint32_t rows)
{
    constexpr int N = Piece<DT>::N, U = 2;
    extern __shared__ __align__(16) uint32_t dynamic[];
    __shared__ uint32_t any[kSortWarps];
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (blockIdx.x >= token_ctas) {
        const uint32_t y = blockIdx.x - token_ctas, both = 2 * min(a.pos_ctas, a.fillers), at = y < both ? y >> 1 : y - both / 2;
        if (!(y < both ? y & 1 : a.fillers > a.pos_ctas)) {
            add_positions<DT, GT>(a, at, (float *)dynamic);
            return;
        }
        uint8_t *found = (uint8_t *)dynamic;
        const uint32_t v0 = at * rows, n = min(rows, a.vocab - v0), per = (uint32_t)(a.hidden * sizeof(typename Elem<GT>::type) / 16);      // 16-byte pieces per row
        for (uint32_t i = threadIdx.x; i < n; i += kSortThreads) found[i] = 0;
        __syncthreads();
        int here = 0;
        for (uint32_t i = threadIdx.x; i < a.n; i += kSortThreads) {
            const uint32_t v = (uint32_t)__ldg(a.ids + i) - v0;
            if (v < n) {
                found[v] = 1;
                here = 1;
            }
        }
        here = __syncthreads_or(here);
        uint4 *out = (uint4 *)a.dtable + (size_t)v0 * per;
        const uint32_t pieces = n * per;
        if (!here) {
#pragma unroll 8
            for (uint32_t i = threadIdx.x; i < pieces; i += kSortThreads) __stcs(out + i, make_uint4(0u, 0u, 0u, 0u));
        } else {
            uint32_t r = threadIdx.x / per, c = threadIdx.x % per;
            const uint32_t dr = kSortThreads / per, dc = kSortThreads % per;
            for (uint32_t i = threadIdx.x; i < pieces; i += kSortThreads) {
                if (!found[r]) __stcs(out + i, make_uint4(0u, 0u, 0u, 0u));
                r += dr;
                c += dc;
                if (c >= per) {
                    c -= per;
                    r++;
                }
            }
        }
        return;
    }
    const uint32_t groups = (a.hidden / N + 31) / 32, t = blockIdx.x / groups, col = ((blockIdx.x - t * groups) * 32 + lane) * N;
    const bool live = col < a.hidden;
    const int32_t id = __ldg(a.ids + t);
    if (blockIdx.x == 0 && a.bad) {
        uint32_t bad = 0;
        for (uint32_t i0 = 0; i0 < a.n; i0 += kSortThreads) bad += __syncthreads_count(i0 + threadIdx.x < a.n && (uint32_t)__ldg(a.ids + min(i0 + threadIdx.x, a.n - 1)) >= a.vocab);
        if (threadIdx.x == 0) *a.bad = bad;
    }
    if ((uint32_t)id >= a.vocab) return;
    int earlier = 0;
    for (uint32_t i = threadIdx.x; i < t; i += kSortThreads) earlier |= __ldg(a.ids + i) == id;
    if (__syncthreads_or(earlier)) return;
    const uint32_t share = ((a.n - t + kSortWarps - 1) / kSortWarps + 31) / 32 * 32, i0 = min(a.n, t + warp * share), i1 = min(a.n, i0 + share);
    float s[N] = {};
    uint32_t mine = 0;
    for (uint32_t i = i0; i < i1; i += 32) {
        uint32_t todo = __ballot_sync(0xffffffffu, i + lane < i1 && __ldg(a.ids + min(i + lane, a.n - 1)) == id);
        mine |= todo;
        while (todo) {
            uint4 u[U];
#pragma unroll
            for (int k = 0; k < U; k++) {
                u[k] = make_uint4(0u, 0u, 0u, 0u);
                if (todo) {
                    if (live) u[k] = __ldg((const uint4 *)((const typename Elem<DT>::type *)a.dout + (size_t)(i + __ffs(todo) - 1) * a.hidden + col));
                    todo &= todo - 1;
                }
            }
#pragma unroll
            for (int k = 0; k < U; k++) Piece<DT>::add(s, u[k]);
        }
    }
    float *part = (float *)dynamic;                          // [warp][N][33]
    if (mine && warp) {
#pragma unroll
        for (int i = 0; i < N; i++) part[(warp * N + i) * 33 + lane] = s[i];
    }
    if (lane == 0) any[warp] = mine;
    __syncthreads();
    if (warp) return;
    for (uint32_t w = 1; w < kSortWarps; w++)
        if (any[w])
#pragma unroll
            for (int i = 0; i < N; i++) s[i] += part[(w * N + i) * 33 + lane];
    if (live) write_sums<GT, N>(a.dtable, (size_t)id * a.hidden + col, s, a.scale, a.accumulate);
}

// Sorted tokens per piece: as many as leave 3000 warps with 32 lanes' columns of a piece each, so that long runs have few parts (us, pieces of 8 / 16 /
// 32 / 64 tokens: 32768 x 1024 fp16 55 / 49 / 45, 8192 x 512 fp32 17.6 / 19.3 / 21.8); from 8 to 64 (262144 x 768 fp16, 32 / 64 / 128: 245 / 240 / 257).
static uint32_t piece_length(uint32_t n, uint32_t hidden)
{
    uint32_t len = 64;
    while (len > 8 && (uint64_t)n / len * ((hidden + 255) / 256) < 3000) len /= 2;
    return len;
}
static uint64_t padded(uint64_t bytes) { return (bytes + 63) / 64 * 64; }
static uint32_t piece_count(uint32_t n, uint32_t hidden) { return (uint32_t)(((uint64_t)n + piece_length(n, hidden) - 1) / piece_length(n, hidden)); }

template <int DT, int GT>
static int launch(cudaStream_t s, GradArgs a)
{
    const int dev = current_device(), sms = device_sm_count(dev);
    if (sms <= 0) return fail("sfb_embedding_grad: cannot query the device");
    constexpr uint32_t N = Piece<DT>::N;
    const uint64_t groups = (a.hidden / N + 31) / 32;
    SFB_REQUIRE(groups * a.len < (1ull << 31) && groups * ((a.pieces + 7) / 8) < (1ull << 31) && (uint64_t)((a.hidden / 4 + 31) / 32) * a.pieces < (1ull << 31),
                "sfb_embedding_grad: too many rows for one launch");
    // positions enough to fill the SMs: a warp each; otherwise several share the batch of one
    uint64_t pos_ctas = 0, fillers = 0;
    if (a.dpos) {
        const uint64_t warps = groups * a.len, want = 16ull * sms;
        a.ways = 1;
        while (a.ways < kSortWarps && warps * a.ways < want && a.batch >= 16 * a.ways) a.ways *= 2;
        pos_ctas = groups * ((a.len + kSortWarps / a.ways - 1) / (kSortWarps / a.ways));
    }
    // Few tokens (graphs of calls, us, three launches / one: 64 tokens x 256 bf16, vocabulary 1000 11.3 / 4.0, 2048 tokens 14.9 / 8.4; 426 x 768 fp32, 30522
    // 22.0 / 20.7; 426 x 2048 fp16, 3408 CTAs 10.7 / 10.2 with eight loads at once; 768 x 768 fp32, 4608 CTAs 23 / 28).
    if (a.n <= kFew && groups * a.n <= kFewCtas) {
        const uint64_t row = (uint64_t)a.hidden * sizeof(typename Elem<GT>::type);
        const uint32_t rows = (uint32_t)(row < 16 * kFill ? 16 * kFill / row : 1);
        a.fillers = a.accumulate ? 0 : (a.vocab + rows - 1) / rows;
        a.pos_ctas = (uint32_t)pos_ctas;
        const uint64_t ctas = groups * a.n + pos_ctas + a.fillers;
        SFB_REQUIRE(ctas < (1ull << 31), "sfb_embedding_grad: too many rows for one launch");
        const size_t sums = sizeof(float) * kSortWarps * N * 33;
        launch_overlapped(few_tokens_kernel<DT, GT>, dim3((unsigned)ctas), dim3(kSortThreads), rows > sums ? rows : sums, s, a, (uint32_t)(groups * a.n), rows);
        return check_launch("sfb_embedding_grad");
    }
    // All rows are zeroed beside the sorting, and those of tokens that do occur are written again (30522 x 768, us: zeroed after the sorting, by its
    // counts, bf16 1024 tokens 43, 32768 60, fp32 1024 tokens 28; beside it 31, 53 and 24).
    if (!a.accumulate) fillers = ((uint64_t)a.vocab * a.hidden * sizeof(typename Elem<GT>::type) / 16 + kFill - 1) / kFill;
    SFB_REQUIRE(a.sorters + pos_ctas + fillers < (1ull << 31), "sfb_embedding_grad: too many rows for one launch");
    a.pos_ctas = (uint32_t)pos_ctas;
    a.fillers = (uint32_t)fillers;
    const uint64_t rows = (a.pieces + 7) / 8;
    size_t smem = (size_t)a.range * kStride * 4;
    if (a.dpos && a.ways > 1 && smem < sizeof(float) * kSortWarps * N * 33) smem = sizeof(float) * kSortWarps * N * 33;
    static DeviceOnce once;
    if (!once.done(dev)) {
        if (cudaFuncSetAttribute(sort_and_positions_kernel<DT, GT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kMaxRange * kStride * 4)) != cudaSuccess)
            return fail("sfb_embedding_grad: cannot reserve shared memory");
        once.mark(dev);
    }
    launch_overlapped(sort_and_positions_kernel<DT, GT>, dim3((unsigned)(a.sorters + pos_ctas + fillers)), dim3(kSortThreads), smem, s, a);
    launch_overlapped(table_grad_kernel<DT, GT>, dim3((unsigned)(groups * rows)), dim3(256), 0, s, a);
    if (a.pieces > 1) launch_overlapped(join_kernel<GT>, dim3((a.hidden / 4 + 31) / 32 * ((a.pieces - 1 + 7) / 8)), dim3(256), 0, s, a);
    return check_launch("sfb_embedding_grad");
}

}  // namespace emb
}  // namespace sfb

using namespace sfb;

extern "C" uint64_t sfb_embedding_grad_workspace(uint32_t batch, uint32_t seq_len, uint32_t hidden, uint32_t vocab)
{
    using namespace emb;
    const uint64_t n = (uint64_t)batch * seq_len;
    if (n >= (1ull << 31)) return 0;
    return 2 * padded(n * 8) + padded(((uint64_t)vocab + 1) * 4) + (uint64_t)piece_count((uint32_t)n, hidden) * 2 * hidden * 4;
}

extern "C" int sfb_embedding_grad(sfb_stream_t stream, void *dtable, void *dpos, const void *dout, const int32_t *ids, uint32_t batch,
                                  uint32_t seq_len, uint32_t hidden, uint32_t vocab, int dtype, int grad_dtype, float scale, int accumulate,
                                  uint32_t *bad_ids, void *workspace)
{
    using namespace emb;
    const char *who = "sfb_embedding_grad";
    SFB_REQUIRE(dtable, "%s: NULL pointer", who);
    SFB_REQUIRE(valid_dtype(dtype) && (grad_dtype == dtype || grad_dtype == SFB_F32), "%s: unknown dtype, or gradients neither fp32 nor of dout's type", who);
    SFB_REQUIRE(hidden >= 8 && hidden % 8 == 0, "%s: hidden=%u must be a multiple of 8", who, hidden);
    SFB_REQUIRE(vocab >= 1 && vocab <= (1u << 27), "%s: vocab=%u must be 1 to 2^27", who, vocab);
    SFB_REQUIRE((((uintptr_t)dtable | (uintptr_t)dpos | (uintptr_t)dout | (uintptr_t)workspace) & 15) == 0, "%s: dtable, dpos, dout and workspace must be 16-byte aligned", who);
    const uint64_t n = (uint64_t)batch * seq_len;
    SFB_REQUIRE(n < (1ull << 31), "%s: too many tokens", who);
    SFB_REQUIRE(n == 0 || (dout && ids && workspace), "%s: NULL pointer", who);
    cudaStream_t s = as_stream(stream);
    if (n == 0) {
        const size_t row = (size_t)hidden * elem_size(grad_dtype);
        cudaError_t e = bad_ids ? cudaMemsetAsync(bad_ids, 0, 4, s) : cudaSuccess;
        if (e == cudaSuccess && !accumulate) e = cudaMemsetAsync(dtable, 0, vocab * row, s);
        if (e == cudaSuccess && !accumulate && dpos && seq_len) e = cudaMemsetAsync(dpos, 0, seq_len * row, s);
        if (e != cudaSuccess) return fail("%s: %s", who, cudaGetErrorString(e));
        clear_error();
        return 0;
    }
    GradArgs a = {dout, ids, dtable, dpos, (uint32_t)n, batch, seq_len, hidden, vocab, 0, 0, 0, 0, 1, piece_length((uint32_t)n, hidden), piece_count((uint32_t)n, hidden), scale, accumulate, bad_ids};
    // a CTA per SM sorts, more where its counters would not fit
    const int sms = device_sm_count(current_device());
    const uint32_t ctas = max((uint32_t)(sms > 0 ? sms : 1), (vocab + kMaxRange - 1) / kMaxRange);
    a.range = (vocab + ctas - 1) / ctas;
    a.sorters = (vocab + a.range - 1) / a.range;
    char *w = (char *)workspace;
    a.sorted = (int2 *)w;
    a.unsorted = (int2 *)(w += padded(n * 8));
    a.starts = (uint32_t *)(w += padded(n * 8));
    a.parts = (float *)(w + padded(((uint64_t)vocab + 1) * 4));
    if (dtype == SFB_F32) return launch<SFB_F32, SFB_F32>(s, a);
    if (dtype == SFB_BF16) return grad_dtype == SFB_F32 ? launch<SFB_BF16, SFB_F32>(s, a) : launch<SFB_BF16, SFB_BF16>(s, a);
    return grad_dtype == SFB_F32 ? launch<SFB_F16, SFB_F32>(s, a) : launch<SFB_F16, SFB_F16>(s, a);
}
