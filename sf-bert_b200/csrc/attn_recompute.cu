// The backward pass of the block-sparse attention from the rows' log-sums (sfb_attention_backward_recompute): nothing of the size of the
// scores is kept from the forward pass.  With x = scale Q.K^T on the kept elements and lse the log of a row's sum of exp(x),
//   P = exp(x - lse),  delta = rowsum(dO * O),  dS = P * (dO.V^T - delta) * scale,  dQ = dS.K,  dK = dS^T.Q,  dV = P^T.dO.
// Here are the rows' constants for every path, and the path of fp32 operands and of every shape that the tcgen05 kernels
// (attn_tc_recompute.cu) do not take.  That one makes P and dS of some (batch, head) pairs at a time in the caller's workspace, in the
// operands' type, and multiplies them by the products of attn_simt.cu: five products per block.  Two kernels that keep both on
// chip, one by rows and one by columns, would make two of them twice, and at fp32 precision a product costs more than a block's
// way through L2.
#include "recompute.cuh"
#include "simt_tile.cuh"

namespace sfb {

// ---- the rows' constants: neg_lse = -lse log2(e), neg_delta = -scale rowsum(dO * O), both [B, H, L] ------------------------------
// Eight lanes per row, 32 R rows of one (batch, head) per CTA; R = 4 where that leaves the SMs enough CTAs: a lane's loads of four rows are on their way
// together.  100 MB of O and dO (8 x 4096 rows of 12 heads of 64): 25 us with cold caches, most of a copy's rate.  A row without kept
// elements has lse = -inf, and P = 0 of it: exp2(x + neg_lse) with neg_lse = -inf too.
template <int DT, uint32_t R>
__global__ void __launch_bounds__(256) row_constants_kernel(const void *__restrict__ O, const void *__restrict__ dO, const float *__restrict__ lse,
                                                           float *__restrict__ neg_lse, float *__restrict__ neg_delta, uint32_t L, uint32_t H, uint32_t d,
                                                           size_t o_pitch, size_t do_pitch, float scale, bool vec)
{
    grid_dependency_wait();
    grid_launch_dependents();
    // the heads of the same positions side by side: they lie in the same rows of memory
    const uint32_t b = blockIdx.y, chunk = blockIdx.x / H, h = blockIdx.x - chunk * H, l0 = chunk * 32 * R + threadIdx.x / 8, part = threadIdx.x & 7;
    float sum[R] = {};
    if (vec) {
        constexpr uint32_t N = DT == SFB_F32 ? 4 : 8;
        for (uint32_t c = part * N; c < d; c += 8 * N) {
            uint4 x[R], y[R];
#pragma unroll
            for (uint32_t k = 0; k < R; k++) {
                const uint32_t l = l0 + 32 * k;
                x[k] = y[k] = make_uint4(0u, 0u, 0u, 0u);
                if (l < L) {
                    x[k] = __ldg((const uint4 *)((const typename Elem<DT>::type *)O + ((size_t)b * L + l) * o_pitch + (size_t)h * d + c));
                    y[k] = __ldg((const uint4 *)((const typename Elem<DT>::type *)dO + ((size_t)b * L + l) * do_pitch + (size_t)h * d + c));
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < R; k++) {
                const uint32_t xw[4] = {x[k].x, x[k].y, x[k].z, x[k].w}, yw[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (DT == SFB_F32) {
                        sum[k] = fmaf(__uint_as_float(xw[i]), __uint_as_float(yw[i]), sum[k]);
                    } else {
                        float x0, x1, y0, y1;
                        tile::widen2<DT>(x0, x1, xw[i]);
                        tile::widen2<DT>(y0, y1, yw[i]);
                        sum[k] = fmaf(x0, y0, fmaf(x1, y1, sum[k]));
                    }
                }
            }
        }
    } else {
#pragma unroll
        for (uint32_t k = 0; k < R; k++) {
            const uint32_t l = l0 + 32 * k;
            if (l < L)
                for (uint32_t c = part; c < d; c += 8)
                    sum[k] = fmaf(Elem<DT>::load(O, ((size_t)b * L + l) * o_pitch + (size_t)h * d + c), Elem<DT>::load(dO, ((size_t)b * L + l) * do_pitch + (size_t)h * d + c), sum[k]);
        }
    }
#pragma unroll
    for (uint32_t k = 0; k < R; k++)
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
#pragma unroll
    for (uint32_t k = 0; k < R; k++) {
        const uint32_t l = l0 + 32 * k;
        if (part != k || l >= L) continue;
        const size_t row = ((size_t)b * H + h) * L + l;
        const float s = lse[row];
        // nothing kept (-inf): the row's dS is empty whatever dO and O hold
        neg_lse[row] = s == -INFINITY ? s : s * -1.4426950408889634f;
        neg_delta[row] = s == -INFINITY ? 0.f : sum[k] * -scale;
    }
}

int attention_row_constants(cudaStream_t s, const void *o, const void *dout, const float *lse, float *neg_lse, float *neg_delta, int dtype, uint32_t B,
                            uint32_t L, uint32_t H, uint32_t d, uint64_t o_pitch, uint64_t do_pitch, float scale)
{
    const uint32_t per = dtype == SFB_F32 ? 4 : 8;
    const bool vec = (((uintptr_t)o | (uintptr_t)dout) & 15) == 0 && o_pitch % per == 0 && do_pitch % per == 0 && d % per == 0;
    const int sms = device_sm_count(current_device());
    const uint32_t R = (uint64_t)L * H * B >= 128ull * 8 * (uint64_t)(sms > 0 ? sms : 1) ? 4 : 1;
    const uint64_t chunks = ((uint64_t)L + 32 * R - 1) / (32 * R);
    SFB_REQUIRE(chunks * H < (1ull << 31), "sfb_attention_backward_recompute: too many rows for one launch");
    const dim3 grid((unsigned)(chunks * H), B);
#define RC_LAUNCH_R(DT, RV) launch_overlapped_few(row_constants_kernel<DT, RV>, grid, dim3(256), 0, s, o, dout, lse, neg_lse, neg_delta, L, H, d, (size_t)o_pitch, (size_t)do_pitch, scale, vec)
#define RC_LAUNCH(DT) { if (R == 4) RC_LAUNCH_R(DT, 4); else RC_LAUNCH_R(DT, 1); }
    if (dtype == SFB_F32) RC_LAUNCH(SFB_F32)
    else if (dtype == SFB_BF16) RC_LAUNCH(SFB_BF16)
    else RC_LAUNCH(SFB_F16)
#undef RC_LAUNCH
#undef RC_LAUNCH_R
    return check_launch("sfb_attention_backward_recompute");
}

// ---- P and dS of one block per CTA (64) or warp (32) --------------------------------------------------------------------------------
struct BlockArgs {
    const uint2 *nt_lut;
    const void *q, *k, *v, *dout, *mask;
    const float *neg_lse, *neg_delta;
    void *p, *ds;
    size_t in_pitch, do_pitch;
    uint32_t first, H, d, nb, blocks, lut_stride, mask_stride;        // first: (batch, head) pair of blockIdx.y = 0
    float scale, scale_log2e;
    bool vec;
};
template <int BS> struct BlockCfg {
    static constexpr int TEAMS = BS == 32 ? 4 : 2, TT = 128 / TEAMS;      // teams that stage keys of their own
    static constexpr uint32_t buf = 32 * tile::kStride;
    static constexpr size_t bytes = sizeof(float) * 2 * TEAMS * buf;
    static_assert(TEAMS * 2 * buf / 4 >= tile::kAgainFloats, "a warp's share holds the tiles of blocks_again");
};
// A warp's 32x32 tile again by plain FMAs: where a score or a product dO.V^T is not finite, of which the split products make NaN.
template <int BS, int DT>
__device__ __noinline__ void blocks_again(float *buf, const BlockArgs &a, size_t rowQ, size_t rowK, size_t rowD, size_t rowC, uint64_t bits, size_t at)
{
    const uint32_t lane = threadIdx.x & 31;
    float x[32], y[32];
    tile::scores_again<DT>(x, buf, a.q, a.k, rowQ, rowK, a.in_pitch, a.d, lane);
    const float nl = a.neg_lse[rowC + lane], nd = a.neg_delta[rowC + lane];
#pragma unroll
    for (int n = 0; n < 32; n++) x[n] = (bits >> n) & 1u ? exp2f(fmaf(x[n], a.scale_log2e, nl)) : 0.f;
    // dO and V have pitches of their own
#pragma unroll
    for (int n = 0; n < 32; n++) y[n] = 0.f;
    tile::Again<32, tile::kAgain> u, w;
    for (uint32_t k = 0; k < a.d; k += tile::kAgain) {
        u.template load<DT>(a.dout, rowD + k, a.do_pitch, a.d - k, lane);
        w.template load<DT>(a.v, rowK + k, a.in_pitch, a.d - k, lane);
        __syncwarp();
        u.template put<1, tile::kAgainRows>(buf, lane);
        w.template put<1, tile::kAgainCols<32>>(buf + tile::kAgain * tile::kAgainRows, lane);
        __syncwarp();
        tile::fma_again<32>(y, buf, buf + tile::kAgain * tile::kAgainRows, lane);
    }
#pragma unroll
    for (int n = 0; n < 32; n++) {
        Elem<DT>::store(a.p, at + (size_t)lane * BS + n, x[n]);
        Elem<DT>::store(a.ds, at + (size_t)lane * BS + n, (bits >> n) & 1u ? x[n] * fmaf(y[n], a.scale, nd) : 0.f);
    }
}
template <int DT>
__device__ __forceinline__ void store_eight(void *out, size_t at, const float (&v)[8])
{
    if constexpr (DT == SFB_F32) {
        *(float4 *)((float *)out + at) = make_float4(v[0], v[1], v[2], v[3]);
        *(float4 *)((float *)out + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == SFB_BF16) {
                __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<uint32_t *>(&h);
            } else {
                __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<uint32_t *>(&h);
            }
        }
        *(uint4 *)((uint16_t *)out + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Both products on the warp tiles of simt_tile.cuh, 32 elements of d at a time: the rows of Q (dO) straight to fragments, a chunk ahead
// in registers, the rows of K (V) through a ring of two chunks per team.  A thread holds eight neighbouring columns of four rows.
// P and dS are rounded to the operands' type, as operands of the products that follow: half a step of 16-bit types, nothing for fp32.
template <int BS, int DT>
__global__ void __launch_bounds__(tile::kThreads, 3) recompute_blocks_kernel(const __grid_constant__ BlockArgs a)
{
    using namespace tile;
    typedef BlockCfg<BS> Cfg;
    constexpr uint32_t PER = BS == 32 ? 4 : 1;               // blocks per CTA
    constexpr int T = kTerms<DT>, TT = Cfg::TT;
    extern __shared__ __align__(16) float sm[];              // [team][2][32 rows]
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t bh = a.first + blockIdx.y, b = bh / a.H, h = bh - b * a.H;
    const uint32_t bid = blockIdx.x * PER + (BS == 32 ? warp : 0);
    if (bid >= a.blocks) return;
    const uint32_t r0 = BS == 64 ? 32 * (warp >> 1) : 0, team = BS == 64 ? warp & 1 : warp, c0 = BS == 64 ? 32 * team : 0;
    const uint32_t rank = BS == 64 ? 32 * (warp >> 1) + lane : lane;
    const uint2 en = a.nt_lut[(size_t)h * a.lut_stride + bid];
    const size_t row = ((size_t)b * a.nb + en.x) * BS + r0, col = ((size_t)b * a.nb + en.y) * BS + c0, head = (size_t)h * a.d;
    const size_t rowQ = row * a.in_pitch + head, rowD = row * a.do_pitch + head, rowK = col * a.in_pitch + head;
    const size_t rowC = ((size_t)bh * a.nb + en.x) * BS + r0;           // of the rows' constants
    float *bufs = sm + team * 2 * Cfg::buf;
    const uint32_t chunks = (a.d + kChunk - 1) / kChunk;

    auto product = [&](float (&acc)[2][4][4], const void *A, size_t rowA, size_t pitchA, const void *B, size_t rowB) {
        Staged<DT, TT, (int)kChunk> held_b;
        Raw4<DT> held_a[8];                                  // [16-element half of the chunk][row 16 m + 8 half + g]
        auto load_a = [&](uint32_t c) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t k = c * kChunk + 16 * (i >> 2) + 4 * t;
                load_raw4<DT>(held_a[i], A, rowA + (size_t)(8 * (i & 3) + g) * pitchA + k, k < a.d ? a.d - k : 0u, a.vec);
            }
        };
        auto issue = [&](uint32_t c) {
            stage_begin(held_b, rank, bufs + (c & 1) * Cfg::buf, kStride, B, rowB + c * kChunk, a.in_pitch, a.d - c * kChunk, a.vec);
            cp_commit();
        };
        issue(0);
        load_a(0);
        stage_end(held_b, rank, bufs, kStride, a.vec);
        for (uint32_t c = 0; c < chunks; c++) {
            cp_wait<0>();
            meet<TT>(1 + team);
            if (c + 1 < chunks) issue(c + 1);
            Frag<T> fa[2][2];
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    float x0[4], x1[4];
                    widen4<DT>(x0, held_a[4 * k + 2 * m]);
                    widen4<DT>(x1, held_a[4 * k + 2 * m + 1]);
                    split_rows<T>(fa[k][m], x0, x1);
                }
            if (c + 1 < chunks) load_a(c + 1);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                Four<T> fb[4];
                load_keys<T, true>(fb, bufs + (c & 1) * Cfg::buf, 16 * k, g, t);
#pragma unroll
                for (int m = 0; m < 2; m++) mma16<4, T, T>(acc[m], fa[k][m], fb);
            }
            if (c + 1 < chunks) stage_end(held_b, rank, bufs + ((c + 1) & 1) * Cfg::buf, kStride, a.vec);
        }
    };
    float x[2][4][4] = {}, y[2][4][4] = {};
    product(x, a.q, rowQ, a.in_pitch, a.k, rowK);
    meet<TT>(1 + team);                                      // the ring's last chunk has been read
    product(y, a.dout, rowD, a.do_pitch, a.v, rowK);

    const bool odd = T > 1 && !(zero_if_finite<4>(x[1], zero_if_finite<4>(x[0], zero_if_finite<4>(y[1], zero_if_finite<4>(y[0], 0.f)))) == 0.f);
    const size_t baseC = ((size_t)blockIdx.y * a.blocks + bid) * BS * BS + (size_t)r0 * BS + c0;
    auto mask_bits = [&](uint32_t r) -> uint32_t {           // of this warp's 32 columns, row r0 + r
        if (!a.mask) return 0xffffffffu;
        if (BS == 64) return (uint32_t)(__ldg((const unsigned long long *)a.mask + (size_t)h * a.mask_stride + (size_t)bid * BS + r0 + r) >> c0);
        return __ldg((const uint32_t *)a.mask + (size_t)h * a.mask_stride + (size_t)bid * BS + r);
    };
    // on the team's shared memory, when its other warp is past the products too
    if (T > 1 && (BS == 64 ? __syncthreads_or(odd) : __any_sync(0xffffffffu, odd)) && __any_sync(0xffffffffu, odd)) {
        blocks_again<BS, DT>(sm + warp * (Cfg::TEAMS * 2 * Cfg::buf / 4), a, rowQ, rowK, rowD, rowC, mask_bits(lane), baseC);
        return;
    }
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t r = 16 * m + 8 * half + g, bits = mask_bits(r) >> (8 * t);
            const float nl = __ldg(a.neg_lse + rowC + r), nd = __ldg(a.neg_delta + rowC + r);
            float p[8], ds[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const bool in = (bits >> k) & 1u;
                p[k] = in ? exp2f(fmaf(x[m][k >> 1][2 * half + (k & 1)], a.scale_log2e, nl)) : 0.f;
                ds[k] = in ? p[k] * fmaf(y[m][k >> 1][2 * half + (k & 1)], a.scale, nd) : 0.f;
            }
            store_eight<DT>(a.p, baseC + (size_t)r * BS + 8 * t, p);
            store_eight<DT>(a.ds, baseC + (size_t)r * BS + 8 * t, ds);
        }
}

// How many (batch, head) pairs go through the workspace at a time: block-rows for every SM to have 32 (us with 8 / 16 / 32, each a share of what
// follows: bf16, blocks of 32, d 64, 4 x 12 heads of 2048 positions, strided 1119 / 793 / 622; fp16, blocks of 64, d 128 1635 / 1308 / 1307; what L2 could
// have kept of P and dS counts for less than the SMs that have nothing left to do at the end of each launch), as long as P and dS take no more
// than 512 MB; one at least; whole batch elements or a part of one's heads, in parts of about the same size.
constexpr uint64_t kRowsPerSm = 32, kMostSms = 148, kMostBytes = 512ull << 20;
static uint32_t pairs_at_a_time(int dtype, uint32_t bs, uint32_t nb, uint32_t blocks, uint32_t B, uint32_t H)
{
    const uint64_t one = 2ull * blocks * bs * bs * elem_size(dtype), all = (uint64_t)B * H, most = one ? kMostBytes / one : all;
    uint64_t n = (kMostSms * kRowsPerSm + nb - 1) / nb;
    if (n > most) n = most;
    if (n > all) n = all;
    if (n < 1) n = 1;
    if (n >= H) {
        const uint64_t elems = n / H, parts = (B + elems - 1) / elems;
        n = (B + parts - 1) / parts * H;
    }
    return (uint32_t)(n < 65535 ? n : 65535 / H ? 65535 / H * H : 65535);
}
uint64_t simt_backward_workspace(int dtype, uint32_t bs, uint32_t nb, uint32_t blocks, uint32_t B, uint32_t H)
{
    return 2ull * pairs_at_a_time(dtype, bs, nb, blocks, B, H) * blocks * bs * bs * elem_size(dtype);
}

int simt_backward_recompute(cudaStream_t s, const BackwardArgs &a, float *neg_lse, float *neg_delta, void *blocks_ws)
{
    const AttnDims &p = a.p;
    const uint32_t bs = a.bs, per = bs == 32 ? 4 : 1, n = pairs_at_a_time(a.dtype, bs, p.nb_a, p.blocks, p.B, p.H);
    const size_t e = elem_size(a.dtype);
    const uint32_t L = p.nb_a * bs, unit = a.dtype == SFB_F32 ? 4 : 8;
    void *P = blocks_ws, *dS = (char *)blocks_ws + (size_t)n * p.blocks * bs * bs * e;
    BlockArgs k = {(const uint2 *)a.nt_lut, a.q, a.k, a.v, a.dout, a.mask, neg_lse, neg_delta, P, dS, (size_t)a.in_pitch, (size_t)a.do_pitch, 0, p.H, p.d, p.nb_a,
                   p.blocks, a.nt_stride, p.mask_stride, a.scale, a.scale * 1.4426950408889634f, false};
    k.vec = (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.dout) & 15) == 0 && a.in_pitch % unit == 0 && a.do_pitch % unit == 0 && p.d % unit == 0;
    for (uint32_t first = 0; first < p.B * p.H; first += 0) {
        // whole batch elements, or some heads of one
        const uint32_t b = first / p.H, h = first % p.H;
        const uint32_t heads = n >= p.H ? p.H : n < p.H - h ? n : p.H - h, elems = n >= p.H ? (n / p.H < p.B - b ? n / p.H : p.B - b) : 1;
        if (p.blocks) {
            k.first = first;
            const dim3 grid((p.blocks + per - 1) / per, heads * elems);
#define RB_LAUNCH(BS, DT) launch_overlapped_few(recompute_blocks_kernel<BS, DT>, grid, dim3(tile::kThreads), BlockCfg<BS>::bytes, s, k)
            if (bs == 32) {
                if (a.dtype == SFB_F32) RB_LAUNCH(32, SFB_F32);
                else if (a.dtype == SFB_BF16) RB_LAUNCH(32, SFB_BF16);
                else RB_LAUNCH(32, SFB_F16);
            } else {
                if (a.dtype == SFB_F32) RB_LAUNCH(64, SFB_F32);
                else if (a.dtype == SFB_BF16) RB_LAUNCH(64, SFB_BF16);
                else RB_LAUNCH(64, SFB_F16);
            }
#undef RB_LAUNCH
            if (check_launch("sfb_attention_backward_recompute")) return 1;
        }
        auto in = [&](const void *x) { return (const char *)x + (((size_t)b * L) * a.in_pitch + (size_t)h * p.d) * e; };
        auto out = [&](void *x) { return (char *)x + (((size_t)b * L) * a.grad_pitch + (size_t)h * p.d) * e; };
        const char *dout = (const char *)a.dout + (((size_t)b * L) * a.do_pitch + (size_t)h * p.d) * e;
        AttnDims part = p;
        part.B = elems;
        part.H = heads;
        part.out_pitch = a.grad_pitch;
        const uint2 *nn = (const uint2 *)a.nn_lut + (size_t)h * p.lut_stride, *tn = (const uint2 *)a.tn_lut + (size_t)h * p.lut_stride;
        part.in_pitch = a.do_pitch;
        if (simt_spmm_nn(s, tn, P, dout, out(a.dv), a.dtype, a.dtype, bs, part, true)) return 1;
        part.in_pitch = a.in_pitch;
        if (simt_spmm_nn(s, tn, dS, in(a.q), out(a.dk), a.dtype, a.dtype, bs, part, true)) return 1;
        if (simt_spmm_nn(s, nn, dS, in(a.k), out(a.dq), a.dtype, a.dtype, bs, part, false)) return 1;
        first += heads * elems;
    }
    return 0;
}

}  // namespace sfb
