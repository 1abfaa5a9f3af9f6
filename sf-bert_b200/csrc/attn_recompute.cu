// The backward pass of the block-sparse attention from the rows' log-sums (sfb_attention_backward_recompute): nothing of the size of the
// scores is kept from the forward pass.  With x = scale Q.K^T on the kept elements and lse the log of a row's sum of exp(x),
//   P = exp(x - lse),  delta = rowsum(dO * O),  dS = P * (dO.V^T - delta) * scale,  dQ = dS.K,  dK = dS^T.Q,  dV = P^T.dO.
// Here are the rows' constants for every path, and the path of fp32 operands and of every shape that the tcgen05 kernels
// (attn_tc_recompute.cu) do not take.  That one makes P and dS of some (batch, head) pairs at a time in the caller's workspace, 16-bit types as
// operands of the products that follow, fp32 as three bf16 numbers each, and one launch makes the three products from them: five products per
// block.  Two kernels that keep both on chip, one by rows and one by columns, would make two of them twice.
#include "recompute.cuh"
#include "simt_tile.cuh"
#include <initializer_list>

namespace sfb {

// ---- the rows' constants: neg_lse = -lse log2(e), neg_delta = -inside rowsum(dO * O), both [B, H, L] (inside: recompute.cuh) --------
// Eight lanes per row, 32 R rows of one (batch, head) per CTA; R = 4 where that leaves the SMs enough CTAs: a lane's loads of four rows are on their way
// together.  100 MB of O and dO (8 x 4096 rows of 12 heads of 64): 25 us with cold caches, most of a copy's rate.  A row without kept
// elements has lse = -inf, and P = 0 of it: exp2(x + neg_lse) with neg_lse = -inf too.
template <int DT, uint32_t R>
__global__ void __launch_bounds__(256) row_constants_kernel(const void *__restrict__ O, const void *__restrict__ dO, const float *__restrict__ lse,
                                                           float *__restrict__ neg_lse, float *__restrict__ neg_delta, uint32_t L, uint32_t H, uint32_t d,
                                                           size_t o_pitch, size_t do_pitch, float inside, bool vec)
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
        neg_delta[row] = s == -INFINITY ? 0.f : sum[k] * -inside;
    }
}

int attention_row_constants(cudaStream_t s, const void *o, const void *dout, const float *lse, float *neg_lse, float *neg_delta, int dtype, uint32_t B,
                            uint32_t L, uint32_t H, uint32_t d, uint64_t o_pitch, uint64_t do_pitch, float inside)
{
    const uint32_t per = dtype == SFB_F32 ? 4 : 8;
    const bool vec = (((uintptr_t)o | (uintptr_t)dout) & 15) == 0 && o_pitch % per == 0 && do_pitch % per == 0 && d % per == 0;
    const int sms = device_sm_count(current_device());
    const uint32_t R = (uint64_t)L * H * B >= 128ull * 8 * (uint64_t)(sms > 0 ? sms : 1) ? 4 : 1;
    const uint64_t chunks = ((uint64_t)L + 32 * R - 1) / (32 * R);
    SFB_REQUIRE(chunks * H < (1ull << 31), "sfb_attention_backward_recompute: too many rows for one launch");
    const dim3 grid((unsigned)(chunks * H), B);
#define RC_LAUNCH_R(DT, RV) launch_overlapped_few(row_constants_kernel<DT, RV>, grid, dim3(256), 0, s, o, dout, lse, neg_lse, neg_delta, L, H, d, (size_t)o_pitch, (size_t)do_pitch, inside, vec)
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
    float inside, scale_log2e;
};
template <int BS> struct BlockCfg {
    static constexpr int TEAMS = BS == 32 ? 4 : 2, TT = 128 / TEAMS;      // teams that stage keys of their own
    static constexpr uint32_t buf = 32 * tile::kStride;
    static constexpr size_t bytes = sizeof(float) * 2 * TEAMS * buf;
    static_assert(TEAMS * 2 * buf / 4 >= tile::kAgainFloats, "a warp's share holds the tiles of blocks_again");
};
// A warp's 32x32 tile again by plain FMAs: where a score or a product dO.V^T is not finite, of which the split products make NaN.
template <int BS>
__device__ __noinline__ void blocks_again(float *buf, const BlockArgs &a, size_t rowQ, size_t rowK, size_t rowD, size_t rowC, uint64_t bits, size_t at)
{
    const uint32_t lane = threadIdx.x & 31;
    float x[32], y[32];
    tile::scores_again<SFB_F32>(x, buf, a.q, a.k, rowQ, rowK, a.in_pitch, a.d, lane);
    const float nl = a.neg_lse[rowC + lane], nd = a.neg_delta[rowC + lane];
#pragma unroll
    for (int n = 0; n < 32; n++) x[n] = (bits >> n) & 1u ? exp2f(fmaf(x[n], a.scale_log2e, nl)) : 0.f;
    // dO and V have pitches of their own
#pragma unroll
    for (int n = 0; n < 32; n++) y[n] = 0.f;
    tile::Again<32, tile::kAgain> u, w;
    for (uint32_t k = 0; k < a.d; k += tile::kAgain) {
        u.template load<SFB_F32>(a.dout, rowD + k, a.do_pitch, a.d - k, lane);
        w.template load<SFB_F32>(a.v, rowK + k, a.in_pitch, a.d - k, lane);
        __syncwarp();
        u.template put<1, tile::kAgainRows>(buf, lane);
        w.template put<1, tile::kAgainCols<32>>(buf + tile::kAgain * tile::kAgainRows, lane);
        __syncwarp();
        tile::fma_again<32>(y, buf, buf + tile::kAgain * tile::kAgainRows, lane);
    }
#pragma unroll
    for (int n = 0; n < 32; n += 2) {
        const float s0 = (bits >> n) & 1u ? x[n] * fmaf(y[n], a.inside, nd) : 0.f, s1 = (bits >> (n + 1)) & 1u ? x[n + 1] * fmaf(y[n + 1], a.inside, nd) : 0.f;
        uint32_t p[3], ds[3];
        tile::split2<3>(p, x[n], x[n + 1]);
        tile::split2<3>(ds, s0, s1);
#pragma unroll
        for (int i = 0; i < 3; i++) {
            *(uint32_t *)((uint16_t *)a.p + at + (size_t)i * BS * BS + (size_t)lane * BS + n) = p[i];
            *(uint32_t *)((uint16_t *)a.ds + at + (size_t)i * BS * BS + (size_t)lane * BS + n) = ds[i];
        }
    }
}
template <int DT> __device__ __forceinline__ uint32_t pack_own(float a, float b)
{
    if constexpr (DT == SFB_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
// fp32: three bf16 planes, `plane` elements apart, whose sum the values are
template <int DT>
__device__ __forceinline__ void store_eight(void *out, size_t at, uint32_t plane, const float (&v)[8])
{
    if constexpr (DT == SFB_F32) {
        uint32_t w[4][3];
#pragma unroll
        for (int i = 0; i < 4; i++) tile::split2<3>(w[i], v[2 * i], v[2 * i + 1]);
#pragma unroll
        for (int i = 0; i < 3; i++) *(uint4 *)((uint16_t *)out + at + i * plane) = make_uint4(w[0][i], w[1][i], w[2][i], w[3][i]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = pack_own<DT>(v[2 * i], v[2 * i + 1]);
        *(uint4 *)((uint16_t *)out + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Both products on the warp tiles of simt_tile.cuh, 32 elements of d at a time: the rows of Q (dO) straight to fragments, a chunk ahead
// in registers, the rows of K (V) through a ring of two chunks per team.  A thread holds eight neighbouring columns of four rows.
// P and dS leave as three bf16 numbers each, whose sum they are.
template <int BS, bool VEC>
__global__ void __launch_bounds__(tile::kThreads, 3) recompute_blocks_kernel(const __grid_constant__ BlockArgs a)
{
    using namespace tile;
    typedef BlockCfg<BS> Cfg;
    constexpr uint32_t PER = BS == 32 ? 4 : 1;               // blocks per CTA
    constexpr int DT = SFB_F32, T = 3, TT = Cfg::TT;
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
                load_raw4<DT>(held_a[i], A, rowA + (size_t)(8 * (i & 3) + g) * pitchA + k, k < a.d ? a.d - k : 0u, VEC);
            }
        };
        auto issue = [&](uint32_t c) {
            stage_begin(held_b, rank, bufs + (c & 1) * Cfg::buf, kStride, B, rowB + c * kChunk, a.in_pitch, a.d - c * kChunk, VEC);
            cp_commit();
        };
        issue(0);
        load_a(0);
        stage_end(held_b, rank, bufs, kStride, VEC);
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
            if (c + 1 < chunks) stage_end(held_b, rank, bufs + ((c + 1) & 1) * Cfg::buf, kStride, VEC);
        }
    };
    float x[2][4][4] = {}, y[2][4][4] = {};
    product(x, a.q, rowQ, a.in_pitch, a.k, rowK);
    meet<TT>(1 + team);                                      // the ring's last chunk has been read
    product(y, a.dout, rowD, a.do_pitch, a.v, rowK);

    const bool odd = !(zero_if_finite<4>(x[1], zero_if_finite<4>(x[0], zero_if_finite<4>(y[1], zero_if_finite<4>(y[0], 0.f)))) == 0.f);
    const size_t baseC = ((size_t)blockIdx.y * a.blocks + bid) * 3 * BS * BS + (size_t)r0 * BS + c0;
    auto mask_bits = [&](uint32_t r) -> uint32_t {           // of this warp's 32 columns, row r0 + r
        if (!a.mask) return 0xffffffffu;
        if (BS == 64) return (uint32_t)(__ldg((const unsigned long long *)a.mask + (size_t)h * a.mask_stride + (size_t)bid * BS + r0 + r) >> c0);
        return __ldg((const uint32_t *)a.mask + (size_t)h * a.mask_stride + (size_t)bid * BS + r);
    };
    // on the team's shared memory, when its other warp is past the products too
    if ((BS == 64 ? __syncthreads_or(odd) : __any_sync(0xffffffffu, odd)) && __any_sync(0xffffffffu, odd)) {
        blocks_again<BS>(sm + warp * (Cfg::TEAMS * 2 * Cfg::buf / 4), a, rowQ, rowK, rowD, rowC, mask_bits(lane), baseC);
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
                ds[k] = in ? p[k] * fmaf(y[m][k >> 1][2 * half + (k & 1)], a.inside, nd) : 0.f;
            }
            store_eight<DT>(a.p, baseC + (size_t)r * BS + 8 * t, BS * BS, p);
            store_eight<DT>(a.ds, baseC + (size_t)r * BS + 8 * t, BS * BS, ds);
        }
}

// ---- the same for 16-bit operands ---------------------------------------------------------------------------------------------------
// A warp makes a 32x32 tile of both products on the tensor cores in the operands' own type, its fragments straight from memory: lane 4 g + t holds
// elements 8 t to 8 t + 7 of each 32 of a row, 16 bytes, and as long as both operands agree it does not matter which slots of two
// k16 steps these are.  Neighbouring blocks are of the same row, whose Q and dO come from L1 for the CTA's other warps.  A thread's columns of
// a row are eight neighbours (the keys are dealt to the n-tiles that way), 16 bytes to store.
template <int DT> __device__ __forceinline__ void mma_own(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (DT == SFB_F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// eight neighbouring elements, n of which exist
__device__ __forceinline__ uint4 load_eight(const uint16_t *p, uint32_t n, bool vec)
{
    if (vec) return n ? __ldg((const uint4 *)p) : make_uint4(0u, 0u, 0u, 0u);
    uint32_t w[4] = {};
#pragma unroll
    for (uint32_t i = 0; i < 8; i++)
        if (i < n) w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float ex2(float x)           // 2 units of 2^-23, and 0 below 2^-126: P is rounded to 16 bits
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int BS, int DT, bool VEC>
__global__ void __launch_bounds__(tile::kThreads, 4) recompute_blocks16_kernel(const __grid_constant__ BlockArgs a)
{
    constexpr uint32_t PER = BS == 32 ? 4 : 1;               // blocks per CTA
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t bh = a.first + blockIdx.y, b = bh / a.H, h = bh - b * a.H;
    const uint32_t bid = blockIdx.x * PER + (BS == 32 ? warp : 0);
    if (bid >= a.blocks) return;
    const uint32_t r0 = BS == 64 ? 32 * (warp >> 1) : 0, c0 = BS == 64 ? 32 * (warp & 1) : 0;
    const uint2 en = a.nt_lut[(size_t)h * a.lut_stride + bid];
    const size_t row = ((size_t)b * a.nb + en.x) * BS + r0, col = ((size_t)b * a.nb + en.y) * BS + c0, head = (size_t)h * a.d;
    const uint32_t key = 8 * (g >> 1) + (g & 1);             // + 2 j: the key of column g of n-tile j, so that columns 2 t, 2 t + 1 are keys 8 t + 2 j + e

    auto product = [&](float (&acc)[2][4][4], const void *A, size_t pitchA, const void *B) {
        const uint16_t *pa = (const uint16_t *)A + (row + g) * pitchA + head + 8 * t, *pb = (const uint16_t *)B + (col + key) * a.in_pitch + head + 8 * t;
#pragma unroll 2
        for (uint32_t k = 0; k < a.d; k += 32) {
            const uint32_t n = k + 8 * t < a.d ? a.d - k - 8 * t : 0u;
            uint4 x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[i] = load_eight(pa + (size_t)(8 * i) * pitchA + k, n, VEC);
                y[i] = load_eight(pb + (size_t)(2 * i) * a.in_pitch + k, n, VEC);
            }
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    mma_own<DT>(acc[m][j], x[2 * m].x, x[2 * m + 1].x, x[2 * m].y, x[2 * m + 1].y, y[j].x, y[j].y);
                    mma_own<DT>(acc[m][j], x[2 * m].z, x[2 * m + 1].z, x[2 * m].w, x[2 * m + 1].w, y[j].z, y[j].w);
                }
        }
    };
    float x[2][4][4] = {}, y[2][4][4] = {};
    product(x, a.q, a.in_pitch, a.k);
    product(y, a.dout, a.do_pitch, a.v);
    const size_t rowC = ((size_t)bh * a.nb + en.x) * BS + r0;           // of the rows' constants
    const size_t baseC = ((size_t)blockIdx.y * a.blocks + bid) * BS * BS + (size_t)r0 * BS + c0;
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t r = 16 * m + 8 * half + g;
            uint32_t bits = 0xffu;
            if (a.mask) {
                if (BS == 64) bits = (uint32_t)(__ldg((const unsigned long long *)a.mask + (size_t)h * a.mask_stride + (size_t)bid * BS + r0 + r) >> (c0 + 8 * t));
                else bits = __ldg((const uint32_t *)a.mask + (size_t)h * a.mask_stride + (size_t)bid * BS + r) >> (8 * t);
            }
            const float nl = __ldg(a.neg_lse + rowC + r), nd = __ldg(a.neg_delta + rowC + r);
            float p[8], ds[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const bool in = (bits >> k) & 1u;
                p[k] = in ? ex2(fmaf(x[m][k >> 1][2 * half + (k & 1)], a.scale_log2e, nl)) : 0.f;
                ds[k] = in ? p[k] * fmaf(y[m][k >> 1][2 * half + (k & 1)], a.inside, nd) : 0.f;
            }
            store_eight<DT>(a.p, baseC + (size_t)r * BS + 8 * t, 0, p);
            store_eight<DT>(a.ds, baseC + (size_t)r * BS + 8 * t, 0, ds);
        }
}

// ---- the three products with P and dS: dV = P^T.dO, dK = dS^T.Q, dQ = dS.K -------------------------------------------------------------
// A CTA makes one block-row (column) of one of them, all of d: a warp 32 x 32 outputs.  The contraction goes 32 elements at a time through a ring of
// kStages stages of shared memory, brought by cp.async.  P and dS are 16-bit there and become fragments by ldmatrix, transposed or not; so do
// 16-bit operands.  fp32: P and dS are three bf16 planes whose sum they are, split once by the kernel that made them (fp32
// blocks would be split again by every warp, or multiplied by FMAs: 7680 blocks of 32, d 128, the whole backward pass 295 us, 273 so), and a warp
// splits its own columns of the other operand.  Each 32 elements are added up from zero and then to the sum, rounded to
// nearest: the tensor core's additions truncate.  Sums have a fixed order.
struct ProductArgs {
    const uint2 *nn, *tn;
    const void *p, *ds, *q, *k, *dout;
    void *dq, *dk, *dv;
    size_t in_pitch, do_pitch, grad_pitch;
    uint32_t first, pairs, H, d, nb, blocks, lut_stride;      // pairs: (batch, head) pairs of this launch, from `first` on
    bool in_vec, do_vec, out_vec;
    float outside;                                            // 16 bits: what dQ and dK are multiplied by
};
constexpr uint32_t kStages = 3;
template <int BS, int W, int DT, bool TRANS> struct ProductCfg {
    static constexpr uint32_t T = DT == SFB_F32 ? 3 : 1, E = DT == SFB_F32 ? 4 : 2;
    static constexpr uint32_t a_rows = TRANS ? 32 : BS, a_cols = TRANS ? BS : 32, a_stride = a_cols * 2 + 16, plane = a_rows * a_stride;
    static constexpr uint32_t b_stride = 32 * W * E + 16, a_bytes = T * plane, stage = a_bytes + 32 * b_stride;
    static constexpr uint32_t threads = 32 * W * (BS / 32);
};
__device__ __forceinline__ void ldmatrix4(uint4 &r, uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint4 &r, uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
}
// fp32 results that are not finite, by FMAs: a product of terms may be inf - inf where the operands' own is a number or an infinity.
// A backward pass whose every gradient is NaN takes eight to ten times as long as one on finite operands.
template <int BS, bool TRANS>
__device__ __noinline__ void product_again(float (&acc)[2][4][4], const uint16_t *P, const float *V, const uint2 *ents, uint32_t count, size_t blocks_at, size_t pitch,
                                           uint32_t r0, uint32_t left, uint32_t g, uint32_t t)
{
    for (int m = 0; m < 2; m++)
        for (int half = 0; half < 2; half++) {
            const uint32_t r = r0 + 16 * m + 8 * half + g;
            float sum[8] = {};
            for (uint32_t e = 0; e < count; e++) {
                const uint2 en = ents[e];
                const uint16_t *block = P + (blocks_at + en.x) * BS * BS * 3;
                for (uint32_t k = 0; k < BS; k++) {
                    const uint32_t at = TRANS ? k * BS + r : r * BS + k;
                    const float x = __uint_as_float((uint32_t)block[at] << 16) +
                                    (__uint_as_float((uint32_t)block[at + BS * BS] << 16) + __uint_as_float((uint32_t)block[at + 2 * BS * BS] << 16));
                    for (uint32_t c = 0; c < 8; c++)
                        if (8 * t + c < left) sum[c] = fmaf(x, V[((size_t)en.y * BS + k) * pitch + 8 * t + c], sum[c]);
                }
            }
            for (int c = 0; c < 8; c++) acc[m][c & 3][2 * half + (c >> 2)] = sum[c];
        }
}
template <int BS, int W, int DT, bool TRANS>
__device__ __forceinline__ void product_rows(char *sm, const ProductArgs &a, uint32_t i, uint32_t y, const void *P, const void *V, size_t pitch, bool vec, void *out, float factor)
{
    typedef ProductCfg<BS, W, DT, TRANS> Cfg;
    constexpr uint32_t T = Cfg::T, E = Cfg::E, PARTS = BS / 32;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t bh = a.first + y, b = bh / a.H, h = bh - b * a.H;
    const uint32_t r0 = 32 * (warp / W), n0 = 32 * (warp % W);
    const uint2 *lut = (TRANS ? a.tn : a.nn) + (size_t)h * a.lut_stride;
    const uint2 head = lut[i], *ents = lut + head.x;
    const uint32_t chunks = head.y * PARTS;
    const size_t baseV = (size_t)b * a.nb * BS * pitch + (size_t)h * a.d;

    uint2 ent = chunks ? ents[0] : make_uint2(0u, 0u);       // of the chunk to be asked for next
    auto issue = [&](uint32_t c) {                           // called for c = 0, 1, 2, ... in turn
        if (c < chunks) {
            const uint32_t part = c % PARTS;
            char *buf = sm + (c % kStages) * Cfg::stage;
            const uint16_t *pa = (const uint16_t *)P + ((size_t)y * a.blocks + ent.x) * BS * BS * T + (TRANS ? part * 32 * BS : part * 32);
            constexpr uint32_t PA = Cfg::a_cols / 8;          // 16-byte pieces per row
#pragma unroll
            for (uint32_t x = threadIdx.x; x < T * Cfg::a_rows * PA; x += Cfg::threads) {
                const uint32_t r = x / PA, c8 = x % PA, pl = r / Cfg::a_rows, rr = r % Cfg::a_rows;
                tile::cp_async16((float *)(buf + r * Cfg::a_stride + c8 * 16), pa + pl * BS * BS + rr * BS + c8 * 8, 16u);
            }
            char *vb = buf + Cfg::a_bytes;
            const char *pv = (const char *)V + (baseV + ((size_t)ent.y * BS + part * 32) * pitch) * E;
            if (vec) {
                constexpr uint32_t PB = 32 * W * E / 16, N = 16 / E;
#pragma unroll
                for (uint32_t x = threadIdx.x; x < 32 * PB; x += Cfg::threads) {
                    const uint32_t r = x / PB, c8 = x % PB, in = c8 * N < a.d ? 16u : 0u;
                    tile::cp_async16((float *)(vb + r * Cfg::b_stride + c8 * 16), pv + (r * pitch + (in ? c8 * N : 0)) * E, in);
                }
            } else {
                for (uint32_t x = threadIdx.x; x < 32 * 32 * W; x += Cfg::threads) {
                    const uint32_t r = x / (32 * W), col = x % (32 * W);
                    if constexpr (E == 4) *(float *)(vb + r * Cfg::b_stride + col * 4) = col < a.d ? __ldg((const float *)pv + r * pitch + col) : 0.f;
                    else *(uint16_t *)(vb + r * Cfg::b_stride + col * 2) = col < a.d ? __ldg((const uint16_t *)pv + r * pitch + col) : (uint16_t)0;
                }
            }
            if (part + 1 == PARTS && c + 1 < chunks) ent = ents[(c + 1) / PARTS];
        }
        tile::cp_commit();
    };
    float acc[2][4][4] = {};
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(sm);
    // where this lane's rows of the 8x8 matrices are: of P (two of rows, two of the contraction) and of a 16-bit operand
    const uint32_t at_a = TRANS ? ((lane & 7) + 8 * (lane >> 4)) * Cfg::a_stride + 2 * (r0 + 8 * ((lane >> 3) & 1)) : (r0 + (lane & 15)) * Cfg::a_stride + 16 * (lane >> 4);
    const uint32_t at_b = Cfg::a_bytes + ((lane & 7) + 8 * ((lane >> 3) & 1)) * Cfg::b_stride + 2 * (n0 + 8 * (lane >> 4));
    for (uint32_t c = 0; c + 1 < kStages; c++) issue(c);
    for (uint32_t c = 0; c < chunks; c++) {
        tile::cp_wait<(int)kStages - 2>();
        __syncthreads();
        issue(c + kStages - 1);
        const uint32_t buf = base + (c % kStages) * Cfg::stage;
        float sum[2][4][4];
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) sum[m][n][e] = 0.f;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            tile::Frag<(int)T> fa[2];
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (uint32_t x = 0; x < T; x++) {
                    if (TRANS) ldmatrix4_trans(fa[m].w[x], buf + at_a + x * Cfg::plane + 16 * k * Cfg::a_stride + 32 * m);
                    else ldmatrix4(fa[m].w[x], buf + at_a + x * Cfg::plane + 16 * m * Cfg::a_stride + 32 * k);
                }
            if constexpr (DT == SFB_F32) {
                // column g of n-tile n is column 4 g + n; elements 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of the contraction
                const float *v = (const float *)(sm + (c % kStages) * Cfg::stage + Cfg::a_bytes + (16 * k + 2 * t) * Cfg::b_stride) + n0 + 4 * g;
                float4 x[4];
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = *(const float4 *)((const char *)v + ((e & 1) + 8 * (e >> 1)) * Cfg::b_stride);
                tile::Four<3> fb[4];
                const float y0[4] = {x[0].x, x[1].x, x[2].x, x[3].x}, y1[4] = {x[0].y, x[1].y, x[2].y, x[3].y}, y2[4] = {x[0].z, x[1].z, x[2].z, x[3].z},
                            y3[4] = {x[0].w, x[1].w, x[2].w, x[3].w};
                tile::split4<3>(fb[0], y0);
                tile::split4<3>(fb[1], y1);
                tile::split4<3>(fb[2], y2);
                tile::split4<3>(fb[3], y3);
#pragma unroll
                for (int m = 0; m < 2; m++) tile::mma16<4, 3, 3>(acc[m], fa[m], fb);
            } else {
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    uint4 fb;
                    ldmatrix4_trans(fb, buf + at_b + 16 * k * Cfg::b_stride + 32 * n);
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        const uint4 &f = fa[m].w[0];
                        mma_own<DT>(sum[m][2 * n], f.x, f.y, f.z, f.w, fb.x, fb.y);
                        mma_own<DT>(sum[m][2 * n + 1], f.x, f.y, f.z, f.w, fb.z, fb.w);
                    }
                }
            }
        }
        if constexpr (DT != SFB_F32) {
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    tile::add2(acc[m][n][0], acc[m][n][1], sum[m][n][0], sum[m][n][1]);
                    tile::add2(acc[m][n][2], acc[m][n][3], sum[m][n][2], sum[m][n][3]);
                }
        }
    }
    const uint32_t left = a.d > n0 ? a.d - n0 : 0;
    if constexpr (DT == SFB_F32) {
        const bool odd = !(tile::zero_if_finite<4>(acc[1], tile::zero_if_finite<4>(acc[0], 0.f)) == 0.f);
        if (__any_sync(0xffffffffu, odd))
            product_again<BS, TRANS>(acc, (const uint16_t *)P, (const float *)V + baseV + n0, ents, head.y, (size_t)y * a.blocks, pitch, r0, left, g, t);
    }
    // rows (columns) without blocks are written as zeros
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const size_t at = ((size_t)b * a.nb * BS + (size_t)i * BS + r0 + 16 * m + 8 * half + g) * a.grad_pitch + (size_t)h * a.d + n0;
            if constexpr (DT == SFB_F32) {
                // columns 8 t + 0..3 are element 2 half of n-tiles 0..3, 8 t + 4..7 element 2 half + 1
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float *o = (float *)out + at + 8 * t + 4 * e;
                    if (a.out_vec) {
                        if (8 * t + 4 * e < left) *(float4 *)o = make_float4(acc[m][0][2 * half + e], acc[m][1][2 * half + e], acc[m][2][2 * half + e], acc[m][3][2 * half + e]);
                    } else {
#pragma unroll
                        for (int n = 0; n < 4; n++)
                            if (8 * t + 4 * e + n < left) o[n] = acc[m][n][2 * half + e];
                    }
                }
            } else {
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const uint32_t w = pack_own<DT>(acc[m][n][2 * half] * factor, acc[m][n][2 * half + 1] * factor), col = 8 * n + 2 * t;
                    uint16_t *o = (uint16_t *)out + at + col;
                    if (a.out_vec) {
                        if (col < left) *(uint32_t *)o = w;
                    } else {
                        if (col < left) o[0] = (uint16_t)w;
                        if (col + 1 < left) o[1] = (uint16_t)(w >> 16);
                    }
                }
            }
        }
}
// dV, dK and dQ of a block side by side: P and dS come from HBM once where they do not fit into L2.  The same block-row of all pairs before the
// next one, and the last eighth of them first: a launch then ends with rows of the middle, and rows and columns that keep everything lie
// at the ends in most layouts (us, pair after pair / row after row / that and the last eighth first / both ends inwards: bf16, blocks of 32, d 64,
// 4 x 12 heads of 2048 positions, strided 212 / 199 / 202 / 208, causal 466 / 463 / 466 / 456; fp32, 4 x 8 heads, BigBird 450 / 437 / 374 / 375).
template <int BS, int W, int DT>
__global__ void __launch_bounds__(32 * W * (BS / 32), 512 / (32 * W * (BS / 32))) products_kernel(const __grid_constant__ ProductArgs a)
{
    extern __shared__ __align__(16) char psm[];
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t n = blockIdx.x / 3, which = blockIdx.x - 3 * n, at = n / a.pairs, y = n - at * a.pairs, i = at < (a.nb + 7) / 8 ? a.nb - 1 - at : at - (a.nb + 7) / 8;
    if (which == 2) {
        product_rows<BS, W, DT, false>(psm, a, i, y, a.ds, a.k, a.in_pitch, a.in_vec, a.dq, a.outside);
    } else {
        product_rows<BS, W, DT, true>(psm, a, i, y, which ? a.ds : a.p, which ? a.q : a.dout, which ? a.in_pitch : a.do_pitch, which ? a.in_vec : a.do_vec, which ? a.dk : a.dv, which ? a.outside : 1.f);
    }
}
template <int BS, int W, int DT>
static int launch_products(cudaStream_t s, const ProductArgs &k)
{
    constexpr size_t bytes = kStages * (ProductCfg<BS, W, DT, true>::stage > ProductCfg<BS, W, DT, false>::stage ? ProductCfg<BS, W, DT, true>::stage
                                                                                                             : ProductCfg<BS, W, DT, false>::stage);
    static DeviceOnce once;
    const int dev = current_device();
    if (!once.done(dev)) {
        if (cudaFuncSetAttribute(products_kernel<BS, W, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
            return fail("sfb_attention_backward_recompute: shared memory configuration failed");
        once.mark(dev);
    }
    launch_overlapped_few(products_kernel<BS, W, DT>, dim3(3 * k.nb * k.pairs), dim3(ProductCfg<BS, W, DT, true>::threads), bytes, s, k);
    return 0;
}

// How many (batch, head) pairs go through the workspace at a time: block-rows for every SM to have 64 (us with 16 / 32 / 64:
// bf16, blocks of 32, d 64, strided, 4 x 12 heads of 2048 positions 242 / 212 / 210, 8 x 16 heads 598 / 528 / 496; what L2 could have kept of P and dS
// counts for less than the SMs that have nothing left to do at the end of each launch), as long as P and dS take no more
// than 512 MB, but one at least: a pair is not divided, so that the workspace is as large as P and dS of a whole one where that is more (bf16, blocks of
// 64, causal: 0.5 GB at 16384 positions, 2 GB at 32768, 8 GB at 65536; fp32 three times as much).  Parts of about the same size.
constexpr uint64_t kRowsPerSm = 64, kMostSms = 148, kMostBytes = 512ull << 20;
static uint64_t score_bytes(int dtype) { return dtype == SFB_F32 ? 6 : 2; }      // three planes, or the operands' type
static uint32_t pairs_at_a_time(int dtype, uint32_t bs, uint32_t nb, uint32_t blocks, uint32_t B, uint32_t H)
{
    const uint64_t one = 2ull * blocks * bs * bs * score_bytes(dtype), all = (uint64_t)B * H, most = one ? kMostBytes / one : all;
    uint64_t n = (kMostSms * kRowsPerSm + nb - 1) / nb;
    if (n > most) n = most;
    if (n > 65535) n = 65535;
    if (n > all) n = all;
    if (n < 1) n = 1;
    const uint64_t parts = (all + n - 1) / n;
    return (uint32_t)(parts ? (all + parts - 1) / parts : 1);
}
uint64_t simt_backward_workspace(int dtype, uint32_t bs, uint32_t nb, uint32_t blocks, uint32_t B, uint32_t H)
{
    return 2ull * pairs_at_a_time(dtype, bs, nb, blocks, B, H) * blocks * bs * bs * score_bytes(dtype);
}

template <int BS, int DT>
static int backward_parts(cudaStream_t s, BlockArgs &k, ProductArgs &o, uint32_t all, uint32_t n, bool vec)
{
    constexpr uint32_t per = BS == 32 ? 4 : 1;
    for (uint32_t first = 0; first < all; first += n) {
        const uint32_t pairs = all - first < n ? all - first : n;
        k.first = o.first = first;
        o.pairs = pairs;
        if (k.blocks) {
            const dim3 grid((k.blocks + per - 1) / per, pairs);
            if constexpr (DT == SFB_F32) launch_overlapped_few(vec ? recompute_blocks_kernel<BS, true> : recompute_blocks_kernel<BS, false>, grid, dim3(tile::kThreads), BlockCfg<BS>::bytes, s, k);
            else launch_overlapped_few(vec ? recompute_blocks16_kernel<BS, DT, true> : recompute_blocks16_kernel<BS, DT, false>, grid, dim3(tile::kThreads), 0, s, k);
        }
        if (k.d <= 32 ? launch_products<BS, 1, DT>(s, o) : k.d <= 64 ? launch_products<BS, 2, DT>(s, o)
            : k.d <= 96 ? launch_products<BS, 3, DT>(s, o) : launch_products<BS, 4, DT>(s, o)) return 1;
        if (check_launch("sfb_attention_backward_recompute")) return 1;
    }
    return 0;
}
int simt_backward_recompute(cudaStream_t s, const BackwardArgs &a, float *neg_lse, float *neg_delta, void *blocks_ws)
{
    const AttnDims &p = a.p;
    const uint32_t n = pairs_at_a_time(a.dtype, a.bs, p.nb_a, p.blocks, p.B, p.H), unit = a.dtype == SFB_F32 ? 4 : 8;
    void *P = blocks_ws, *dS = (char *)blocks_ws + (size_t)n * p.blocks * a.bs * a.bs * score_bytes(a.dtype);
    auto rows = [&](std::initializer_list<const void *> at, uint64_t pitch) {      // rows of heads that are 16-byte aligned
        uintptr_t all = 0;
        for (const void *x : at) all |= (uintptr_t)x;
        return (all & 15) == 0 && pitch % unit == 0 && p.d % unit == 0;
    };
    const bool in = rows({a.q, a.k, a.v}, a.in_pitch), dout = rows({a.dout}, a.do_pitch);
    BlockArgs k = {(const uint2 *)a.nt_lut, a.q, a.k, a.v, a.dout, a.mask, neg_lse, neg_delta, P, dS, (size_t)a.in_pitch, (size_t)a.do_pitch, 0, p.H, p.d, p.nb_a,
                   p.blocks, a.nt_stride, p.mask_stride, a.inside, a.scale * 1.4426950408889634f};
    ProductArgs o = {(const uint2 *)a.nn_lut, (const uint2 *)a.tn_lut, P, dS, a.q, a.k, a.dout, a.dq, a.dk, a.dv, (size_t)a.in_pitch, (size_t)a.do_pitch, (size_t)a.grad_pitch, 0, 0,
                     p.H, p.d, p.nb_a, p.blocks, p.lut_stride, in, dout, rows({a.dq, a.dk, a.dv}, a.grad_pitch), a.scale / a.inside};
    const uint32_t all = p.B * p.H;
#define BP(BS) (a.dtype == SFB_F32 ? backward_parts<BS, SFB_F32>(s, k, o, all, n, in && dout) : a.dtype == SFB_BF16 ? backward_parts<BS, SFB_BF16>(s, k, o, all, n, in && dout) \
                                                                                                    : backward_parts<BS, SFB_F16>(s, k, o, all, n, in && dout))
    return a.bs == 32 ? BP(32) : BP(64);
#undef BP
}

}  // namespace sfb
