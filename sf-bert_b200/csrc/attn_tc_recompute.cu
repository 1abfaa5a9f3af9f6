// The backward pass that makes the probabilities again (recompute.cuh), on the tensor cores (tcgen05) for 16-bit operands, block_size 64,
// head size 64.  neg_lse = -lse log2(e) and neg_delta = -scale rowsum(dO * O) come from attn_recompute.cu; then
//   P = exp2(S scale log2(e) + neg_lse),  dS = P * (dP scale + neg_delta),   S = Q.K^T,  dP = dO.V^T,   dQ = dS.K,  dK = dS^T.Q,  dV = P^T.dO.
//
// Two kernels, the same code seen from two sides (COL): an item is 128 "own" positions (queries of two block-rows, or keys of two
// block-columns) of one (batch, head) and a walk over the union of their blocks.  Nothing of the size of the scores is written anywhere and no sum
// is shared between CTAs, so no atomics: each side makes S and dP for itself, 7 products per block instead of 5.  Per step of 64 other
// positions:
//     S  = own1 . Z^T      own1: Q (K), Z: the step's rows of K (Q)
//     dP = own2 . Y^T      own2: dO (V), Y: the step's rows of V (dO)
//     P and dS             256 threads, one own position and 32 of the 64 others each, straight out of TMEM and back, as 16-bit operands
//     out += dS . Z        dQ (dK)
//     COL: dV += P . Y     (for COL S and dP are already transposed: their lanes are keys)
// What bounds it: 8192 exponentials per step and side (512 cycles of the SM's MUFU), 3 or 4 products of 128 cycles, and the chain from barrier to
// barrier between them.  Two CTAs per SM, so that one's products and waits run under the other's arithmetic.
// A CTA starts with the item of its own index and takes over items that have not been started (cluster launch control), long rows and
// columns paired with each other and first.
// Warps: 0-7 P, dS and the epilogue; 8 TMA; 9 issues S (and dV), 10 dP and out; 11 plans the unions of the coming items.
// TMEM (256 columns).  Rows: S 64, dP 64, dS 32, dQ 64: S and dP of the next step run as soon as this step's are in registers.  Columns: S 64, dP 64,
// dK 64, dV 64: P lies over S and dS over dP, each warp's over its own columns of them, so that the next S waits for this
// step's dV, and the next dP for its dK.
#include "recompute.cuh"
#include "tc_common.cuh"

namespace sfb {
namespace tc {

constexpr uint32_t kRcStages = 4;
constexpr uint32_t kRcStageBytes = 2 * kTileBytes;               // Z, Y
constexpr uint32_t kRcThreads = 12 * 32;
constexpr uint32_t kRcMaxUnion = 256;

struct RcShared {
    uint64_t in_full[kRcStages], in_empty[kRcStages], own_full, own_free, s_full, s_free, p_full, dv_done, dp_full, dp_free, ds_full, ds_free, o_final, o_free;
    uint64_t list_ready[2], list_free[2], clc_bar, drained[2];
    alignas(16) uint32_t clc_response[4];
    uint32_t tmem_base, abort_flag, list_n[2], list_bh[2], list_own[2][2];      // list_own: the two rows (columns)
    alignas(16) float neg_lse[kRcStages][64], neg_delta[kRcStages][64];         // COL: of the step's queries
    alignas(16) uint64_t mask[kRcStages][2][64];                                // COL: the step's two blocks of mask words
    UnionEntry lists[2][kRcMaxUnion];
};
constexpr size_t kRcSmem = 1024 + 2 * kQBytes + kRcStages * kRcStageBytes + sizeof(RcShared);
static_assert(2 * (kRcSmem + 1024) <= 228 * 1024, "two CTAs per SM");

struct RcParams {
    const uint2 *lut;          // nn_lut (rows) or tn_lut (columns)
    const float *neg_lse, *neg_delta;        // [B, H, L]
    const uint64_t *mask;
    void *out1, *out2;         // dQ, - or dK, dV
    uint32_t B, H, nb, blocks, lut_stride, mask_stride, pitch;        // pitch: elements between consecutive rows of the gradients
    float scale, scale_log2e;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}
#define TMEM_ST_8(addr, r)                                                                                              \
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), \
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])                                                    \
                 : "memory")

template <bool COL, bool MASK, bool BF16>
__global__ void __launch_bounds__(kRcThreads, 2)
recompute_tc_kernel(const __grid_constant__ CUtensorMap own1_map, const __grid_constant__ CUtensorMap own2_map, const __grid_constant__ CUtensorMap zmap,
                    const __grid_constant__ CUtensorMap ymap, const RcParams p)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *own1 = smem, *own2 = smem + kQBytes, *stages = smem + 2 * kQBytes;
    RcShared *st = (RcShared *)(stages + kRcStages * kRcStageBytes);

    const uint32_t warp = uniform_warp(), lane = threadIdx.x & 31;
    const uint32_t L = p.nb * 64;
    volatile uint32_t *abort_flag = &st->abort_flag;
    const uint32_t fmt = BF16 ? 1u : 0u;

    if (threadIdx.x == 0) {
        prefetch_map(own1_map);
        prefetch_map(own2_map);
        prefetch_map(zmap);
        prefetch_map(ymap);
        for (uint32_t s = 0; s < kRcStages; s++) { mbar_init(&st->in_full[s], 1); mbar_init(&st->in_empty[s], COL ? 2 : 1); }
        mbar_init(&st->own_full, 1);
        mbar_init(&st->own_free, 2);
        mbar_init(&st->s_full, 1);
        mbar_init(&st->s_free, 8);
        mbar_init(&st->p_full, 8);
        mbar_init(&st->dv_done, 1);
        mbar_init(&st->dp_full, 1);
        mbar_init(&st->dp_free, 8);
        mbar_init(&st->ds_full, 8);
        mbar_init(&st->ds_free, 1);
        mbar_init(&st->o_final, COL ? 2 : 1);
        mbar_init(&st->o_free, 8);
        for (int i = 0; i < 2; i++) {
            mbar_init(&st->list_ready[i], 1);
            mbar_init(&st->list_free[i], 11);      // TMA, two issuers, eight worker warps
            mbar_init(&st->drained[i], 1);
        }
        mbar_init(&st->clc_bar, 1);
        st->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&st->tmem_base)), "r"(256u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = st->tmem_base;
    // 16 others' operand words of a warp's half: rows' dS has columns of its own, columns' P and dS lie over S and dP
    const uint32_t t_s = tmem, t_dp = tmem + 64, t_p = t_s, t_ds = COL ? t_dp : tmem + 128, half_step = COL ? 32 : 16;
    const uint32_t t_out = COL ? tmem + 128 : tmem + 192, t_dv = tmem + 192;
    grid_dependency_wait();
    grid_launch_dependents();

    if (warp == 11) {
        // ===== planner: the coming items and their unions, up to two ahead =====
        uint32_t id = blockIdx.x;
        const uint32_t first_pairs = p.lut_stride == 0 ? long_pairs(p.lut, p.nb, p.blocks, lane) : 0;
        for (uint32_t k = 0;; k++) {
            const uint32_t slot = k & 1;
            if (id != kNoItem && lane == 0) {
                fence_proxy_async();                          // the last answer has been read
                clc_request(st->clc_response, &st->clc_bar);
            }
            if (k >= 2 && !mbar_wait_warp(&st->list_free[slot], ((k >> 1) - 1) & 1, abort_flag, 110)) break;
            uint32_t n = 0, bh = kNoItem, own[2] = {kNoItem, kNoItem};
            if (id != kNoItem) {
                const ItemAt it = locate_item(p.lut, p.lut_stride, p.B, p.H, p.nb, p.blocks, first_pairs, id, lane, !COL);
                bh = it.b * p.H + it.h;
                own[0] = it.own[0];
                own[1] = it.own[1];
                n = warp_union(p.lut + (size_t)it.h * p.lut_stride, own, st->lists[slot], kRcMaxUnion, lane);
                if (n == kNoItem) {                           // more blocks than the caller's maximum: recorded, zeros written
                    if (lane == 0) atomicCAS(&g_status, 0u, (9u << 24) | (blockIdx.x & 0xffffffu));
                    n = 0;
                }
            }
            if (lane == 0) {
                st->list_n[slot] = n;
                st->list_bh[slot] = bh;
                st->list_own[slot][0] = own[0];
                st->list_own[slot][1] = own[1];
                mbar_arrive(&st->list_ready[slot]);
            }
            if (id == kNoItem) break;
            if (!mbar_wait_warp(&st->clc_bar, k & 1, abort_flag, 111)) break;
            id = clc_item(st->clc_response);
            __syncwarp();
        }
    } else if (warp == 8) {
        // ===== TMA producer =====
        if (elect_one()) {
            uint32_t g = 0, kq = 0;                           // steps, items with blocks
            bool alive = true;
            for (uint32_t k = 0; alive; k++) {
                const uint32_t slot = k & 1;
                if (!mbar_wait(&st->list_ready[slot], (k >> 1) & 1, abort_flag, 112)) break;
                const uint32_t bh = st->list_bh[slot], T = st->list_n[slot];
                if (bh == kNoItem) break;
                const uint32_t b = bh / p.H, h = bh - b * p.H;
                const int32_t x = (int32_t)(h * 64), row0 = (int32_t)(b * L), beyond = (int32_t)(p.B * L);
                for (uint32_t t = 0; t < T; t++, g++) {
                    const uint32_t s = g % kRcStages;
                    if (g >= kRcStages && !mbar_wait(&st->in_empty[s], ((g / kRcStages) - 1) & 1, abort_flag, 113)) { alive = false; break; }
                    const uint32_t base = smem_u32(stages + s * kRcStageBytes);
                    const UnionEntry ent = st->lists[slot][t];
                    const uint32_t words = COL && MASK ? 512u * __popc(ent.flags & 3u) : 0u;
                    mbar_expect_tx(&st->in_full[s], kRcStageBytes + (COL ? 512u : 0u) + words);
                    tma_load_2d(base, &zmap, &st->in_full[s], x, row0 + (int32_t)(ent.col * 64));
                    tma_load_2d(base + kTileBytes, &ymap, &st->in_full[s], x, row0 + (int32_t)(ent.col * 64));
                    if (COL) {
                        const size_t at = (size_t)bh * L + (size_t)ent.col * 64;
                        bulk_load(smem_u32(st->neg_lse[s]), p.neg_lse + at, 256, &st->in_full[s]);
                        bulk_load(smem_u32(st->neg_delta[s]), p.neg_delta + at, 256, &st->in_full[s]);
                        if (MASK) {
                            const uint64_t *m = p.mask + (size_t)h * p.mask_stride;
#pragma unroll
                            for (uint32_t o = 0; o < 2; o++)
                                if ((ent.flags >> o) & 1u) bulk_load(smem_u32(st->mask[s][o]), m + (size_t)ent.blk[o] * 64, 512, &st->in_full[s]);
                        }
                    }
                    if (t == 0) {
                        // the item before has made its last S and dP
                        if (kq >= 1 && !mbar_wait(&st->own_free, (kq - 1) & 1, abort_flag, 114)) { alive = false; break; }
                        mbar_expect_tx(&st->own_full, 2 * kQBytes);
#pragma unroll
                        for (uint32_t o = 0; o < 2; o++) {
                            const int32_t y = st->list_own[slot][o] == kNoItem ? beyond : row0 + (int32_t)(st->list_own[slot][o] * 64);
                            tma_load_2d(smem_u32(own1) + o * kTileBytes, &own1_map, &st->own_full, x, y);
                            tma_load_2d(smem_u32(own2) + o * kTileBytes, &own2_map, &st->own_full, x, y);
                        }
                        kq++;
                    }
                }
                if (alive) mbar_arrive(&st->list_free[slot]);
            }
        }
    } else if (warp == 9) {
        // ===== S = own1 . Z^T (and dV += P . Y) =====
        if (elect_one()) {
            const uint32_t idesc_s = instr_desc(fmt, fmt, 128, 64, 0), idesc_dv = instr_desc(fmt, fmt, 128, 64, 1);
            const uint64_t a_desc = smem_desc_sw128(smem_u32(own1));
            uint32_t g = 0, kq = 0;
            bool alive = true;
            for (uint32_t k = 0; alive; k++) {
                const uint32_t slot = k & 1;
                if (!mbar_wait(&st->list_ready[slot], (k >> 1) & 1, abort_flag, 115)) break;
                const uint32_t T = st->list_n[slot];
                if (st->list_bh[slot] == kNoItem) break;
                if (T > 0 && !mbar_wait(&st->own_full, kq & 1, abort_flag, 116)) break;
                for (uint32_t t = 0; t < T; t++, g++) {
                    const uint32_t s = g % kRcStages;
                    const bool ready = mbar_try_wait(&st->in_full[s], (g / kRcStages) & 1);
                    // rows: the last S is in registers; columns: the last P, which lies over it, has been multiplied
                    if (g >= 1 && !mbar_wait(COL ? &st->dv_done : &st->s_free, (g - 1) & 1, abort_flag, 117)) { alive = false; break; }
                    if (!ready && !mbar_wait(&st->in_full[s], (g / kRcStages) & 1, abort_flag, 118)) { alive = false; break; }
                    tcgen05_fence_after();
                    const uint32_t base = smem_u32(stages + s * kRcStageBytes);
                    const uint64_t z_desc = smem_desc_sw128(base), y_desc = smem_desc_sw128(base + kTileBytes);
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; kk++) umma_f16(t_s, a_desc + 2 * kk, z_desc + 2 * kk, idesc_s, kk);
                    umma_commit(&st->s_full);
                    if (t + 1 == T) umma_commit(&st->own_free);
                    if (COL) {
                        // the accumulator still holds the previous item's dV until its epilogue has read it
                        if (t == 0 && kq >= 1 && !mbar_wait(&st->o_free, (kq - 1) & 1, abort_flag, 119)) { alive = false; break; }
                        if (!mbar_wait(&st->p_full, g & 1, abort_flag, 120)) { alive = false; break; }
                        tcgen05_fence_after();
#pragma unroll
                        for (uint32_t kk = 0; kk < 4; kk++)
                            umma_f16_ts(t_dv, t_p + half_step * (kk >> 1) + 8 * (kk & 1), y_desc + 128 * kk, idesc_dv, (t | kk) ? 1u : 0u);
                        umma_commit(&st->dv_done);
                        umma_commit(&st->in_empty[s]);
                        if (t + 1 == T) umma_commit(&st->o_final);
                    }
                }
                if (T > 0) kq++;
                if (alive) mbar_arrive(&st->list_free[slot]);
            }
        }
    } else if (warp == 10) {
        // ===== dP = own2 . Y^T and out += dS . Z =====
        if (elect_one()) {
            const uint32_t idesc_dp = instr_desc(fmt, fmt, 128, 64, 0), idesc_out = instr_desc(fmt, fmt, 128, 64, 1);
            const uint64_t a_desc = smem_desc_sw128(smem_u32(own2));
            uint32_t g = 0, kq = 0;
            bool alive = true;
            auto issue_dp = [&](uint32_t gg, bool last) -> bool {
                const uint32_t s = gg % kRcStages;
                const bool ready = mbar_try_wait(&st->in_full[s], (gg / kRcStages) & 1);
                // rows: the last dP is in registers; columns: the last dS, which lies over it, has been multiplied
                if (gg >= 1 && !mbar_wait(COL ? &st->ds_free : &st->dp_free, (gg - 1) & 1, abort_flag, 121)) return false;
                if (!ready && !mbar_wait(&st->in_full[s], (gg / kRcStages) & 1, abort_flag, 122)) return false;
                tcgen05_fence_after();
                const uint64_t y_desc = smem_desc_sw128(smem_u32(stages + s * kRcStageBytes + kTileBytes));
#pragma unroll
                for (uint32_t kk = 0; kk < 4; kk++) umma_f16(t_dp, a_desc + 2 * kk, y_desc + 2 * kk, idesc_dp, kk);
                umma_commit(&st->dp_full);
                if (last) umma_commit(&st->own_free);
                return true;
            };
            for (uint32_t k = 0; alive; k++) {
                const uint32_t slot = k & 1;
                if (!mbar_wait(&st->list_ready[slot], (k >> 1) & 1, abort_flag, 123)) break;
                const uint32_t T = st->list_n[slot];
                if (st->list_bh[slot] == kNoItem) break;
                if (T > 0) {
                    if (!mbar_wait(&st->own_full, kq & 1, abort_flag, 124)) break;
                    if (!issue_dp(g, T == 1)) break;
                }
                for (uint32_t t = 0; t < T; t++, g++) {
                    const uint32_t s = g % kRcStages;
                    // rows: the next dP under this step's arithmetic
                    if (!COL && t + 1 < T && !issue_dp(g + 1, t + 2 == T)) { alive = false; break; }
                    if (t == 0 && kq >= 1 && !mbar_wait(&st->o_free, (kq - 1) & 1, abort_flag, 125)) { alive = false; break; }
                    if (!mbar_wait(&st->ds_full, g & 1, abort_flag, 126)) { alive = false; break; }
                    tcgen05_fence_after();
                    const uint64_t z_desc = smem_desc_sw128(smem_u32(stages + s * kRcStageBytes));
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; kk++)
                        umma_f16_ts(t_out, t_ds + half_step * (kk >> 1) + 8 * (kk & 1), z_desc + 128 * kk, idesc_out, (t | kk) ? 1u : 0u);
                    umma_commit(&st->ds_free);
                    umma_commit(&st->in_empty[s]);            // S and dP of this step are complete: their values made this dS
                    if (t + 1 == T) umma_commit(&st->o_final);
                    if (COL && t + 1 < T && !issue_dp(g + 1, t + 2 == T)) { alive = false; break; }
                }
                if (T > 0) kq++;
                if (alive) mbar_arrive(&st->list_free[slot]);
            }
        }
    } else {
        // ===== P, dS and the epilogue: own position r, half of the other side's 64 =====
        const uint32_t quarter = warp & 3, ch = warp >> 2;
        const uint32_t cb = ch * 32, r = quarter * 32 + lane, half = r >> 6;
        const uint32_t lane_field = (quarter * 32) << 16;
        const uint64_t scale2 = pk64(p.scale, p.scale), sl2 = pk64(p.scale_log2e, p.scale_log2e);
        uint32_t g = 0, kq = 0;                              // steps, items with blocks finished
        bool alive = true;
        for (uint32_t k = 0; alive; k++) {
            const uint32_t slot = k & 1;
            if (!mbar_wait_warp(&st->list_ready[slot], (k >> 1) & 1, abort_flag, 127)) break;
            const uint32_t bh = st->list_bh[slot], T = st->list_n[slot];
            if (bh == kNoItem) break;
            const uint32_t blk = st->list_own[slot][half], b = bh / p.H, h = bh - b * p.H;
            const UnionEntry *list = st->lists[slot];
            uint64_t nl2 = 0, nd2 = 0;
            if (!COL) {
                // this query's constants; of a row that is not there P is 0
                float nl = -INFINITY, nd = 0.f;
                if (blk != kNoItem) {
                    const size_t at = (size_t)bh * L + (size_t)blk * 64 + (r & 63);
                    nl = __ldg(p.neg_lse + at);
                    nd = __ldg(p.neg_delta + at);
                }
                nl2 = pk64(nl, nl);
                nd2 = pk64(nd, nd);
            }
            // rows: this row's mask word of step t, fetched a step ahead
            auto mask_word = [&](uint32_t t) -> uint32_t {
                if (!((list[t].flags >> half) & 1u)) return 0u;
                return (uint32_t)(__ldg(p.mask + (size_t)h * p.mask_stride + (size_t)list[t].blk[half] * 64 + (r & 63)) >> cb);
            };
            uint32_t mw_next = !COL && MASK && T > 0 ? mask_word(0) : 0u;
            for (uint32_t t = 0; t < T; t++, g++) {
                const uint32_t s = g % kRcStages;
                // whether this row (column) has the step's block: the same for the whole warp.  Where it has not, P and dS are zeros
                const bool mine = __any_sync(0xffffffffu, (list[t].flags >> half) & 1u);
                uint32_t keep = mw_next;                     // rows: bit j: column cb + j
                if (!COL && MASK && t + 1 < T) mw_next = mask_word(t + 1);
                const bool in_ok = !COL || mbar_try_wait(&st->in_full[s], (g / kRcStages) & 1);
                if (!mbar_wait_warp(&st->s_full, g & 1, abort_flag, 128)) { alive = false; break; }
                tcgen05_fence_after();
                uint32_t v[32];
                TMEM_LD_32((v), t_s + lane_field + cb);
                // the queries' constants and mask words came with the barrier that the product waited for; observing it makes them visible here
                if (COL && !__all_sync(0xffffffffu, in_ok) && !mbar_wait_warp(&st->in_full[s], (g / kRcStages) & 1, abort_flag, 129)) { alive = false; break; }
                tmem_wait_ld();
                if (!COL) {
                    tcgen05_fence_before();
                    mbar_arrive_warp(&st->s_free, lane);
                }
                // P in place of the scores, fp32
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    uint64_t n2 = nl2;
                    if (COL) n2 = *(const uint64_t *)(st->neg_lse[s] + cb + 2 * j);
                    float x0, x1;
                    up64(fma2p(pk64(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), sl2, n2), x0, x1);
                    v[2 * j] = __float_as_uint(ex2_approx(x0));
                    v[2 * j + 1] = __float_as_uint(ex2_approx(x1));
                }
                if (MASK && mine) {
                    if (COL) {
                        // bit r of the words of the 32 queries: a lane looks at one, and all lanes at each where one of them is not all ones
                        const uint32_t *w = (const uint32_t *)st->mask[s][half] + 2 * cb + (quarter & 1);
                        if (!__all_sync(0xffffffffu, w[2 * lane] == 0xffffffffu)) {
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (!((w[2 * j] >> lane) & 1u)) v[j] = 0u;
                        }
                    } else if (!__all_sync(0xffffffffu, keep == 0xffffffffu)) {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (!((keep >> j) & 1u)) v[j] = 0u;
                    }
                }
                if (COL) {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t w[8];
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            w[j] = mine ? pack2(__uint_as_float(v[16 * c + 2 * j]), __uint_as_float(v[16 * c + 2 * j + 1]), BF16) : 0u;
                        TMEM_ST_8(t_p + lane_field + cb + 8 * c, w);
                    }
                    tmem_wait_st();
                    tcgen05_fence_before();
                    mbar_arrive_warp(&st->p_full, lane);
                }
                const bool ds_ok = COL || g == 0 || mbar_try_wait(&st->ds_free, (g - 1) & 1);
                if (!mbar_wait_warp(&st->dp_full, g & 1, abort_flag, 130)) { alive = false; break; }
                tcgen05_fence_after();
                if (!COL && !__all_sync(0xffffffffu, ds_ok) && !mbar_wait_warp(&st->ds_free, (g - 1) & 1, abort_flag, 131)) { alive = false; break; }
                tcgen05_fence_after();
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t u[16], w[8];
                    TMEM_LD_16((u), t_dp + lane_field + cb + 16 * c);
                    tmem_wait_ld();
                    if (!COL && c == 1) {
                        tcgen05_fence_before();
                        mbar_arrive_warp(&st->dp_free, lane);
                    }
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        uint64_t d2 = nd2;
                        if (COL) d2 = *(const uint64_t *)(st->neg_delta[s] + cb + 16 * c + 2 * j);
                        const uint64_t x = fma2p(pk64(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1])), scale2, d2);
                        float e0, e1;
                        up64(mul2p(x, pk64(__uint_as_float(v[16 * c + 2 * j]), __uint_as_float(v[16 * c + 2 * j + 1]))), e0, e1);
                        w[j] = pack2(e0, e1, BF16);
                    }
                    if (!mine) {
#pragma unroll
                        for (int j = 0; j < 8; j++) w[j] = 0u;
                    }
                    TMEM_ST_8(t_ds + lane_field + half_step * ch + 8 * c, w);
                }
                tmem_wait_st();
                tcgen05_fence_before();
                mbar_arrive_warp(&st->ds_full, lane);
            }
            if (!alive) break;
            if (T > 0 && !mbar_wait_warp(&st->o_final, kq & 1, abort_flag, 132)) break;
            tcgen05_fence_after();
            const size_t at = ((size_t)b * L + (size_t)blk * 64 + (r & 63)) * p.pitch + (size_t)h * 64 + cb;
#pragma unroll
            for (int o = 0; o < (COL ? 2 : 1); o++) {
                uint16_t *dst = (uint16_t *)(o ? p.out2 : p.out1) + at;
                uint32_t v[32];
                if (T > 0) {
                    TMEM_LD_32((v), (o ? t_dv : t_out) + lane_field + cb);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j++) v[j] = 0u;              // rows and columns without blocks have zero gradients
                }
                if (blk != kNoItem)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        uint32_t y[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) y[j] = pack2(__uint_as_float(v[8 * c + 2 * j]), __uint_as_float(v[8 * c + 2 * j + 1]), BF16);
                        *(uint4 *)(dst + 8 * c) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
            }
            if (T > 0) {
                tcgen05_fence_before();
                mbar_arrive_warp(&st->o_free, lane);
                kq++;
            }
            mbar_arrive_warp(&st->list_free[slot], lane);
        }
    }

    // ---- teardown (also the way out after a timeout) ----
    tcgen05_fence_before();
    __syncthreads();
    if (st->abort_flag) {
        if ((warp == 9 || warp == 10) && lane == 0) {
            umma_commit(&st->drained[warp - 9]);
            for (uint32_t i = 0; i < kWaitLimit && !mbar_try_wait(&st->drained[warp - 9], 0); i++) {}
        }
        if (warp == 8 && lane == 0) {
            const uint64_t t0 = clock64();
            while (clock64() - t0 < 2000000ull) {}
        }
        __syncthreads();
    }
    if (warp == 8) {
        __syncwarp();
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u) : "memory");
    }
}

}  // namespace tc

bool tc_backward_recompute_supported(int dtype, uint32_t bs, const AttnDims &p, uint32_t nn_max, uint32_t tn_max)
{
    using namespace tc;
    return (dtype == SFB_BF16 || dtype == SFB_F16) && bs == 64 && p.d == 64 &&
           (p.nb_a <= kRcMaxUnion || (nn_max && tn_max && 2 * (uint64_t)nn_max <= kRcMaxUnion && 2 * (uint64_t)tn_max <= kRcMaxUnion)) &&
           (uint64_t)p.B * p.nb_a * 64 < (1ull << 31) - 64 && (uint64_t)((p.nb_a + 1) / 2) * p.B * p.H < (1ull << 31);
}

template <bool COL, bool MASK, bool BF16>
static int launch_side(cudaStream_t s, const CUtensorMap &own1, const CUtensorMap &own2, const CUtensorMap &z, const CUtensorMap &y, const tc::RcParams &prm)
{
    using namespace tc;
    static DeviceOnce once;
    const int dev = current_device();
    if (!once.done(dev)) {
        if (cudaFuncSetAttribute(recompute_tc_kernel<COL, MASK, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRcSmem) != cudaSuccess)
            return fail("sfb_attention_backward_recompute: cannot reserve %zu bytes of shared memory", kRcSmem);
        once.mark(dev);
    }
    const dim3 grid((prm.nb + 1) / 2 * prm.B * prm.H);
    launch_overlapped(recompute_tc_kernel<COL, MASK, BF16>, grid, dim3(kRcThreads), kRcSmem, s, own1, own2, z, y, prm);
    return 0;
}

int tc_backward_recompute(cudaStream_t s, const BackwardArgs &a, const float *neg_lse, const float *neg_delta)
{
    using namespace tc;
    const AttnDims &p = a.p;
    const int bf = a.dtype == SFB_BF16;
    const uint64_t rows = (uint64_t)p.B * p.nb_a * 64;
    CUtensorMap qm, km, vm, dm;
    if (make_map(&qm, a.q, rows, p.H, bf, 64, a.in_pitch) || make_map(&km, a.k, rows, p.H, bf, 64, a.in_pitch) || make_map(&vm, a.v, rows, p.H, bf, 64, a.in_pitch) ||
        make_map(&dm, a.dout, rows, p.H, bf, 64, a.do_pitch))
        return 1;
    RcParams row = {(const uint2 *)a.nn_lut, neg_lse, neg_delta, (const uint64_t *)a.mask, a.dq, nullptr, p.B, p.H, p.nb_a, p.blocks, p.lut_stride, p.mask_stride,
                    (uint32_t)a.grad_pitch, a.scale, a.scale * 1.4426950408889634f};
    RcParams col = row;
    col.lut = (const uint2 *)a.tn_lut;
    col.out1 = a.dk;
    col.out2 = a.dv;
#define SIDES(M, BF) (launch_side<false, M, BF>(s, qm, dm, km, vm, row) || launch_side<true, M, BF>(s, km, vm, qm, dm, col))
    if (a.mask ? (bf ? SIDES(true, true) : SIDES(true, false)) : (bf ? SIDES(false, true) : SIDES(false, false))) return 1;
#undef SIDES
    return check_launch("sfb_attention_backward_recompute");
}

int tc_status_clear_recompute()
{
    const uint32_t zero = 0;
    cudaError_t e = cudaMemcpyToSymbol(tc::g_status, &zero, sizeof(uint32_t));
    if (e != cudaSuccess) return fail("sfb_device_status_clear: %s", cudaGetErrorString(e));
    return 0;
}

int tc_status_recompute(uint32_t *out)
{
    cudaError_t e = cudaMemcpyFromSymbol(out, tc::g_status, sizeof(uint32_t));
    if (e != cudaSuccess) return fail("sfb_device_status: %s", cudaGetErrorString(e));
    return 0;
}

}  // namespace sfb
