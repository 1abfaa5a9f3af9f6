// The backward pass that makes the probabilities again (recompute.cuh), on the tensor cores (tcgen05) for 16-bit operands, block_size 64,
// head size 64.  neg_lse = -lse log2(e) and neg_delta = -inside rowsum(dO * O) come from attn_recompute.cu; then
//   P = exp2(S scale log2(e) + neg_lse),  dS = P * (dP inside + neg_delta),   S = Q.K^T,  dP = dO.V^T,
//   dQ = outside dS.K,  dK = outside dS^T.Q,  dV = P^T.dO,   inside outside = scale (recompute.cuh).
//
// Two kernels, the same code seen from two sides (COL): an item is 128 "own" positions (queries of two block-rows, or keys of two
// block-columns) of one (batch, head) and a walk over the union of their blocks.  Nothing of the size of the scores is written anywhere and no sum
// is shared between CTAs, so no atomics: each side makes S and dP for itself, 7 products per block instead of 5.  Per step of 64 other
// positions:
//     S  = own1 . Z^T      own1: Q (K), Z: the step's rows of K (Q)
//     dP = own2 . Y^T      own2: dO (V), Y: the step's rows of V (dO)
//     P and dS             128 threads, one own position each, straight out of TMEM and back, as 16-bit operands
//     out += dS . Z        dQ (dK)
//     COL: dV += P . Y     (for COL S and dP are already transposed: their lanes are keys)
// One persistent CTA per SM with three groups of four worker warps that take the steps in turn.  What bounds it is a warp's way through a step: at
// 64 full block-rows 1010 cycles per step and SM (rows) and 1230 (columns), of which the exponentials would take 512 by
// themselves and the products 432 and 590; without exponentials 790 and 1190, with a quarter of each product 960 and 1180 (measured in copies
// of this code).  What counts is therefore how little a warp does besides:
//   - a thread has a whole row of 64, with two waits and two arrivals per step (half a row per thread in eight warps per group: 1060 and 1515);
//   - nothing is done for a half of the own positions that has not the step's block, in one branch around all of it;
//   - own1 and own2 are copied to TMEM, so that a product reads 8 KB of shared memory instead of 24; the columns' constants are read
//     there by 16-byte loads of that address space (through a generic pointer: + 17 %);
//   - a chain of MMAs on one accumulator takes 115 cycles per MMA whatever its N up to 128, so the next S and dP are issued by threads of their own as
//     soon as their buffer is free.  Rows: three buffers of each.  Columns, whose accumulators take twice the room: three of S
//     and two of dP (two and three: + 15 %; P apart from S: + 12 %; four groups with a P and a dS for all: + 30 %).
// A CTA starts with the item of its own index and takes over items that have not been started (cluster launch control), long rows and
// columns paired with each other and first.  An item's epilogue falls to the groups in turn, the others go on.
// Warps: 0-11 P, dS and the epilogue; 12 TMA; 13 issues S, 14 dP, 15 out, 16 dV; 17 plans the unions of the coming items.  The control warpgroups hand
// registers to the workers (setmaxnreg): 640 threads x 96 = 12 x 32 x 128 + 8 x 32 x 48.
#include "recompute.cuh"
#include "tc_common.cuh"
#include <stddef.h>

namespace sfb {
namespace tc {

constexpr uint32_t kRcStages = 8;
constexpr uint32_t kRcStageBytes = 2 * kTileBytes;               // Z, Y
constexpr uint32_t kRcGroups = 3, kRcWorkers = 4 * kRcGroups;
constexpr uint32_t kRcThreads = 20 * 32;
constexpr uint32_t kRcMaxUnion = 256;
// TMEM columns.  S of three steps in turn (columns: P over it), dP (dS over it) of three, columns two; dQ, or dK and dV; own1, own2
template <bool COL> struct RcCols {
    static constexpr uint32_t dps = COL ? 2 : 3, dp = 192, out = dp + 64 * dps, own = 448;
    static_assert(out + (COL ? 128 : 64) == own && own + 64 == 512, "all of it");
};

struct RcShared {
    uint64_t in_full[kRcStages], in_empty[kRcStages], own_full[2], own_free[2], own_done[2], o_free;
    uint64_t o_final[kRcGroups];     // by the group whose turn the epilogue is: it waits for each completion, and must not mistake an earlier one for it
    uint64_t s_full[kRcGroups], s_free[kRcGroups], p_full[kRcGroups], p_free[kRcGroups], dp_full[kRcGroups], ds_full[kRcGroups], ds_free[kRcGroups];
    uint64_t list_ready[2], list_free[2], clc_bar, drained[4];
    alignas(16) uint32_t clc_response[4];
    uint32_t tmem_base, abort_flag, list_n[2], list_bh[2], list_own[2][2];      // list_own: the two rows (columns)
    alignas(16) float neg_lse[kRcStages][64], neg_delta[kRcStages][64];         // COL: of the step's queries
    alignas(16) uint64_t mask[kRcStages][2][64];                                // COL: the step's two blocks of mask words
    UnionEntry lists[2][kRcMaxUnion];
};
constexpr size_t kRcSmem = 1024 + 4 * kQBytes + kRcStages * kRcStageBytes + sizeof(RcShared);
static_assert(kRcSmem <= 227 * 1024, "shared memory budget");

struct RcParams {
    const uint2 *lut;          // nn_lut (rows) or tn_lut (columns)
    const float *neg_lse, *neg_delta;        // [B, H, L]
    const uint64_t *mask;
    void *out1, *out2;         // dQ, - or dK, dV
    uint32_t B, H, nb, blocks, lut_stride, mask_stride, sms, pitch;   // pitch: elements between consecutive rows of the gradients
    float inside, outside, scale_log2e;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}
// 128 rows x 32 bytes of a K-major tile in shared memory -> 128 lanes x 8 columns: the A operand of one MMA.  Ordered before the MMAs that the
// thread issues after it
__device__ __forceinline__ void copy_to_tmem(uint32_t tmem, uint64_t desc)
{
    asm volatile("tcgen05.cp.cta_group::1.128x256b [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// A wait that is mostly over when it begins: one look and a vote
__device__ __forceinline__ bool look_or_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *abort_flag, uint32_t code)
{
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || mbar_wait_warp(bar, parity, abort_flag, code);
}
// from shared memory by its own address space (a pointer into the aligned dynamic array is a generic one to the compiler); kept in order with the waits
__device__ __forceinline__ void lds_pairs(uint64_t (&v)[2], uint32_t addr)
{
    asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(v[0]), "=l"(v[1]) : "r"(addr));
}
__device__ __forceinline__ uint32_t lds_word(uint32_t addr)
{
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}

// P * (dP * inside + neg_delta) for a pair, rounded to the 16-bit type
template <bool BF16>
__device__ __forceinline__ uint32_t ds_pair(uint32_t dp0, uint32_t dp1, uint32_t p0, uint32_t p1, uint64_t inside2, uint64_t delta2)
{
    const uint64_t x = fma2p(pk64(__uint_as_float(dp0), __uint_as_float(dp1)), inside2, delta2);
    float e0, e1;
    up64(mul2p(x, pk64(__uint_as_float(p0), __uint_as_float(p1))), e0, e1);
    return pack2(e0, e1, BF16);
}

// Where rows grow (or shrink) from one end to the other (causal layouts: no row is much longer than the average, long_pairs is 0, but one end's less
// than half of the other's) and all heads have one LUT, the items go by groups of as many (batch, head)s as are a few items for every SM: the pair at
// the long end of all of a group, then the next one, so that a launch ends with its shortest items (3 x 12 causal heads of 832 positions,
// 252 items: 51 -> 44 us).  Within a group Z and Y stay in L2.  Elsewhere pairs of one (batch, head) follow each other; looking for the order of all of
// them took 1.2 us at the start of every CTA.
__device__ __forceinline__ ItemAt locate_from_end(uint32_t B, uint32_t H, uint32_t nb, uint32_t group, bool last, uint32_t id, bool back)
{
    const uint32_t npairs = (nb + 1) / 2, per = group * npairs, g = id / per, in = id - g * per;
    const uint32_t heads = B * H - g * group < group ? B * H - g * group : group, k = in / heads, pair = last ? npairs - 1 - k : k;
    uint32_t at = g * group + in - k * heads;
    if (back) at = B * H - 1 - at;
    ItemAt it;
    it.h = at / B;
    it.b = at - it.h * B;
    it.own[0] = 2 * pair;
    it.own[1] = 2 * pair + 1 < nb ? 2 * pair + 1 : kNoItem;
    return it;
}

template <bool COL, bool MASK, bool BF16>
__global__ void __launch_bounds__(kRcThreads, 1)
recompute_tc_kernel(const __grid_constant__ CUtensorMap own1_map, const __grid_constant__ CUtensorMap own2_map, const __grid_constant__ CUtensorMap zmap,
                    const __grid_constant__ CUtensorMap ymap, const RcParams p)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *own = smem, *stages = smem + 4 * kQBytes;           // own: own1 and own2 of two items in turn
    RcShared *st = (RcShared *)(stages + kRcStages * kRcStageBytes);
    typedef RcCols<COL> Cols;

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
        for (int i = 0; i < 2; i++) {
            mbar_init(&st->own_full[i], 1);
            mbar_init(&st->own_free[i], 2);
            mbar_init(&st->own_done[i], 1);
            mbar_init(&st->list_ready[i], 1);
            mbar_init(&st->list_free[i], (COL ? 5 : 4) + kRcWorkers);      // TMA, the issuers, the worker warps
        }
        for (uint32_t i = 0; i < kRcGroups; i++) {
            mbar_init(&st->s_full[i], 1);
            mbar_init(&st->s_free[i], 4);
            mbar_init(&st->p_full[i], 4);
            mbar_init(&st->p_free[i], 1);
            mbar_init(&st->dp_full[i], 1);
            mbar_init(&st->ds_full[i], 4);
            mbar_init(&st->ds_free[i], 1);
            mbar_init(&st->o_final[i], COL ? 2 : 1);
        }
        mbar_init(&st->o_free, COL ? 8 : 4);
        for (int i = 0; i < 4; i++) mbar_init(&st->drained[i], 1);
        mbar_init(&st->clc_bar, 1);
        st->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&st->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = st->tmem_base;
    grid_dependency_wait();
    grid_launch_dependents();

    // An issuer's walk over its items' steps: step(t, T, g, kq) issues what it has for one, g counting all of them and kq the items with blocks.
    auto issue_all = [&](uint32_t code, auto &&start, auto &&step) {
        uint32_t g = 0, kq = 0, q = 0, ph = 0;              // step g is group q's ph-th modulo 2
        for (uint32_t k = 0;; k++) {
            const uint32_t slot = k & 1;
            if (!mbar_wait(&st->list_ready[slot], (k >> 1) & 1, abort_flag, code)) return;
            const uint32_t T = st->list_n[slot];
            if (st->list_bh[slot] == kNoItem) return;
            if (T > 0) {
                if (!start(kq)) return;
                for (uint32_t t = 0; t < T; t++, g++) {
                    if (!step(t + 1 == T, t == 0, g, q, ph, kq)) return;
                    if (++q == kRcGroups) {
                        q = 0;
                        ph ^= 1;
                    }
                }
                kq++;
            }
            mbar_arrive(&st->list_free[slot]);
        }
    };

    if (warp >= kRcWorkers) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 17) {
            // ===== planner: the coming items and their unions, up to two ahead =====
            uint32_t id = blockIdx.x;
            const uint32_t first_pairs = p.lut_stride == 0 ? long_pairs(p.lut, p.nb, p.blocks, lane) : 0, npairs = (p.nb + 1) / 2;
            const uint32_t at_first = p.lut[0].y, at_last = p.lut[p.nb - 1].y, group = (4 * p.sms + npairs - 1) / npairs;
            const bool grows = p.lut_stride == 0 && first_pairs == 0 && (2 * at_first < at_last || 2 * at_last < at_first);
            for (uint32_t k = 0;; k++) {
                const uint32_t slot = k & 1;
                if (id != kNoItem && lane == 0) {
                    fence_proxy_async();                          // the last answer has been read
                    clc_request(st->clc_response, &st->clc_bar);
                }
                if (k >= 2 && !mbar_wait_warp(&st->list_free[slot], ((k >> 1) - 1) & 1, abort_flag, 110)) break;
                uint32_t n = 0, bh = kNoItem, rows[2] = {kNoItem, kNoItem};
                if (id != kNoItem) {
                    const ItemAt it = grows ? locate_from_end(p.B, p.H, p.nb, group, at_last > at_first, id, !COL)
                                              : locate_item(p.lut, p.lut_stride, p.B, p.H, p.nb, p.blocks, first_pairs, id, lane, !COL);
                    bh = it.b * p.H + it.h;
                    rows[0] = it.own[0];
                    rows[1] = it.own[1];
                    n = warp_union(p.lut + (size_t)it.h * p.lut_stride, rows, st->lists[slot], kRcMaxUnion, lane);
                    if (n == kNoItem) {                           // more blocks than the caller's maximum: recorded, zeros written
                        if (lane == 0) atomicCAS(&g_status, 0u, (9u << 24) | (blockIdx.x & 0xffffffu));
                        n = 0;
                    }
                }
                if (lane == 0) {
                    st->list_n[slot] = n;
                    st->list_bh[slot] = bh;
                    st->list_own[slot][0] = rows[0];
                    st->list_own[slot][1] = rows[1];
                    mbar_arrive(&st->list_ready[slot]);
                }
                if (id == kNoItem) break;
                if (!mbar_wait_warp(&st->clc_bar, k & 1, abort_flag, 111)) break;
                id = clc_item(st->clc_response);
                __syncwarp();
            }
        } else if (warp == 12) {
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
                    if (T > 0) {
                        // the item two before has gone on to TMEM
                        const uint32_t ob = kq & 1;
                        if (kq >= 2 && !mbar_wait(&st->own_free[ob], ((kq >> 1) - 1) & 1, abort_flag, 114)) break;
                        mbar_expect_tx(&st->own_full[ob], 2 * kQBytes);
                        const uint32_t base = smem_u32(own + ob * 2 * kQBytes);
#pragma unroll
                        for (uint32_t o = 0; o < 2; o++) {
                            const int32_t y = st->list_own[slot][o] == kNoItem ? beyond : row0 + (int32_t)(st->list_own[slot][o] * 64);
                            tma_load_2d(base + o * kTileBytes, &own1_map, &st->own_full[ob], x, y);
                            tma_load_2d(base + kQBytes + o * kTileBytes, &own2_map, &st->own_full[ob], x, y);
                        }
                        kq++;
                    }
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
                    }
                    if (alive) mbar_arrive(&st->list_free[slot]);
                }
            }
        } else if (warp == 13 || warp == 14) {
            // ===== S = own1 . Z^T: as soon as the group's last one is in registers (COL: as P, which lies over it, has been multiplied);
            // dP = own2 . Y^T: as soon as dS, which lies over the group's last one, has been multiplied =====
            const bool is_s = warp == 13;
            if (elect_one()) {
                const uint32_t idesc = instr_desc(fmt, fmt, 128, 64, 0), a = tmem + Cols::own + (is_s ? 0 : 32);
                uint64_t *full = is_s ? st->s_full : st->dp_full, *free_ = is_s ? (COL ? st->p_free : st->s_free) : st->ds_free, *done = &st->own_done[is_s ? 0 : 1];
                const uint32_t ring = is_s ? 3 : Cols::dps, ring0 = is_s ? 0 : Cols::dp;
                uint32_t at = 0, lap = 0;                         // buffer of the step, times round modulo 2
                issue_all(is_s ? 115 : 123,
                          [&](uint32_t kq) {
                              // the item's own tile to TMEM, where the item before is no longer read
                              if (kq >= 1 && !mbar_wait(done, (kq - 1) & 1, abort_flag, is_s ? 136 : 137)) return false;
                              if (!mbar_wait(&st->own_full[kq & 1], (kq >> 1) & 1, abort_flag, is_s ? 116 : 124)) return false;
                              tcgen05_fence_after();
                              const uint64_t desc = smem_desc_sw128(smem_u32(own + (kq & 1) * 2 * kQBytes + (is_s ? 0 : kQBytes)));
#pragma unroll
                              for (uint32_t kk = 0; kk < 4; kk++) copy_to_tmem(a + 8 * kk, desc + 2 * kk);
                              umma_commit(&st->own_free[kq & 1]);
                              return true;
                          },
                          [&](bool last, bool, uint32_t g, uint32_t q, uint32_t, uint32_t) {
                              const uint32_t s = g % kRcStages;
                              const bool ready = mbar_try_wait(&st->in_full[s], (g / kRcStages) & 1);
                              if (g >= ring && !mbar_wait(&free_[at], lap ^ 1, abort_flag, is_s ? 117 : 121)) return false;
                              if (!ready && !mbar_wait(&st->in_full[s], (g / kRcStages) & 1, abort_flag, is_s ? 118 : 122)) return false;
                              tcgen05_fence_after();
                              const uint64_t b_desc = smem_desc_sw128(smem_u32(stages + s * kRcStageBytes + (is_s ? 0 : kTileBytes)));
#pragma unroll
                              for (uint32_t kk = 0; kk < 4; kk++) umma_f16_ts(tmem + ring0 + 64 * at, a + 8 * kk, b_desc + 2 * kk, idesc, kk);
                              umma_commit(&full[q]);
                              if (last) umma_commit(done);
                              if (++at == ring) {
                                  at = 0;
                                  lap ^= 1;
                              }
                              return true;
                          });
            }
        } else if (warp == 15 || (COL && warp == 16)) {
            // ===== out += dS . Z, dV += P . Y =====
            const bool is_dv = warp == 16;
            if (elect_one()) {
                const uint32_t idesc = instr_desc(fmt, fmt, 128, 64, 1), acc = tmem + Cols::out + (is_dv ? 64 : 0);
                uint64_t *full = is_dv ? st->p_full : st->ds_full, *free_ = is_dv ? st->p_free : st->ds_free;
                const uint32_t ring = is_dv ? 3 : Cols::dps, ring0 = is_dv ? 0 : Cols::dp;
                uint32_t at = 0;
                issue_all(is_dv ? 119 : 125, [&](uint32_t) { return true; },
                          [&](bool last, bool first, uint32_t g, uint32_t q, uint32_t ph, uint32_t kq) {
                              const uint32_t s = g % kRcStages;
                              // the accumulator still holds the item before until its epilogue has read it
                              if (first && kq >= 1 && !mbar_wait(&st->o_free, (kq - 1) & 1, abort_flag, is_dv ? 120 : 126)) return false;
                              if (!mbar_wait(&full[q], ph, abort_flag, is_dv ? 129 : 127)) return false;
                              tcgen05_fence_after();
                              const uint64_t b_desc = smem_desc_sw128(smem_u32(stages + s * kRcStageBytes + (is_dv ? kTileBytes : 0)));
                              // 16 words of each half of the others lie over the first 16 columns of that half
#pragma unroll
                              for (uint32_t kk = 0; kk < 4; kk++)
                                  umma_f16_ts(acc, tmem + ring0 + 64 * at + 32 * (kk >> 1) + 8 * (kk & 1), b_desc + 128 * kk, idesc, first && kk == 0 ? 0u : 1u);
                              umma_commit(&free_[at]);
                              umma_commit(&st->in_empty[s]);      // S and dP of this step are complete: their values made this operand
                              if (last) umma_commit(&st->o_final[kq % kRcGroups]);
                              if (++at == ring) at = 0;
                              return true;
                          });
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
        // ===== P, dS and the epilogue: own position r, every third step =====
        const uint32_t grp = warp >> 2, quarter = warp & 3;
        const uint32_t r = quarter * 32 + lane, half = r >> 6;
        const uint32_t lane_field = (quarter * 32) << 16;
        const uint32_t t_s = tmem + 64 * grp + lane_field;
        const uint64_t inside2 = pk64(p.inside, p.inside), sl2 = pk64(p.scale_log2e, p.scale_log2e);
        uint32_t turn = 0, lap = 0, ph = 0;                  // whose epilogue, times round modulo 2 (of items with blocks); this group's steps modulo 2
        uint32_t g = 0, wait = grp;                          // steps of all groups; how many of them come before this group's next
        bool alive = true;
        for (uint32_t k = 0; alive; k++) {
            const uint32_t slot = k & 1;
            if (!mbar_wait_warp(&st->list_ready[slot], (k >> 1) & 1, abort_flag, 128)) break;
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
            auto mask_word = [&](uint32_t t) -> uint64_t {
                if (!((list[t].flags >> half) & 1u)) return 0ull;
                return __ldg(p.mask + (size_t)h * p.mask_stride + (size_t)list[t].blk[half] * 64 + (r & 63));
            };
            uint32_t t = wait;                               // the first step of this item that is the group's
            uint64_t mw_next = !COL && MASK && t < T ? mask_word(t) : 0ull;
            const uint32_t list_at = smem_u32(list) + (uint32_t)offsetof(UnionEntry, flags);
            uint32_t flags = t < T ? lds_word(list_at + t * (uint32_t)sizeof(UnionEntry)) : 0u;
            for (; t < T; t += kRcGroups, ph ^= 1) {
                const uint32_t gg = g + t, s = gg % kRcStages, t_dp = tmem + Cols::dp + 64 * (COL ? gg & 1 : grp) + lane_field;
                // whether this row (column) has the step's block: the same for the whole warp
                const bool mine = __any_sync(0xffffffffu, (flags >> half) & 1u);
                const uint64_t keep = mw_next;               // rows: bit j: column j
                if (t + kRcGroups < T) {
                    flags = lds_word(list_at + (t + kRcGroups) * (uint32_t)sizeof(UnionEntry));
                    if (!COL && MASK) mw_next = mask_word(t + kRcGroups);
                }
                if (!look_or_wait(&st->s_full[grp], ph, abort_flag, 130)) { alive = false; break; }
                tcgen05_fence_after();
                if (mine) {
                    uint32_t v[64];
                    TMEM_LD_32((v), t_s);
                    TMEM_LD_32((v + 32), t_s + 32);
                    // the queries' constants and mask words came with the barrier that the product waited for; observing it makes them visible here
                    if (COL && !look_or_wait(&st->in_full[s], (gg / kRcStages) & 1, abort_flag, 131)) { alive = false; break; }
                    tmem_wait_ld();
                    if (!COL) {
                        tcgen05_fence_before();
                        mbar_arrive_warp(&st->s_free[grp], lane);
                    }
                    // P in place of the scores, fp32
                    const uint32_t nl_at = smem_u32(st->neg_lse[s]), nd_at = smem_u32(st->neg_delta[s]);
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        uint64_t n2[2] = {nl2, nl2};
                        if (COL) lds_pairs(n2, nl_at + 16 * j);
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float x0, x1;
                            up64(fma2p(pk64(__uint_as_float(v[4 * j + 2 * e]), __uint_as_float(v[4 * j + 2 * e + 1])), sl2, n2[e]), x0, x1);
                            v[4 * j + 2 * e] = __float_as_uint(ex2_approx(x0));
                            v[4 * j + 2 * e + 1] = __float_as_uint(ex2_approx(x1));
                        }
                    }
                    if (MASK) {
                        if (COL) {
                            // bit r of the words of the 64 queries: a lane looks at two, and all lanes at each where one of them is not all ones
                            const uint32_t *w = (const uint32_t *)st->mask[s][half] + (quarter & 1);
                            if (!__all_sync(0xffffffffu, (w[2 * lane] & w[2 * lane + 64]) == 0xffffffffu)) {
#pragma unroll
                                for (int j = 0; j < 64; j++)
                                    if (!((w[2 * j] >> lane) & 1u)) v[j] = 0u;
                            }
                        } else if (!__all_sync(0xffffffffu, keep == ~0ull)) {
#pragma unroll
                            for (int j = 0; j < 64; j++)
                                if (!((keep >> j) & 1u)) v[j] = 0u;
                        }
                    }
                    if (COL) {
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            uint32_t w[16];
#pragma unroll
                            for (int j = 0; j < 16; j++) w[j] = pack2(__uint_as_float(v[32 * c + 2 * j]), __uint_as_float(v[32 * c + 2 * j + 1]), BF16);
                            TMEM_ST_16(t_s + 32 * c, (w));
                        }
                        tmem_wait_st();
                        tcgen05_fence_before();
                        mbar_arrive_warp(&st->p_full[grp], lane);
                    }
                    if (!look_or_wait(&st->dp_full[grp], ph, abort_flag, 133)) { alive = false; break; }
                    tcgen05_fence_after();
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t u[32], w[16];
                        TMEM_LD_32((u), t_dp + 32 * c);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            uint64_t n2[2] = {nd2, nd2};
                            if (COL) lds_pairs(n2, nd_at + 128 * c + 16 * j);
#pragma unroll
                            for (int e = 0; e < 2; e++)
                                w[2 * j + e] = ds_pair<BF16>(u[4 * j + 2 * e], u[4 * j + 2 * e + 1], v[32 * c + 4 * j + 2 * e], v[32 * c + 4 * j + 2 * e + 1], inside2, n2[e]);
                        }
                        TMEM_ST_16(t_dp + 32 * c, (w));
                    }
                } else {
                    // a block that this row (column) has not: P and dS are zeros, whatever the products are (0 times infinity is not 0)
                    const uint32_t none[16] = {};
                    if (COL) {
                        TMEM_ST_16(t_s, (none));
                        TMEM_ST_16(t_s + 32, (none));
                        tmem_wait_st();
                        tcgen05_fence_before();
                        mbar_arrive_warp(&st->p_full[grp], lane);
                    } else {
                        mbar_arrive_warp(&st->s_free[grp], lane);
                    }
                    if (!look_or_wait(&st->dp_full[grp], ph, abort_flag, 133)) { alive = false; break; }
                    tcgen05_fence_after();
                    TMEM_ST_16(t_dp, (none));
                    TMEM_ST_16(t_dp + 32, (none));
                }
                tmem_wait_st();
                tcgen05_fence_before();
                mbar_arrive_warp(&st->ds_full[grp], lane);
            }
            if (!alive) break;
            wait = t - T;                                    // steps of the items to come before this group's next
            // the epilogue falls to the groups in turn: dQ or dK to one, dV to the next one
            const uint32_t what = grp >= turn ? grp - turn : grp + kRcGroups - turn;
            if (what < (COL ? 2u : 1u)) {
                if (T > 0 && !mbar_wait_warp(&st->o_final[turn], lap, abort_flag, 135)) break;
                tcgen05_fence_after();
                uint16_t *dst = (uint16_t *)(what ? p.out2 : p.out1) + ((size_t)b * L + (size_t)blk * 64 + (r & 63)) * p.pitch + (size_t)h * 64;
                uint32_t v[64];
                if (T > 0) {
                    const uint32_t acc = tmem + Cols::out + lane_field + 64 * what;
                    TMEM_LD_32((v), acc);
                    TMEM_LD_32((v + 32), acc + 32);
                    tmem_wait_ld();
                    tcgen05_fence_before();
                    mbar_arrive_warp(&st->o_free, lane);
                } else {
#pragma unroll
                    for (int j = 0; j < 64; j++) v[j] = 0u;  // rows and columns without blocks have zero gradients
                }
                const float factor = what ? 1.f : p.outside;
                if (blk != kNoItem)
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        uint32_t y[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) y[j] = pack2(__uint_as_float(v[8 * c + 2 * j]) * factor, __uint_as_float(v[8 * c + 2 * j + 1]) * factor, BF16);
                        *(uint4 *)(dst + 8 * c) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
            }
            if (T > 0 && ++turn == kRcGroups) {
                turn = 0;
                lap ^= 1;
            }
            g += T;
            mbar_arrive_warp(&st->list_free[slot], lane);
        }
    }

    // ---- teardown (also the way out after a timeout) ----
    tcgen05_fence_before();
    __syncthreads();
    if (st->abort_flag) {
        if (warp >= 13 && warp <= 16 && lane == 0) {
            umma_commit(&st->drained[warp - 13]);
            for (uint32_t i = 0; i < kWaitLimit && !mbar_try_wait(&st->drained[warp - 13], 0); i++) {}
        }
        if (warp == 12 && lane == 0) {
            const uint64_t t0 = clock64();
            while (clock64() - t0 < 2000000ull) {}
        }
        __syncthreads();
    }
    if (warp == 12) {
        __syncwarp();
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
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
        // what the warpgroups hand to each other is what the block is launched with: with less the workers would wait for ever
        cudaFuncAttributes attr;
        if (cudaFuncGetAttributes(&attr, recompute_tc_kernel<COL, MASK, BF16>) != cudaSuccess || attr.numRegs < 96)
            return fail("sfb_attention_backward_recompute: built with too few registers for its warpgroups");
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
    const int bf = a.dtype == SFB_BF16, sms = device_sm_count(current_device());
    const uint64_t rows = (uint64_t)p.B * p.nb_a * 64;
    CUtensorMap qm, km, vm, dm;
    if (make_map(&qm, a.q, rows, p.H, bf, 64, a.in_pitch) || make_map(&km, a.k, rows, p.H, bf, 64, a.in_pitch) || make_map(&vm, a.v, rows, p.H, bf, 64, a.in_pitch) ||
        make_map(&dm, a.dout, rows, p.H, bf, 64, a.do_pitch))
        return 1;
    RcParams row = {(const uint2 *)a.nn_lut, neg_lse, neg_delta, (const uint64_t *)a.mask, a.dq, nullptr, p.B, p.H, p.nb_a, p.blocks, p.lut_stride, p.mask_stride, (uint32_t)(sms > 0 ? sms : 1),
                    (uint32_t)a.grad_pitch, a.inside, a.scale / a.inside, a.scale * 1.4426950408889634f};
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
