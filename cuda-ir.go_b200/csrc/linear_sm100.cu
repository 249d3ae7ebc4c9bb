// linear_sm100.cu - the products of the feed-forward operators (cudair_linear,
// cudair_gated and their gradients) on persistent CTA pairs.
//
//   plain   D = act(A.B + bias) + residual, Z = A.B + bias kept if asked
//   gated   H = act(A.Wg) * (A.Wu), both products kept if asked
//   sum     dX = dG.Wg^T + dU.Wu^T: one accumulator over both contractions
//   pair    dWg = X^T.dG and dWu = X^T.dU: one grid over both problems
//
// Mathematics.  Every one of these is a sum over k of 16-bit products held in
// fp32 (TMEM), then a function of one or two accumulators element by element.
// So one mainloop serves all: what differs is which tensor maps a k-block's
// tiles come from, and what the epilogue does.
//   gated: tcgen05.mma.cta_group::2 takes the first half of its N columns from
//     the even CTA's shared memory and the second half from the odd one's.
//     The even CTA loads Wg's columns and the odd CTA Wu's, so one accumulator
//     row holds G in its first half and U in its second: the epilogue thread
//     that owns the row has both without an exchange, and X is read once.
//   sum: k-blocks past the first contraction's end come from the second pair
//     of maps and go into the same accumulator; dX is written once.
//   transposed operands (dA = dZ.B^T, dB = A^T.dZ, weights stored N x K) are
//     read as they lie in memory: the shared-memory descriptors say whether k
//     or the rows run along a tile's 128-byte swizzle rows.
//
// What bounds it: the tensor pipe, for the sizes it is meant for (M > 128;
// 2 M N K flop against 2 (MK + NK + MN) bytes).  Roles, ring and bounded waits
// are those of gemm_sm100.cu: warp 0 TMA producer, warp 1 TMEM owner and MMA
// issuer (even CTA), warps 2-5 epilogue.  Two accumulators of NT columns
// alternate, so a tile's epilogue runs under the next tile's mainloop.
//
// The epilogue writes each thread's row straight from registers, 32 bytes a
// store (a whole sector): no staging in shared memory, which goes to the ring
// instead (seven 32 KB stages with NT = 256, nine 24 KB stages with NT = 128).
#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

#include "cudair_internal.h"
#include "linear_epilogue.cuh"
#include "linear_internal.h"
#include "sm100.cuh"

namespace cudair {
namespace ffn {

constexpr int BK = 64;
constexpr int THREADS = 192;
constexpr int PM = 256;  // rows per pair tile, 128 per CTA
constexpr uint32_t A_STAGE = 128 * BK * 2;
constexpr uint32_t BAR_BYTES = 256;
constexpr int GROUP_M = 8;  // row-blocks visited together (A and B panels shared in L2)

template <int NT>
struct PairCfg {
    static constexpr int HALF = NT / 2;  // B columns per CTA
    static constexpr uint32_t B_STAGE = HALF * BK * 2;
    static constexpr uint32_t STAGE = A_STAGE + B_STAGE;
    static constexpr int STAGES = static_cast<int>((227 * 1024 - 1024 - BAR_BYTES) / STAGE);
    static constexpr uint32_t TMEM_COLS = 2 * NT;
    static constexpr size_t SMEM = 1024 + STAGES * STAGE + BAR_BYTES;
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
    static_assert(2 * STAGES * 8 + 5 * 8 + 8 <= BAR_BYTES, "barrier area");
};

struct Maps {
    CUtensorMap a[2], b[2];
};

struct PairArgs {
    int M, N;
    int num_kb;   // k-blocks of one contraction
    int parts;    // contractions per accumulator (sum: 2)
    int problems; // independent problems (pair: 2)
    int a_mn, b_mn;
    uint32_t idesc;
    int bf16, act;
    Mat d[2], z[2], residual;
    const void *bias;
    int bias16;
    unsigned int *status;
};

__device__ __forceinline__ void drain_wait(uint64_t *bar, uint32_t parity, unsigned int *status) {
    int never = 0;
    mbar_wait(bar, parity, &never, status, kSiteDrain);
}

// Tile index -> row-block and column-block: groups of GROUP_M row-blocks
// visited column by column, every other group from the far end.
__device__ __forceinline__ void tile_coords(int t, int num_m, int num_n, int &m_blk, int &n_blk) {
    const int per_group = GROUP_M * num_n;
    const int group = t / per_group;
    const int first_m = group * GROUP_M;
    const int gsize = min(num_m - first_m, GROUP_M);
    const int r = t - group * per_group;
    m_blk = first_m + r % gsize;
    n_blk = r / gsize;
    if (group & 1) n_blk = num_n - 1 - n_blk;
}

__device__ __forceinline__ void load_acc(bool any, uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    if (any) {
        tmem_ld_32x32b_x32(taddr, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
    } else {  // an empty sum (K = 0)
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0.0f;
    }
}

template <bool GATED, int NT>
__global__ void __launch_bounds__(THREADS, 1)
    product_pair_kernel(const __grid_constant__ Maps maps, const __grid_constant__ PairArgs p) {
    using Cfg = PairCfg<NT>;
    constexpr int STAGES = Cfg::STAGES;
    constexpr int TILE_N = GATED ? Cfg::HALF : NT;  // columns of D per tile
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    uint8_t *smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);  // same offset in both CTAs

    uint8_t *sA = smem;
    uint8_t *sB = smem + STAGES * A_STAGE;
    uint64_t *bars = reinterpret_cast<uint64_t *>(sB + STAGES * Cfg::B_STAGE);
    uint64_t *full = bars;                   // used in the even CTA only
    uint64_t *empty = bars + STAGES;         // both CTAs
    uint64_t *acc_full = bars + 2 * STAGES;  // both CTAs
    uint64_t *acc_empty = acc_full + 2;      // even CTA only
    uint64_t *drain = acc_empty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const uint32_t warp = warp_id(), lane = lane_id();
    const uint32_t rank = cluster_ctarank();  // 0 = even CTA (issues the MMAs)
    const int cluster = static_cast<int>(blockIdx.x >> 1);
    const int num_clusters = static_cast<int>(gridDim.x >> 1);
    const int num_m = (p.M + PM - 1) / PM;
    const int num_n = (p.N + TILE_N - 1) / TILE_N;
    const int per_problem = num_m * num_n;
    const int num_tiles = per_problem * p.problems;
    const int num_kb = p.num_kb * p.parts;
    const uint32_t peer_abort = mapa_shared(smem_u32(const_cast<int *>(abort_flag)), rank ^ 1u);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 8);  // the epilogue warps of both CTAs
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, Cfg::TMEM_COLS);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    cluster_sync();  // barriers of both CTAs initialised before any remote arrive
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    if (threadIdx.x == 0) grid_launch_dependents();  // cudair_set_gemm_pdl

    auto give_up = [&]() { st_shared_cluster_u32(peer_abort, 1u); };

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        if (lane == 0) {
            grid_dependency_wait();
            const uint64_t policy = l2_policy_evict_normal();
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (int t = cluster; t < num_tiles && ok; t += num_clusters) {
                const int prob = t / per_problem;
                int m_blk, n_blk;
                tile_coords(t - prob * per_problem, num_m, num_n, m_blk, n_blk);
                // Rows and columns beyond the matrices arrive as zeros (the
                // maps clip), so every stage carries the same bytes.
                const int m_mine = m_blk * PM + 128 * static_cast<int>(rank);
                const int n_mine = n_blk * TILE_N + (GATED ? 0 : Cfg::HALF * static_cast<int>(rank));
                for (int kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, p.status, kSiteProducerEmpty)) {
                        give_up();
                        ok = false;
                        break;
                    }
                    const uint32_t full_even = mapa_shared(smem_u32(&full[stage]), 0);
                    if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * Cfg::STAGE);
                    const int part = kb >= p.num_kb ? 1 : 0;
                    const int k0 = (kb - part * p.num_kb) * BK;
                    const int sel = prob | part;
                    const CUtensorMap *ma = &maps.a[sel];
                    const CUtensorMap *mb = &maps.b[GATED ? rank : sel];
                    uint8_t *da = sA + stage * A_STAGE, *db = sB + stage * Cfg::B_STAGE;
                    if (p.a_mn) {
                        tma_load_2d_pair(da, ma, full_even, m_mine, k0, policy);
                        tma_load_2d_pair(da + 64 * BK * 2, ma, full_even, m_mine + 64, k0, policy);
                    } else {
                        tma_load_2d_pair(da, ma, full_even, k0, m_mine, policy);
                    }
                    if (p.b_mn) {
#pragma unroll
                        for (int j = 0; j < Cfg::HALF / 64; ++j)
                            tma_load_2d_pair(db + j * 64 * BK * 2, mb, full_even, n_mine + 64 * j, k0, policy);
                    } else {
                        tma_load_2d_pair(db, mb, full_even, k0, n_mine, policy);
                    }
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // This CTA's copies complete on the even CTA's barriers, which
            // only that CTA can wait on: give them time to land.
            if (!ok) spin_ns(2000000);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- MMA issuer (even CTA) ----------------
        if (lane == 0 && rank == 0 && num_kb > 0) {
            grid_dependency_wait();
            // k along the swizzle rows: 32 bytes per 16-wide step, 8-row groups
            // 1 KB apart.  Rows along them: 16 k-rows of 128 bytes per step,
            // 64-row blocks 8 KB apart.
            const uint32_t a_step = p.a_mn ? 2048u : 32u, a_lbo = p.a_mn ? 64u * BK * 2 : 16u;
            const uint32_t b_step = p.b_mn ? 2048u : 32u, b_lbo = p.b_mn ? 64u * BK * 2 : 16u;
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
            bool ok = true, issued_any = false;
            for (int t = cluster; t < num_tiles && ok; t += num_clusters) {
                if (!mbar_wait(&acc_empty[acc], acc_phase ^ 1u, abort_flag, p.status, kSiteMmaAccEmpty)) {
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                for (int kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait(&full[stage], phase, abort_flag, p.status, kSiteMmaFull)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t a_base = smem_u32(sA + stage * A_STAGE);
                    const uint32_t b_base = smem_u32(sB + stage * Cfg::B_STAGE);
#pragma unroll
                    for (int kk = 0; kk < BK / 16; ++kk)
                        umma_f16_ss_pair(tmem_base + acc * NT, smem_desc_sw128(a_base + kk * a_step, a_lbo, 1024),
                                         smem_desc_sw128(b_base + kk * b_step, b_lbo, 1024), p.idesc,
                                         (kb | kk) != 0 ? 1u : 0u);
                    issued_any = true;
                    umma_commit_pair_multicast(&empty[stage], 0x3);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                umma_commit_pair_multicast(&acc_full[acc], 0x3);
                acc ^= 1u;
                if (acc == 0) acc_phase ^= 1u;
            }
            if (!ok) {
                give_up();
                if (issued_any) {
                    umma_commit_pair_local(drain);
                    drain_wait(drain, 0, p.status);
                }
            }
        }
        __syncwarp();
    } else {
        // ---------------- epilogue (warps 2..5, both CTAs) ----------------
        grid_dependency_wait();  // the outputs may be the preceding kernel's inputs
        const uint32_t q = warp & 3u;  // the TMEM lane quarter this warp may read
        const bool bf16 = p.bf16 != 0;
        uint32_t acc = 0, acc_phase = 0;
        for (int t = cluster; t < num_tiles; t += num_clusters) {
            const int prob = t / per_problem;
            int m_blk, n_blk;
            tile_coords(t - prob * per_problem, num_m, num_n, m_blk, n_blk);
            const int row0 = m_blk * PM + 128 * static_cast<int>(rank) + static_cast<int>(q * 32);
            const int row = row0 + static_cast<int>(lane);
            const int n0 = n_blk * TILE_N;
            const bool live = row < p.M;
            if (num_kb > 0) {
                if (!mbar_wait(&acc_full[acc], acc_phase, abort_flag, p.status, kSiteEpilogueAccFull)) {
                    give_up();
                    break;
                }
                tc_fence_after_sync();
            }
            const uint32_t t_row = tmem_base + ((q * 32u) << 16) + acc * NT;
            if (row0 < p.M) {  // the whole warp: TMEM loads are warp-wide
#pragma unroll 1
                for (int c = 0; c < TILE_N; c += 32) {
                    const int col = n0 + c;
                    if (col >= p.N) break;
                    float v[32];
                    load_acc(num_kb > 0, t_row + c, v);
                    if (GATED) {
                        float u[32];
                        load_acc(num_kb > 0, t_row + Cfg::HALF + c, u);
                        if (p.z[0].p && live) {
                            store_row32(p.z[0], row, col, p.N, bf16, v);
                            store_row32(p.z[1], row, col, p.N, bf16, u);
                        }
                        with_act(p.act, [&](auto tag) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = act_value<decltype(tag)::value>(v[j]) * u[j];
                        });
                    } else {
                        if (p.bias) {
                            // Lane l reads column l's bias; a shuffle hands it on.
                            float b = 0.0f;
                            const int bc = col + static_cast<int>(lane);
                            if (bc < p.N)
                                b = p.bias16 ? from16(static_cast<const uint16_t *>(p.bias)[bc], bf16)
                                             : static_cast<const float *>(p.bias)[bc];
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] += __shfl_sync(0xFFFFFFFFu, b, j);
                        }
                        if (p.z[0].p && live) store_row32(p.z[0], row, col, p.N, bf16, v);
                        if (p.act != CUDAIR_ACT_NONE)
                            with_act(p.act, [&](auto tag) {
#pragma unroll
                                for (int j = 0; j < 32; ++j) v[j] = act_value<decltype(tag)::value>(v[j]);
                            });
                        if (p.residual.p && live) add_row32(p.residual, row, col, p.N, bf16, v);
                    }
                    if (live) store_row32(p.d[prob], row, col, p.N, bf16, v);
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (num_kb > 0 && lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[acc]), 0));
            acc ^= 1u;
            if (acc == 0) acc_phase ^= 1u;
        }
        __syncwarp();
    }

    // Neither CTA leaves (or frees TMEM) while the other may still touch its
    // shared memory or TMEM.
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
    }
}

// ---- host side ---------------------------------------------------------------------

int operand_map(CUtensorMap *out, const Operand &o, int64_t rows, int64_t depth, uint32_t box_rows, bool bf16) {
    const uint64_t dims[2] = {static_cast<uint64_t>(o.mn ? rows : depth),
                              static_cast<uint64_t>(o.mn ? depth : rows)};
    const uint64_t strides[1] = {static_cast<uint64_t>(o.ld) * 2};
    const uint32_t box[2] = {64, o.mn ? 64u : box_rows};
    return encode_tiled_internal(out, bf16 ? CUDAIR_TENSOR_MAP_BFLOAT16 : CUDAIR_TENSOR_MAP_FLOAT16, 2,
                                 reinterpret_cast<uint64_t>(o.p), dims, strides, box, nullptr,
                                 CUDAIR_INTERLEAVE_NONE, CUDAIR_SWIZZLE_128B, CUDAIR_L2_PROMOTION_256B,
                                 CUDAIR_OOB_FILL_NONE);
}

namespace {

std::mutex g_pair_mu;
int g_pairs[64];  // CTA pairs resident at once, per device (0: not asked yet)

template <bool GATED, int NT>
cudaError_t prepare_kernel(int sm_count, int *clusters) {
    cudaError_t e = cudaFuncSetAttribute(product_pair_kernel<GATED, NT>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(PairCfg<NT>::SMEM));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (sm_count / 2)), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = PairCfg<NT>::SMEM;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaOccupancyMaxActiveClusters(clusters, product_pair_kernel<GATED, NT>, &cfg);
}

int resident_pairs(int sm_count, int *pairs) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_error(e, "cudaGetDevice");
    std::lock_guard<std::mutex> lk(g_pair_mu);  // dev is in 0..63: the device check passed
    if (g_pairs[dev] == 0) {
        int n = 0;
        if ((e = prepare_kernel<false, 256>(sm_count, &n)) != cudaSuccess ||
            (e = prepare_kernel<true, 256>(sm_count, &n)) != cudaSuccess)
            return cuda_error(e, "product_pair_kernel set-up");
        if (n < 1) return set_error(CUDAIR_ERR_CUDA, "cudair: no CTA pair of the linear kernels fits this device");
        g_pairs[dev] = n;
    }
    *pairs = g_pairs[dev];
    return CUDAIR_OK;
}

template <bool GATED, int NT>
cudaError_t launch_pair(const Maps &maps, const PairArgs &args, int pairs, bool pdl, cudaStream_t stream) {
    constexpr int TILE_N = GATED ? NT / 2 : NT;
    const int64_t tiles = static_cast<int64_t>((args.M + static_cast<int64_t>(PM) - 1) / PM) *
                          ((args.N + static_cast<int64_t>(TILE_N) - 1) / TILE_N) * args.problems;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs)), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = PairCfg<NT>::SMEM;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, product_pair_kernel<GATED, NT>, maps, args);
}

}  // namespace

int product_pair_launch(const Product &p, int sm_count, unsigned int *status, cudaStream_t stream) {
    int pairs = 0;
    int rc = resident_pairs(sm_count, &pairs);
    if (rc != CUDAIR_OK) return rc;
    constexpr int NT = 256;
    alignas(64) Maps maps = {};
    const bool gated = p.form == Form::gated;
    if (p.K > 0) {
        const int as = p.form == Form::plain || gated ? 1 : 2, bs = p.form == Form::plain ? 1 : 2;
        for (int i = 0; i < as; ++i)
            if ((rc = operand_map(&maps.a[i], p.a[i], p.M, p.K, 128, p.bf16)) != CUDAIR_OK) return rc;
        for (int i = 0; i < bs; ++i)
            if ((rc = operand_map(&maps.b[i], p.b[i], p.N, p.K, NT / 2, p.bf16)) != CUDAIR_OK) return rc;
    }
    PairArgs args = {};
    args.M = static_cast<int>(p.M);
    args.N = static_cast<int>(p.N);
    args.num_kb = static_cast<int>((p.K + BK - 1) / BK);
    args.parts = p.form == Form::sum ? 2 : 1;
    args.problems = p.form == Form::pair ? 2 : 1;
    args.a_mn = p.a[0].mn;
    args.b_mn = p.b[0].mn;
    args.idesc = idesc_f16_f32(PM, NT, p.a[0].mn, p.b[0].mn, p.bf16);
    args.bf16 = p.bf16;
    args.act = p.act;
    for (int i = 0; i < 2; ++i) {
        args.d[i] = mat_of(p.d[i]);
        args.z[i] = mat_of(p.z[i]);
    }
    args.residual = mat_of(p.residual);
    args.bias = p.bias;
    args.bias16 = p.bias16;
    args.status = status;
    const cudaError_t e = gated ? launch_pair<true, NT>(maps, args, pairs, p.pdl(), stream)
                                : launch_pair<false, NT>(maps, args, pairs, p.pdl(), stream);
    return e == cudaSuccess ? CUDAIR_OK : cuda_error(e, "product_pair_kernel launch");
}

}  // namespace ffn
}  // namespace cudair
