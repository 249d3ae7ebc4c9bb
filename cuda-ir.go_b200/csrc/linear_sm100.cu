// linear_sm100.cu - the products of the feed-forward operators (cudair_linear,
// cudair_gated and their gradients) on persistent CTA pairs.
//
//   linear    D = act(A.B + bias) + residual, Z = A.B + bias kept if asked
//   gated     H = act(A.Wg) * (A.Wu), both products kept if asked
//   gradients dA = dZ.B^T and dB = A^T.dZ; dX = dG.Wg^T + dU.Wu^T, dWg = X^T.dG
//             and dWu = X^T.dU: up to three jobs in one launch
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
//   dX: k-blocks past the first contraction's end come from the second pair of
//     maps and go into the same accumulator; dX is written once.
//   several jobs: their tiles are dealt out together, long ones first, so that
//     no job ends on a wave of its own that leaves SMs idle.
//   transposed operands (dA = dZ.B^T, dB = A^T.dZ, weights stored N x K) are
//     read as they lie in memory: the shared-memory descriptors say whether k
//     or the rows run along a tile's 128-byte swizzle rows.
//
// What bounds it: the tensor pipe, for the sizes it is meant for (M > 128;
// 2 M N K flop against 2 (MK + NK + MN) bytes).  Roles, ring and bounded waits
// are those of gemm_sm100.cu, with a second producer: warp 0 loads A, warp 10 loads B
// (one thread issuing the four copies of a k-block whose operands both have rows along
// memory fell behind: weight gradients of 5632 x 2048 over 1024 rows 42.6 -> 37
// us), warp 1 TMEM owner and MMA issuer (even CTA), warps 2-9 epilogue (two
// per lane quarter).  Two accumulators of 256 columns alternate, so a tile's
// epilogue runs under the next tile's mainloop; or one of 512 columns is handed
// over in halves.
//
// Below that bound, what limits a k-block is the way from L2: 32 KB into an SM
// in 0.29 us with few SMs busy (59 bytes a clock), 0.37 us with all (13 TB/s
// in all).  Outputs of few tiles with a long contraction are short of SMs: a tile's
// contraction is not cut here (512 x 4096 x 4096: 44 tiles, 60 SMs idle, 26 us).
// With a short contraction the epilogue is the longer part (8192 x 14336 x 512:
// eight k-blocks are 3 us of a tile's 4.2 without an activation): a warp loads,
// computes and stores one chunk after another.
//
// The epilogue writes each thread's row straight from registers, 32 bytes a
// store (a whole sector): no staging in shared memory, which goes to the ring
// instead (seven 32 KB stages, or four of 48 KB).  The residual's columns are
// requested ahead of their use, the first before the accumulator is waited for
// (8192^3 in wide tiles with bias, relu and residual: 947 us with four warps
// and loads where they are used, 905 us).
#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>
#include <utility>

#include "cudair_internal.h"
#include "linear_epilogue.cuh"
#include "linear_internal.h"
#include "sm100.cuh"

namespace cudair {
namespace ffn {

constexpr int BK = 64;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS + 32;  // the last warp loads B
constexpr int PM = 256;  // rows per pair tile, 128 per CTA
constexpr uint32_t A_STAGE = 128 * BK * 2;
constexpr uint32_t BAR_BYTES = 256 + 512;  // barriers, and the jobs' arguments
constexpr int GROUP_M = 8;  // row-blocks visited together (A and B panels shared in L2)

// A tile takes NB accumulator blocks of bn columns (the MMA's N, at most BN).
// NB = 1: two accumulators that alternate.  NB = 2: one of up to 512 columns
// that fills TMEM, for a quarter fewer operand bytes per flop.  bn is chosen per
// call so that the tiles fill whole waves (see tile_time).
constexpr int BN = 256;
template <int NB>
struct PairCfg {
    static constexpr uint32_t B_BLOCK = BN / 2 * BK * 2;  // this CTA's half of a block
    static constexpr uint32_t B_STAGE = NB * B_BLOCK;
    static constexpr uint32_t STAGE = A_STAGE + B_STAGE;
    static constexpr int STAGES = static_cast<int>((227 * 1024 - 1024 - BAR_BYTES) / STAGE);
    static constexpr size_t SMEM = 1024 + STAGES * STAGE + BAR_BYTES;
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
    static_assert(2 * STAGES * 8 + 5 * 8 + 8 <= 256, "barrier area");
};
constexpr uint32_t TMEM_COLS = 512;

struct Maps {
    CUtensorMap a[kMaxJobs][2], b[kMaxJobs][2];
};

// Division by a fixed d of n < 2^31: (n mul) >> (31 + l) with l = ceil(log2 d)
// and mul = ceil(2^(31 + l) / d), which is exact there.
struct Div {
    uint32_t mul, shift;
    __device__ __forceinline__ int operator()(int n) const {
        return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift);
    }
};

struct JobArgs {
    Mat d;
    int M, N, num_m, num_n;
    int num_kb, all_kb;  // k-blocks of one contraction, and of all that an accumulator sums
    int a_mn, b_mn;
    uint32_t idesc;
    int per_group;       // tiles of a group of GROUP_M row-blocks
    Div group, last;     // by per_group; by the row-blocks of the last group
    uint32_t bytes;      // both CTAs' copies of a k-block
};
static_assert(sizeof(JobArgs) % 4 == 0, "copied by words");

// The tiles of all jobs are numbered through, job after job.  Job 0 has the
// longest ones: pair c takes its tiles c, c + C, ... (C pairs), so the first
// pairs get one more than the others.  Of the rest every pair takes `rounds`, a
// round that is not full from the last pair down, and the pairs with one long
// tile less share what remains: all end at about the same time.
struct PairArgs {
    JobArgs job[kMaxJobs];
    int first[kMaxJobs + 1];  // a job's first tile; the end
    int own, more;            // tiles of job 0 of every pair; pairs that take one more
    int rounds;
    int bn;  // columns of an accumulator block, a multiple of 32 (gated: of 64)
    int act;
    Mat z[2], residual;
    const void *bias;
    int bias16;
    unsigned int *status;
};

// The i-th tile of pair c of C, -1 after its last.
__device__ __forceinline__ int tile_of(const PairArgs &p, int i, int c, int C) {
    const int n0 = p.first[1], end = p.first[kMaxJobs], more = p.more;
    const int own = p.own + (c < more ? 1 : 0);
    if (i < own) return i * C + c;
    const int j = i - own;
    int t = end;
    if (j < p.rounds)
        t = n0 + j * C + C - 1 - c;
    else if (c >= more)
        t = n0 + p.rounds * C + (j - p.rounds) * (C - more) + C - 1 - c;
    return t < end ? t : -1;
}
template <int V>
struct Index {
    static constexpr int value = V;
};
__device__ __forceinline__ int job_of(const PairArgs &p, int t) {
    return (t >= p.first[1] ? 1 : 0) + (t >= p.first[2] ? 1 : 0);
}

__device__ __forceinline__ void drain_wait(uint64_t *bar, uint32_t parity, unsigned int *status) {
    int never = 0;
    mbar_wait(bar, parity, &never, status, kSiteDrain);
}

// Tile index -> row-block and column-block: groups of GROUP_M row-blocks
// visited column by column, every other group from the far end.
__device__ __forceinline__ void tile_coords(const JobArgs &job, int t, int &m_blk, int &n_blk) {
    const int group = job.group(t);
    const int first_m = group * GROUP_M;
    const int r = t - group * job.per_group;
    const int left = job.num_m - first_m;
    n_blk = left >= GROUP_M ? r / GROUP_M : job.last(r);
    m_blk = first_m + r - n_blk * (left >= GROUP_M ? GROUP_M : left);
    if (group & 1) n_blk = job.num_n - 1 - n_blk;
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

// Arrives on an mbarrier of the cluster without ordering memory: what it hands
// over is tensor memory whose loads have completed.  (A releasing arrival first waits
// for the warp's stores to D: 3500 clocks a tile.)
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// Two warps share an accumulator block's 32 rows of a TMEM lane quarter; each
// takes about half of its columns of D, in chunks of 32 and at most this many.
template <bool GATED>
constexpr int kWarpCols = (GATED ? BN / 2 : BN) / (EPI_WARPS / 4);

// One warp's 32 rows (one per lane) and `cols` columns from n0 on; t_row is
// where they start in TMEM.  `next` holds the residual's first 32 columns, and lane
// l of `bias` the warp's columns l, l + 32, ...: both were requested before the
// accumulator was waited for.  The residual's further columns are requested while the
// ones before them are worked on.
template <bool GATED, bool bf16>
__device__ __forceinline__ void epilogue_block(const PairArgs &p, const JobArgs &job, uint32_t t_row, int row,
                                               int n0, int cols, bool live, bool any, Row32 &next,
                                               const float (&bias)[kWarpCols<GATED> / 32], uint32_t acc_empty) {
#pragma unroll 1
    for (int c = 0; c < cols; c += 32) {
        const int col = n0 + c;
        if (col >= job.N) break;
        float v[32], u[GATED ? 32 : 1];
        load_acc(any, t_row + c, v);
        if constexpr (GATED) load_acc(any, t_row + p.bn / 2 + c, u);
        // The last columns are read: the block goes back to the MMA warp while
        // they are worked on.
        if (any && (c + 32 >= cols || col + 32 >= job.N)) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane_id() == 0) mbar_arrive_cluster_relaxed(acc_empty);
        }
        if constexpr (GATED) {
            if (p.z[0].p && live) {
                store_row32(p.z[0], row, col, job.N, bf16, v);
                store_row32(p.z[1], row, col, job.N, bf16, u);
            }
            with_act(p.act, [&](auto tag) {
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    act_pair<decltype(tag)::value>(v[j], v[j + 1]);
                    unpair(mul2(pair(v[j], v[j + 1]), pair(u[j], u[j + 1])), v[j], v[j + 1]);
                }
            });
        } else {
            if (p.bias) {
                float mine = bias[0];
#pragma unroll
                for (int k = 1; k < kWarpCols<GATED> / 32; ++k)
                    if (c == 32 * k) mine = bias[k];
#pragma unroll
                for (int j = 0; j < 32; j += 2)
                    unpair(add2(pair(v[j], v[j + 1]),
                                pair(__shfl_sync(0xFFFFFFFFu, mine, j), __shfl_sync(0xFFFFFFFFu, mine, j + 1))),
                           v[j], v[j + 1]);
            }
            if (p.z[0].p && live) store_row32(p.z[0], row, col, job.N, bf16, v);
            if (p.act != CUDAIR_ACT_NONE)
                with_act(p.act, [&](auto tag) {
#pragma unroll
                    for (int j = 0; j < 32; j += 2) act_pair<decltype(tag)::value>(v[j], v[j + 1]);
                });
            if (p.residual.p && live) {
                add_row32(next, p.residual.f32, bf16, v);
                if (c + 32 < cols && col + 32 < job.N)
                    fetch_row32(p.residual, row, col + 32, job.N, next);
            }
        }
        if (live) store_row32(job.d, row, col, job.N, bf16, v);
    }
}

template <bool GATED, int NB, bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
    product_pair_kernel(const __grid_constant__ Maps maps, const __grid_constant__ PairArgs p) {
    using Cfg = PairCfg<NB>;
    constexpr int STAGES = Cfg::STAGES;
    const int half = p.bn / 2;                  // a CTA's columns of B per block
    const int block_n = GATED ? half : p.bn;    // columns of D per accumulator block
    const int tile_n = NB * block_n;            // ... and per tile
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
    // The jobs' arguments: indexed here they are read from shared memory, where
    // an indexed place in the arguments themselves is read through memory, again at
    // every use between asm statements (gated 4096 x 14336 x 4096: 750 against 641 us).
    JobArgs *jobs = reinterpret_cast<JobArgs *>(reinterpret_cast<uint8_t *>(bars) + 256);
    static_assert(kMaxJobs * sizeof(JobArgs) <= BAR_BYTES - 256, "jobs area");

    const uint32_t warp = warp_id(), lane = lane_id();
    const uint32_t rank = cluster_ctarank();  // 0 = even CTA (issues the MMAs)
    const int cluster = static_cast<int>(blockIdx.x >> 1);
    const int num_clusters = static_cast<int>(gridDim.x >> 1);
    const uint32_t peer_abort = mapa_shared(smem_u32(const_cast<int *>(abort_flag)), rank ^ 1u);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 2 * EPI_WARPS);  // those of both CTAs
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, TMEM_COLS);
        tmem_relinquish_pair();
    }
    if (threadIdx.x < kMaxJobs * sizeof(JobArgs) / 4)
        reinterpret_cast<uint32_t *>(jobs)[threadIdx.x] = reinterpret_cast<const uint32_t *>(p.job)[threadIdx.x];
    __syncwarp();
    tc_fence_before_sync();
    cluster_sync();  // barriers of both CTAs initialised before any remote arrive
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    auto give_up = [&]() { st_shared_cluster_u32(peer_abort, 1u); };

    if (warp == 0 || warp == 2 + EPI_WARPS) {
        // ---------------- TMA producers (both CTAs): A, B ----------------
        if (lane == 0) {
            grid_dependency_wait();
            // Only now may the next kernel of the stream start (cudair_set_gemm_pdl):
            // then all before this one have ended, and that kernel may request
            // weights that this one does not write before it waits for this one.
            if (warp == 0) grid_launch_dependents();
            const uint64_t policy = l2_policy_evict_normal();
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            // One operand of one tile of job J.  Both are template parameters:
            // with an indexed tensor map, or copies under a condition of the
            // thread's, the compiler cannot tell that what the copy instruction needs
            // is uniform, and the loop that makes it so sets the pace (1024 x
            // 4096 x 8192: 60 us against 52).
            auto load_tile = [&](auto operand, auto tag, int t) -> bool {
                constexpr bool FOR_A = decltype(operand)::value == 0;
                constexpr int J = decltype(tag)::value;
                const JobArgs &job = p.job[J];
                const int num_kb = job.all_kb;
                int m_blk, n_blk;
                tile_coords(job, t, m_blk, n_blk);
                const CUtensorMap *map = FOR_A ? &maps.a[J][0] : &maps.b[J][GATED ? rank : 0];
                // Rows and columns beyond the matrices arrive as zeros (the
                // maps clip), so every stage carries the same bytes.
                const int m_mine = m_blk * PM + 128 * static_cast<int>(rank);
                // A block takes the first half of its columns of B from the even
                // CTA, the others from the odd one: of one weight, or (gated)
                // of the two.
                const int n_mine = n_blk * tile_n + (GATED ? 0 : half * static_cast<int>(rank));
                int k0 = 0;
                for (int kb = 0; kb < num_kb; ++kb, k0 += BK) {
                    if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, p.status, kSiteProducerEmpty)) return false;
                    const uint32_t full_even = mapa_shared(smem_u32(&full[stage]), 0);
                    if (FOR_A && rank == 0) mbar_arrive_expect_tx(&full[stage], job.bytes);
                    if (!GATED && kb == job.num_kb) {  // the second contraction
                        ++map;
                        k0 = 0;
                    }
                    if constexpr (FOR_A) {
                        uint8_t *da = sA + stage * A_STAGE;
                        if (job.a_mn) {
                            tma_load_2d_pair(da, map, full_even, m_mine, k0, policy);
                            tma_load_2d_pair(da + 64 * BK * 2, map, full_even, m_mine + 64, k0, policy);
                        } else {
                            tma_load_2d_pair(da, map, full_even, k0, m_mine, policy);
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < NB; ++h) {
                            uint8_t *db = sB + stage * Cfg::B_STAGE + h * Cfg::B_BLOCK;
                            const int n = n_mine + h * block_n;
                            if (job.b_mn) {
                                tma_load_2d_pair(db, map, full_even, n, k0, policy);
                                if (half > 64) tma_load_2d_pair(db + 64 * BK * 2, map, full_even, n + 64, k0, policy);
                            } else {
                                tma_load_2d_pair(db, map, full_even, k0, n, policy);
                            }
                        }
                    }
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                return true;
            };
            auto load_all = [&](auto operand) {
                for (int i = 0, t; ok && (t = tile_of(p, i, cluster, num_clusters)) >= 0; ++i) {
                    if (GATED || t < p.first[1])
                        ok = load_tile(operand, Index<0>{}, t);
                    else if (t < p.first[2])
                        ok = load_tile(operand, Index<1>{}, t - p.first[1]);
                    else
                        ok = load_tile(operand, Index<2>{}, t - p.first[2]);
                }
            };
            if (warp == 0)
                load_all(Index<0>{});
            else
                load_all(Index<1>{});
            if (!ok) {
                give_up();
                // This CTA's copies complete on the even CTA's barriers, which
                // only that CTA can wait on: give them time to land.
                spin_ns(2000000);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- MMA issuer (even CTA) ----------------
        if (lane == 0 && rank == 0) {
            grid_dependency_wait();
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
            bool ok = true, issued_any = false;
            // k along the swizzle rows: 32 bytes per 16-wide step, 8-row groups
            // 1 KB apart.  Rows along them: 16 k-rows of 128 bytes per step,
            // 64-row blocks 8 KB apart.
            uint32_t a_step = 0, a_lbo = 0, b_step = 0, b_lbo = 0, idesc = 0;
            // The MMAs of the k-block in stage st into blocks [lo, hi) of the
            // accumulator; `first` overwrites it.
            auto issue = [&](uint32_t st, bool first, int lo, int hi) {
                const uint32_t a_base = smem_u32(sA + st * A_STAGE);
                const uint32_t b_base = smem_u32(sB + st * Cfg::B_STAGE);
#pragma unroll
                for (int kk = 0; kk < BK / 16; ++kk) {
                    const uint64_t a_desc = smem_desc_sw128(a_base + kk * a_step, a_lbo, 1024);
                    for (int h = lo; h < hi; ++h)
                        umma_f16_ss_pair(tmem_base + (acc + h) * BN, a_desc,
                                         smem_desc_sw128(b_base + h * Cfg::B_BLOCK + kk * b_step, b_lbo, 1024),
                                         idesc, first && kk == 0 ? 0u : 1u);
                }
                issued_any = true;
            };
            auto wait_full = [&]() {
                if (!mbar_wait(&full[stage], phase, abort_flag, p.status, kSiteMmaFull)) return false;
                tc_fence_after_sync();
                return true;
            };
            auto wait_acc = [&](uint32_t b) {
                if (!mbar_wait(&acc_empty[b], acc_phase ^ 1u, abort_flag, p.status, kSiteMmaAccEmpty)) return false;
                tc_fence_after_sync();
                return true;
            };
            auto advance = [&]() {
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            };
            // k-blocks [lo, hi), all blocks, releasing each stage.
            auto plain = [&](int lo, int hi) {
                for (int kb = lo; kb < hi; ++kb) {
                    if (!wait_full()) return false;
                    issue(stage, kb == 0, 0, NB);
                    umma_commit_pair_multicast(&empty[stage], 0x3);
                    advance();
                }
                return true;
            };
            // NB = 2: one accumulator cannot be drained under the next tile's
            // mainloop, so its two blocks are handed over separately.  In a
            // tile's first and last ring-full of k-blocks, block 0 is
            // multiplied for all of them before block 1: block 0's epilogue
            // starts while block 1's last MMAs run, and the next tile starts
            // on block 0 while block 1 is being drained.
            auto window = [&](int lo, int hi, bool first, bool last) {
                const uint32_t st0 = stage;
                if (first && !wait_acc(0)) return false;
                for (int kb = lo; kb < hi; ++kb) {
                    if (!wait_full()) return false;
                    issue(stage, kb == 0, 0, 1);
                    advance();
                }
                if (last) umma_commit_pair_multicast(&acc_full[0], 0x3);
                if (first && !wait_acc(1)) return false;
                uint32_t st = st0;
                for (int kb = lo; kb < hi; ++kb) {
                    issue(st, kb == 0, 1, 2);
                    umma_commit_pair_multicast(&empty[st], 0x3);
                    if (++st == STAGES) st = 0;
                }
                if (last) umma_commit_pair_multicast(&acc_full[1], 0x3);
                return true;
            };
            for (int i = 0, t; ok && (t = tile_of(p, i, cluster, num_clusters)) >= 0; ++i) {
                const JobArgs &job = jobs[job_of(p, t)];
                const int num_kb = job.all_kb;
                if (num_kb == 0) continue;  // an empty sum: the epilogue's alone
                a_step = job.a_mn ? 2048u : 32u;
                a_lbo = job.a_mn ? 64u * BK * 2 : 16u;
                b_step = job.b_mn ? 2048u : 32u;
                b_lbo = job.b_mn ? 64u * BK * 2 : 16u;
                idesc = job.idesc;
                if (NB == 2) {
                    const int head = min(STAGES, num_kb), tail = max(head, num_kb - STAGES);
                    ok = window(0, head, true, head == num_kb) && plain(head, tail) &&
                         (tail == num_kb || window(tail, num_kb, false, true));
                    acc_phase ^= 1u;
                } else {
                    ok = wait_acc(acc) && plain(0, num_kb);
                    if (!ok) break;
                    umma_commit_pair_multicast(&acc_full[acc], 0x3);
                    acc ^= 1u;
                    if (acc == 0) acc_phase ^= 1u;
                }
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
        // ---------------- epilogue (warps 2..9, both CTAs) ----------------
        grid_dependency_wait();  // the outputs may be the preceding kernel's inputs
        const uint32_t q = warp & 3u;  // the TMEM lane quarter this warp may read
        // Which of the quarter's warps this is, and its columns of a block.
        const int side = static_cast<int>(warp - 2u) / 4;
        const int split_at = (block_n / 32 + 1) / 2 * 32;
        const int first_col = side ? split_at : 0, cols = side ? block_n - split_at : split_at;
        uint32_t acc = 0, acc_phase = 0;
        for (int i = 0, t; (t = tile_of(p, i, cluster, num_clusters)) >= 0; ++i) {
            const int j = job_of(p, t);
            const JobArgs job = jobs[j];
            const int num_kb = job.all_kb;
            int m_blk, n_blk;
            tile_coords(job, t - p.first[j], m_blk, n_blk);
            const int row0 = m_blk * PM + 128 * static_cast<int>(rank) + static_cast<int>(q * 32);
            const int row = row0 + static_cast<int>(lane);
            const int n0 = n_blk * tile_n;
            const bool live = row < job.M;
            bool aborted = false;
#pragma unroll 1
            for (int h = 0; h < NB; ++h) {
                const uint32_t bar = acc + h;  // NB = 2: block h's own barriers
                const int col0 = n0 + h * block_n + first_col;
                Row32 res;
                float bias[kWarpCols<GATED> / 32] = {};
                if (!GATED && p.bias) {
#pragma unroll
                    for (int k = 0; k < kWarpCols<GATED> / 32; ++k) {
                        const int bc = col0 + 32 * k + static_cast<int>(lane);
                        if (bc < job.N)
                            bias[k] = p.bias16 ? from16(static_cast<const uint16_t *>(p.bias)[bc], BF16)
                                               : static_cast<const float *>(p.bias)[bc];
                    }
                }
                if (!GATED && p.residual.p && live && col0 < job.N)
                    fetch_row32(p.residual, row, col0, job.N, res);
                if (num_kb > 0) {
                    // The warp stops as one: TMEM loads are warp-wide.
                    if (!__all_sync(0xFFFFFFFFu, mbar_wait(&acc_full[bar], acc_phase, abort_flag, p.status,
                                                           kSiteEpilogueAccFull))) {
                        give_up();
                        aborted = true;
                        break;
                    }
                    tc_fence_after_sync();
                }
                const uint32_t mine_empty = mapa_shared(smem_u32(&acc_empty[bar]), 0);
                const uint32_t t_row = tmem_base + ((q * 32u) << 16) + bar * BN + first_col;
                if (row0 < job.M && col0 < job.N)  // the whole warp: TMEM loads are warp-wide
                    epilogue_block<GATED, BF16>(p, job, t_row, row, col0, cols, live, num_kb > 0, res, bias,
                                                mine_empty);
                else if (num_kb > 0 && lane == 0)  // nothing of it lies in D
                    mbar_arrive_cluster_relaxed(mine_empty);
                __syncwarp();
            }
            if (aborted) break;
            if (num_kb > 0) {
                if (NB == 1) acc ^= 1u;
                if (acc == 0) acc_phase ^= 1u;
            }
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
        tmem_dealloc_pair(tmem_base, TMEM_COLS);
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

Div divide_by(int d) {
    Div v;
    uint32_t l = 0;
    while ((1ll << l) < d) ++l;
    v.shift = 31 + l;
    v.mul = static_cast<uint32_t>(((1ull << v.shift) + static_cast<uint64_t>(d) - 1) / static_cast<uint64_t>(d));
    return v;
}

std::mutex g_pair_mu;
int g_pairs[64];  // CTA pairs resident at once, per device (0: not asked yet)

template <bool GATED, int NB, bool BF16>
cudaError_t prepare_kernel(int sm_count, int *clusters) {
    cudaError_t e = cudaFuncSetAttribute(product_pair_kernel<GATED, NB, BF16>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(PairCfg<NB>::SMEM));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (sm_count / 2)), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = PairCfg<NB>::SMEM;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaOccupancyMaxActiveClusters(clusters, product_pair_kernel<GATED, NB, BF16>, &cfg);
}

int resident_pairs(int sm_count, int *pairs) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_error(e, "cudaGetDevice");
    std::lock_guard<std::mutex> lk(g_pair_mu);  // dev is in 0..63: the device check passed
    if (g_pairs[dev] == 0) {
        int n = 0;
        if ((e = prepare_kernel<false, 1, false>(sm_count, &n)) != cudaSuccess ||
            (e = prepare_kernel<false, 1, true>(sm_count, &n)) != cudaSuccess ||
            (e = prepare_kernel<false, 2, false>(sm_count, &n)) != cudaSuccess ||
            (e = prepare_kernel<false, 2, true>(sm_count, &n)) != cudaSuccess ||
            (e = prepare_kernel<true, 1, false>(sm_count, &n)) != cudaSuccess ||
            (e = prepare_kernel<true, 1, true>(sm_count, &n)) != cudaSuccess ||
            (e = prepare_kernel<true, 2, false>(sm_count, &n)) != cudaSuccess ||
            (e = prepare_kernel<true, 2, true>(sm_count, &n)) != cudaSuccess)
            return cuda_error(e, "product_pair_kernel set-up");
        if (n < 1) return set_error(CUDAIR_ERR_CUDA, "cudair: no CTA pair of the linear kernels fits this device");
        g_pairs[dev] = n;
    }
    *pairs = g_pairs[dev];
    return CUDAIR_OK;
}

// The width of a tile, NB blocks of bn accumulator columns, and the time of one
// of its k-blocks in microseconds, in four waves and in a single one, which runs at
// a higher clock (72 tiles of 2048 rows a wave, K 1024 and 4096).  Below 192 columns
// a tile gains nothing more: 0.30 for 160 columns and 0.29 for 128.  What the widths are for is whole
// waves: 800 x 5504 x 6208 is 88 tiles of 256 columns, two waves on 74 pairs, but
// 60 of 384.
struct Width {
    int nb, bn;
    double many, single;
};
constexpr Width kWidths[] = {{1, 256, 0.371, 0.319}, {1, 224, 0.343, 0.317}, {1, 192, 0.323, 0.308},
                             {2, 256, 0.731, 0.673}, {2, 224, 0.639, 0.560}, {2, 192, 0.551, 0.473}};

// A tile's time.  Rows of B along memory come in twice as many copies, rows of
// A and B (weight gradients) more still, which narrow tiles feel.  A tile of
// two blocks ends with an epilogue that nothing hides.
double tile_time(const Job &j, const Width &w, bool gated, bool one_wave) {
    double block = one_wave ? w.single : w.many;
    if (w.nb == 1 && j.a[0].mn)
        block = one_wave ? 0.36 : 0.40;
    else if (w.nb == 1 && j.b[0].mn)
        block *= 1.03;
    const double kb = static_cast<double>((j.K + BK - 1) / BK * j.parts);
    return kb * block + (w.nb == 1 ? 0.2 : gated ? 6.0 : 3.5);
}

// How the tiles of all jobs are dealt out (see PairArgs), and how long that
// takes.  `order` sorts the jobs by the length of their tiles.
struct Deal {
    int order[kMaxJobs];
    int64_t first[kMaxJobs + 1];
    int64_t rounds = 0;
    double time = 0.0;
};
Deal deal(const Product &p, const Width &w, int pairs) {
    Deal d;
    // Longest contractions first.
    for (int i = 0; i < p.jobs; ++i) d.order[i] = i;
    auto depth = [&](int i) { return p.job[d.order[i]].K * p.job[d.order[i]].parts; };
    for (int i = 1; i < p.jobs; ++i)
        for (int k = i; k > 0 && depth(k) > depth(k - 1); --k) std::swap(d.order[k], d.order[k - 1]);
    const int64_t tile_n = static_cast<int64_t>(w.bn) * w.nb / p.tiles_of_b();
    d.first[0] = 0;
    for (int i = 0; i < kMaxJobs; ++i) {
        int64_t n = 0;
        if (i < p.jobs) {
            const Job &j = p.job[d.order[i]];
            n = (j.M + PM - 1) / PM * ((j.N + tile_n - 1) / tile_n);
        }
        d.first[i + 1] = d.first[i] + n;
    }
    const int64_t C = d.first[kMaxJobs] < pairs ? d.first[kMaxJobs] : pairs;
    const int64_t n0 = d.first[1], n1 = d.first[kMaxJobs] - n0, more = n0 % C;
    const bool one_wave = d.first[kMaxJobs] <= pairs;
    const double a = tile_time(p.job[d.order[0]], w, p.gated, one_wave);
    const double b = p.jobs > 1 ? tile_time(p.job[d.order[1]], w, p.gated, one_wave) : 0.0;
    const double own = static_cast<double>(n0 / C) * a;
    if (n1 == 0 || more == 0) {
        d.time = own + (more ? a : 0.0) + static_cast<double>((n1 + C - 1) / C) * b;
        return d;
    }
    // Level: the pairs without one more long tile do its time in short ones.
    const int64_t level = static_cast<int64_t>((static_cast<double>(n1) - a * static_cast<double>(C - more) / b) / C);
    d.time = 1e30;
    for (int64_t s = level > 1 ? level - 1 : 0; s <= level + 2 && s <= (n1 + C - 1) / C; ++s) {
        const int64_t left = n1 - s * C;  // below zero: the last round is short of that many
        const double hi = own + a + static_cast<double>(left < -more + 1 ? s - 1 : s) * b;
        const double lo = own + static_cast<double>(s + (left > 0 ? (left + C - more - 1) / (C - more) : 0)) * b;
        const double t = hi > lo ? hi : lo;
        if (t < d.time) {
            d.time = t;
            d.rounds = s;
        }
    }
    if (d.time == 1e30) d.time = own + a;  // the short tiles end before one more long one
    return d;
}

Deal best_deal(const Product &p, int pairs, Width *width) {
    Deal best;
    best.time = 1e300;
    for (const Width &w : kWidths) {
        if (p.gated && w.bn % 64) continue;  // its columns of D are half as many
        if (p.width && p.width != w.bn * w.nb) continue;
        const Deal d = deal(p, w, pairs);
        if (d.time < best.time) {
            best = d;
            *width = w;
        }
    }
    return best;
}

template <bool GATED, int NB>
cudaError_t launch_pair(const Maps &maps, const PairArgs &args, int pairs, bool bf16, bool pdl,
                        cudaStream_t stream) {
    const int tiles = args.first[kMaxJobs];
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
    cfg.dynamicSmemBytes = PairCfg<NB>::SMEM;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    return bf16 ? cudaLaunchKernelEx(&cfg, product_pair_kernel<GATED, NB, true>, maps, args)
                : cudaLaunchKernelEx(&cfg, product_pair_kernel<GATED, NB, false>, maps, args);
}

}  // namespace

int product_pair_time(const Product &p, int sm_count, double *us) {
    int pairs = 0;
    const int rc = resident_pairs(sm_count, &pairs);
    if (rc != CUDAIR_OK) return rc;
    Width w;
    *us = (p.gated ? 7.5 : 6.0) + best_deal(p, pairs, &w).time;  // launch, set-up and the last epilogue
    return CUDAIR_OK;
}

int product_pair_launch(const Product &p, int sm_count, unsigned int *status, cudaStream_t stream) {
    int pairs = 0;
    int rc = resident_pairs(sm_count, &pairs);
    if (rc != CUDAIR_OK) return rc;
    Width w;
    const Deal d = best_deal(p, pairs, &w);
    if (d.first[kMaxJobs] > INT32_MAX / 2)
        return set_error(CUDAIR_ERR_INVALID, "cudair: linear: %lld tiles are too many", (long long)d.first[kMaxJobs]);
    alignas(64) Maps maps = {};
    PairArgs args = {};
    const int tile_n = w.bn * w.nb / p.tiles_of_b();
    args.bn = w.bn;
    for (int i = 0; i <= kMaxJobs; ++i) args.first[i] = static_cast<int>(d.first[i]);
    args.rounds = static_cast<int>(d.rounds);
    const int C = args.first[kMaxJobs] < pairs ? args.first[kMaxJobs] : pairs;
    args.own = args.first[1] / C;
    args.more = args.first[1] % C;
    for (int i = 0; i < p.jobs; ++i) {
        const Job &j = p.job[d.order[i]];
        JobArgs &o = args.job[i];
        o.M = static_cast<int>(j.M);
        o.N = static_cast<int>(j.N);
        o.num_m = static_cast<int>((j.M + PM - 1) / PM);
        o.num_n = static_cast<int>((j.N + tile_n - 1) / tile_n);
        o.num_kb = static_cast<int>((j.K + BK - 1) / BK);
        o.all_kb = o.num_kb * j.parts;
        o.per_group = GROUP_M * o.num_n;
        o.group = divide_by(o.per_group);
        o.last = divide_by((o.num_m - 1) % GROUP_M + 1);
        o.a_mn = j.a[0].mn;
        o.b_mn = j.b[0].mn;
        o.idesc = idesc_f16_f32(PM, static_cast<uint32_t>(w.bn), j.a[0].mn, j.b[0].mn, p.bf16);
        // Rows of B along memory come in whole 64-column boxes.
        const int cols = j.b[0].mn ? (w.bn / 2 + 63) / 64 * 64 : w.bn / 2;
        o.bytes = 2 * (A_STAGE + static_cast<uint32_t>(w.nb * cols) * BK * 2);
        o.d = mat_of(j.d);
        if (j.K == 0) continue;
        for (int k = 0; k < j.parts; ++k)
            if ((rc = operand_map(&maps.a[i][k], j.a[k], j.M, j.K, 128, p.bf16)) != CUDAIR_OK) return rc;
        for (int k = 0; k < (p.gated ? 2 : j.parts); ++k)
            if ((rc = operand_map(&maps.b[i][k], j.b[k], j.N, j.K, static_cast<uint32_t>(w.bn / 2), p.bf16)) != CUDAIR_OK)
                return rc;
    }
    args.act = p.act;
    for (int i = 0; i < 2; ++i) args.z[i] = mat_of(p.z[i]);
    args.residual = mat_of(p.residual);
    args.bias = p.bias;
    args.bias16 = p.bias16;
    args.status = status;
    const bool pdl = p.pdl();
    const bool wide = w.nb == 2;
    const cudaError_t e = p.gated ? (wide ? launch_pair<true, 2>(maps, args, pairs, p.bf16, pdl, stream)
                                          : launch_pair<true, 1>(maps, args, pairs, p.bf16, pdl, stream))
                                  : (wide ? launch_pair<false, 2>(maps, args, pairs, p.bf16, pdl, stream)
                                          : launch_pair<false, 1>(maps, args, pairs, p.bf16, pdl, stream));
    return e == cudaSuccess ? CUDAIR_OK : cuda_error(e, "product_pair_kernel launch");
}

}  // namespace ffn
}  // namespace cudair
