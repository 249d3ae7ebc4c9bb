// linear_split_sm100.cu - the products of the feed-forward operators where a
// grid of 256-row tiles would leave most SMs idle: few rows (decode steps and
// short batches) and small outputs with a long contraction (weight gradients
// of small layers).
//
// Mathematics: D^T = B^T . A^T.  The operands are swapped, so the 128-row side
// of tcgen05.mma runs over N, which is long, and its column side over M,
// rounded up to 16 only: one token costs 16 columns.  The contraction is cut
// into `split` runs of k-blocks, one per CTA of a cluster:
//   D[m, n] = epilogue(sum over ranks r of P_r[m, n]),
// P_r the rank's fp32 partial product.  Each rank leaves P_r in its own shared
// memory; after a cluster barrier the ranks share out the rows, and each reads
// its rows' parts from all ranks over distributed shared memory, adds them in
// a fixed order (its own first, then round the ranks), and runs the epilogue.
// So there is no workspace, no counter and no atomic: the result does not
// depend on timing, and calls may overlap on any streams and in any graphs.
//   gated: two accumulators per CTA (Wg's and Wu's 128 columns), so G and U
//     of an element meet in the thread that adds its parts.
//
// What bounds it: the one pass over the weights through HBM (M <= 64), so what
// counts is bytes in flight on every SM: a TMA ring of about 100 KB per CTA, and
// two CTAs per SM where there are enough.  Measured (weights from HBM): gated 1
// x 14336 x 4096 40.0 us, 5.9 TB/s, and 64 rows 41 us; 16 x 14336 x 4096 23.1
// us, 5.1 TB/s; 1 x 4096 x 4096 10.5 us, of which the stream is 4.6 us, set-up and
// launch 4 us, the join 1.6 us; 2 x 256 x 128 3.7 us.
//
// Tensor memory and clusters: tcgen05.alloc blocks until columns are free, and a
// rank that holds columns waits for its cluster's other ranks.  Two clusters
// that each held columns on one SM and waited for them on another would wait
// for good, so the CTAs of this kernel on an SM never ask for more columns than
// it has: a CTA's shared memory is at least its share of the SM's, in the
// proportion of its columns to 512 (smem_floor), whatever launches run side by side.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "cudair_internal.h"
#include "linear_epilogue.cuh"
#include "linear_internal.h"
#include "sm100.cuh"

namespace cudair {
namespace ffn {
namespace split {

constexpr int BK = 64;
constexpr int NT = 128;  // columns of D per tile (the MMA's 128 rows)
constexpr int MAX_SPLIT = 8;  // the portable cluster size
constexpr int MAX_STAGES = 12;
__host__ __device__ constexpr int threads(int epi_warps) { return 64 + 32 * epi_warps; }
constexpr uint32_t W_BOX = 64 * BK * 2;
constexpr uint32_t W_TILE = NT * BK * 2;  // 16 KB
constexpr uint32_t BAR_BYTES = 256;
constexpr size_t SM_SMEM = 228 * 1024;  // per SM, 1 KB of it reserved per CTA
static_assert(2 * MAX_STAGES * 8 + 2 * 8 + 8 <= BAR_BYTES, "barrier area");

struct Maps {
    CUtensorMap w[kMaxJobs][2], x[kMaxJobs][2];
};

struct JobArgs {
    int M, N;
    int num_kb, parts;   // k-blocks of one contraction; contractions per accumulator
    int mt;              // rows of D per tile, a multiple of 16 (of 64 where A's rows run along memory)
    int m_tiles, first;  // row tiles; the job's first tile
    int run, longer;     // k-blocks of a rank; the first `longer` ranks take one more
    int w_mn, x_mn;
    uint32_t idesc;
    int w_early;  // B is a weight that nothing still running writes
    Mat d;
};

struct Args {
    JobArgs job[kMaxJobs];
    int jobs, split, stages;
    uint32_t x_stage, tmem_cols;  // the largest of the jobs
    int bf16, act;
    Mat z[2], residual;
    const void *bias;
    int bias16;
    unsigned int *status;
};

__device__ __forceinline__ uint32_t cluster_id() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
    return r;
}
// All threads of the cluster; orders no memory accesses.
__device__ __forceinline__ void cluster_sync_relaxed() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// Four columns of a row from col on, below N.
__device__ __forceinline__ void store4(const Mat &m, long long row, int col, int N, bool bf16,
                                       const float (&v)[4]) {
    if (m.f32) {
        float *p = static_cast<float *>(m.p) + row * m.ld + col;
        if (col + 4 <= N) {
            *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < N) p[j] = v[j];
        }
    } else {
        uint16_t *p = static_cast<uint16_t *>(m.p) + row * m.ld + col;
        if (col + 4 <= N) {
            *reinterpret_cast<uint2 *>(p) = make_uint2(pack16(v[0], v[1], bf16), pack16(v[2], v[3], bf16));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < N) p[j] = to16(v[j], bf16);
        }
    }
}
// The same four columns as they lie in memory (two words of 16-bit values, or
// four), and added to v.
__device__ __forceinline__ uint4 fetch4(const Mat &m, long long row, int col, int N) {
    uint4 r = make_uint4(0, 0, 0, 0);
    if (m.f32) {
        const float *p = static_cast<const float *>(m.p) + row * m.ld + col;
        if (col + 4 <= N) {
            r = *reinterpret_cast<const uint4 *>(p);
        } else {
            r.x = __float_as_uint(p[0]);
            if (col + 1 < N) r.y = __float_as_uint(p[1]);
            if (col + 2 < N) r.z = __float_as_uint(p[2]);
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(m.p) + row * m.ld + col;
        if (col + 4 <= N) {
            const uint2 w = *reinterpret_cast<const uint2 *>(p);
            r.x = w.x;
            r.y = w.y;
        } else {
            r.x = p[0];
            if (col + 1 < N) r.x |= static_cast<uint32_t>(p[1]) << 16;
            if (col + 2 < N) r.y = p[2];
        }
    }
    return r;
}
__device__ __forceinline__ void add4(uint4 r, bool f32, bool bf16, float (&v)[4]) {
    if (f32) {
        v[0] += __uint_as_float(r.x);
        v[1] += __uint_as_float(r.y);
        v[2] += __uint_as_float(r.z);
        v[3] += __uint_as_float(r.w);
    } else {
        float lo, hi;
        unpack16(r.x, bf16, lo, hi);
        v[0] += lo;
        v[1] += hi;
        unpack16(r.y, bf16, lo, hi);
        v[2] += lo;
        v[3] += hi;
    }
}

// A kernel of the same block that uses no tensor memory, to ask the driver
// how many clusters fit (it counts one CTA per SM for any kernel that
// allocates tensor memory; two of these do share an SM).
__global__ void __launch_bounds__(threads(8), 2) occupancy_kernel() {}

// The sums and the epilogue.  Rank r of SPLIT takes rows r, r + SPLIT, ... of the
// tile; a warp takes whole rows, four columns a lane (`mine`: where the
// lane's columns of this CTA's parts start).  An element's parts are added from
// its own rank's on, round the ranks: a fixed order.  What bounds it is the
// network between SMs, about 15 bytes a clock for each (64 rows of two ranks took
// 5800 clocks when the own rank's part went through it too).
template <bool GATED, int SPLIT, int EPI_WARPS>
__device__ __forceinline__ void join(const Args &p, const JobArgs &job, uint32_t mine, int rank, int m0, int n0,
                                     int rows) {
    constexpr int W_TILES = GATED ? 2 : 1;
    constexpr int WARPS = threads(EPI_WARPS) / 32;
    constexpr int LOADS = SPLIT * W_TILES;  // per row
    // Rows that are worked on together, as registers allow.
    constexpr int BATCH = EPI_WARPS > 4 ? (LOADS >= 8 ? 1 : 2) : LOADS >= 16 ? 1 : LOADS >= 4 ? 2 : 4;
    const uint32_t warp = warp_id();
    const int mt = job.mt, col = n0 + static_cast<int>(lane_id()) * 4;
    if (col >= job.N) return;
    const bool bf16 = p.bf16 != 0;
    float bias[4] = {};
    if (p.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < job.N)
                bias[j] = p.bias16 ? from16(static_cast<const uint16_t *>(p.bias)[col + j], bf16)
                                   : static_cast<const float *>(p.bias)[col + j];
    }
    uint32_t from[SPLIT];
#pragma unroll
    for (int r = 1; r < SPLIT; ++r) from[r] = mapa_shared(mine, static_cast<uint32_t>((rank + r) % SPLIT));
    const int own = (rows - rank + SPLIT - 1) / SPLIT;  // rows of this rank
    for (int k0 = static_cast<int>(warp) * BATCH; k0 < own; k0 += WARPS * BATCH) {
        // Row b of the batch is there.  (Without it, nothing is loaded: no read
        // of another CTA's memory may be left that nothing waits for.)
        auto there = [&](int b) { return k0 + b < own; };
        auto row = [&](int b) { return rank + (k0 + b) * SPLIT; };
        float v[W_TILES][BATCH][4] = {};
        uint4 res[BATCH] = {};
        {
            float4 t[W_TILES][BATCH][SPLIT];
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                if (!there(b)) break;
#pragma unroll
                for (int i = 0; i < W_TILES; ++i) {
                    const uint32_t at = static_cast<uint32_t>(i * mt + row(b)) * (NT * 4);
#pragma unroll
                    for (int r = 1; r < SPLIT; ++r) t[i][b][r] = ld_cluster_f4(from[r] + at);
                    t[i][b][0] = ld_shared_f4(mine + at);
                }
                if (p.residual.p) res[b] = fetch4(p.residual, m0 + row(b), col, job.N);
            }
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                if (!there(b)) break;
#pragma unroll
                for (int i = 0; i < W_TILES; ++i)
#pragma unroll
                    for (int r = 0; r < SPLIT; ++r) {
                        v[i][b][0] += t[i][b][r].x;
                        v[i][b][1] += t[i][b][r].y;
                        v[i][b][2] += t[i][b][r].z;
                        v[i][b][3] += t[i][b][r].w;
                    }
            }
        }
        if (!GATED) {
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[0][b][j] += bias[j];
        }
        if (p.z[0].p) {
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
                if (there(b)) {
#pragma unroll
                    for (int i = 0; i < W_TILES; ++i) store4(p.z[i], m0 + row(b), col, job.N, bf16, v[i][b]);
                }
        }
        if (GATED || p.act != CUDAIR_ACT_NONE)
            with_act(p.act, [&](auto tag) {
#pragma unroll
                for (int b = 0; b < BATCH; ++b)
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        act_pair<decltype(tag)::value>(v[0][b][j], v[0][b][j + 1]);
                        if (GATED) {
                            v[0][b][j] *= v[W_TILES - 1][b][j];
                            v[0][b][j + 1] *= v[W_TILES - 1][b][j + 1];
                        }
                    }
            });
        if (p.residual.p) {
#pragma unroll
            for (int b = 0; b < BATCH; ++b) add4(res[b], p.residual.f32, bf16, v[0][b]);
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
            if (there(b)) store4(job.d, m0 + row(b), col, job.N, bf16, v[0][b]);
    }
}

template <bool GATED, int EPI_WARPS>
__global__ void __launch_bounds__(threads(EPI_WARPS), 2)
    product_split_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args p) {
    constexpr int W_TILES = GATED ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    uint8_t *smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);  // the same offset in every rank

    const uint32_t x_stage = p.x_stage;
    const int STAGES = p.stages;
    uint8_t *sW = smem;
    uint8_t *sX = smem + STAGES * W_TILES * W_TILE;
    uint64_t *bars = reinterpret_cast<uint64_t *>(sX + STAGES * x_stage);
    uint64_t *full = bars;
    uint64_t *empty = bars + STAGES;
    uint64_t *acc_full = bars + 2 * STAGES;
    uint64_t *drain = acc_full + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    float *part = reinterpret_cast<float *>(smem);  // the ring's memory, once the MMAs are done: [acc][m][n]

    const uint32_t warp = warp_id(), lane = lane_id();
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    const int rank = static_cast<int>(cluster_ctarank());
    int tile = static_cast<int>(cluster_id()), ji = 0;
    if (p.jobs > 1 && tile >= p.job[1].first) ji = p.jobs > 2 && tile >= p.job[2].first ? 2 : 1;
    const JobArgs job = ji == 0 ? p.job[0] : ji == 1 ? p.job[1] : p.job[2];  // fixed places: in registers
    tile -= job.first;
    const int mt = job.mt;
    int m0 = 0, n0 = tile * NT;
    if (job.m_tiles > 1) {
        const unsigned n = static_cast<unsigned>(tile) / static_cast<unsigned>(job.m_tiles);
        m0 = (tile - static_cast<int>(n) * job.m_tiles) * mt;
        n0 = static_cast<int>(n) * NT;
    }
    const int rows = min(mt, job.M - m0);
    const int kb0 = rank * job.run + min(rank, job.longer);
    const int kb1 = kb0 + job.run + (rank < job.longer ? 1 : 0);
    const int head = min(kb1 - kb0, STAGES);
    const int part_kb = job.num_kb, w_mn = job.w_mn, x_mn = job.x_mn;
    const CUtensorMap *map_w = &maps.w[ji][0], *map_x = &maps.x[ji][0];
    const uint64_t policy = l2_policy_evict_normal();
    auto load_w = [&](int kb, int st) {
        const int part = kb >= part_kb ? 1 : 0;
        const int k0 = (kb - part * part_kb) * BK;
        mbar_arrive_expect_tx(&full[st], W_TILES * W_TILE + static_cast<uint32_t>(mt) * BK * 2);
#pragma unroll
        for (int i = 0; i < W_TILES; ++i) {
            const CUtensorMap *mw = map_w + (GATED ? i : part);
            uint8_t *dst = sW + (st * W_TILES + i) * W_TILE;
            if (w_mn) {
                tma_load_2d(dst, mw, &full[st], n0, k0, policy);
                tma_load_2d(dst + W_BOX, mw, &full[st], n0 + 64, k0, policy);
            } else {
                tma_load_2d(dst, mw, &full[st], k0, n0, policy);
            }
        }
    };
    auto load_x = [&](int kb, int st) {
        const int part = kb >= part_kb ? 1 : 0;
        const int k0 = (kb - part * part_kb) * BK;
        uint8_t *dst = sX + st * x_stage;
        if (x_mn) {
            for (int j = 0; j < mt; j += 64)
                tma_load_2d(dst + j * (BK * 2), map_x + part, &full[st], m0 + j, k0, policy);
        } else {
            tma_load_2d(dst, map_x + part, &full[st], k0, m0, policy);
        }
    };

    // The producer thread, which set up the barriers, requests the first
    // ring-full at once: the rest of the set-up runs under the copies.  Its
    // weights may be requested before the preceding kernel ends (launch mode 2).
    if (threadIdx.x == 0) {
        if (!job.w_early) grid_dependency_wait();
        for (int i = 0; i < head; ++i) {
            load_w(kb0 + i, i);
            if (!job.w_early) load_x(kb0 + i, i);
        }
        if (job.w_early) {
            grid_dependency_wait();
            for (int i = 0; i < head; ++i) load_x(kb0 + i, i);
        }
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, p.tmem_cols);
        tmem_relinquish();
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    // cudair_set_gemm_pdl: only now, with its columns in hand, so that no CTA of
    // the next kernel takes them and waits for this one; and past the producer's wait
    // for the preceding kernel (the barrier above), so that all before have ended.
    if (threadIdx.x == 64) grid_launch_dependents();

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            int st = 0;
            uint32_t phase = 0, issued = head;
            bool ok = true;
            for (int kb = kb0 + head; kb < kb1; ++kb) {
                if (!mbar_wait(&empty[st], phase, abort_flag, p.status, kSiteProducerEmpty)) {
                    ok = false;
                    break;
                }
                load_w(kb, st);
                load_x(kb, st);
                ++issued;
                if (++st == STAGES) {
                    st = 0;
                    phase ^= 1u;
                }
            }
            if (!ok) {
                // Let the copies still in flight land before the CTA exits.
                int never = 0;
                const uint32_t outstanding = min(issued, static_cast<uint32_t>(STAGES));
                for (uint32_t i = 1; i <= outstanding; ++i) {
                    const uint32_t idx = issued - i;
                    mbar_wait(&full[idx % STAGES], (idx / STAGES) & 1u, &never, p.status, kSiteDrain);
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (lane == 0 && kb1 > kb0) {
            grid_dependency_wait();
            const uint32_t w_step = w_mn ? 2048u : 32u, w_lbo = w_mn ? W_BOX : 16u;
            const uint32_t x_step = x_mn ? 2048u : 32u, x_lbo = x_mn ? W_BOX : 16u;
            const uint32_t idesc = job.idesc;
            int st = 0;
            uint32_t phase = 0;
            bool ok = true, issued_any = false;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(&full[st], phase, abort_flag, p.status, kSiteMmaFull)) {
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                const uint32_t w_base = smem_u32(sW + st * W_TILES * W_TILE);
                const uint32_t x_base = smem_u32(sX + st * x_stage);
#pragma unroll
                for (int kk = 0; kk < BK / 16; ++kk) {
                    const uint64_t x_desc = smem_desc_sw128(x_base + kk * x_step, x_lbo, 1024);
#pragma unroll
                    for (int i = 0; i < W_TILES; ++i)
                        umma_f16_ss(tmem_base + i * mt,
                                    smem_desc_sw128(w_base + i * W_TILE + kk * w_step, w_lbo, 1024), x_desc,
                                    idesc, (kb - kb0) | kk ? 1u : 0u);
                }
                issued_any = true;
                umma_commit(&empty[st]);
                if (++st == STAGES) {
                    st = 0;
                    phase ^= 1u;
                }
            }
            if (ok) {
                umma_commit(acc_full);
            } else if (issued_any) {
                int never = 0;
                umma_commit(drain);
                mbar_wait(drain, 0, &never, p.status, kSiteDrain);
            }
        }
        __syncwarp();
    } else {
        // ---------------- parts: TMEM -> shared memory ----------------
        // Two warps to a lane quarter, every other 16 columns each.
        const uint32_t q = warp & 3u;
        const int half = static_cast<int>(warp - 2u) >> 2;
        float *mine = part + q * 32 + lane;
        if (kb1 > kb0) {
            // The warp stops as one: TMEM loads are warp-wide.
            if (__all_sync(0xFFFFFFFFu, mbar_wait(acc_full, 0, abort_flag, p.status, kSiteEpilogueAccFull))) {
                tc_fence_after_sync();
#pragma unroll 1
                for (int i = 0; i < W_TILES; ++i)
#pragma unroll 1
                    for (int c = half * 16; c < rows; c += EPI_WARPS * 4) {
                        uint32_t r[16];
                        tmem_ld_32x32b_x16(tmem_base + ((q * 32u) << 16) + i * mt + c, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) mine[(i * mt + c + j) * NT] = __uint_as_float(r[j]);
                    }
            }
        } else {  // an empty run: K = 0, or fewer k-blocks than ranks
            for (int i = 0; i < W_TILES; ++i)
                for (int c = half; c < rows; c += EPI_WARPS / 4) mine[(i * mt + c) * NT] = 0.0f;
        }
        __syncwarp();
        tc_fence_before_sync();
    }
    __syncwarp();
    if (p.split > 1)
        cluster_sync();
    else
        __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, p.tmem_cols);
    }

    grid_dependency_wait();
    const uint32_t mine = smem_u32(part) + lane * 16u;
    switch (p.split) {
        case 1: join<GATED, 1, EPI_WARPS>(p, job, mine, rank, m0, n0, rows); break;
        case 2: join<GATED, 2, EPI_WARPS>(p, job, mine, rank, m0, n0, rows); break;
        case 4: join<GATED, 4, EPI_WARPS>(p, job, mine, rank, m0, n0, rows); break;
        default: join<GATED, 8, EPI_WARPS>(p, job, mine, rank, m0, n0, rows); break;
    }
    // No rank leaves while its parts are being read.  Relaxed: the reads are
    // done, and the stores need no waiting for (a releasing barrier waits for
    // them: 1.2 us).
    __syncwarp();
    if (p.split > 1) cluster_sync_relaxed();
}

// ---- host side -----------------------------------------------------------------------

namespace {

constexpr size_t ring_bytes(int w_tiles, int mt, int stages) {
    return static_cast<size_t>(stages) * (w_tiles * W_TILE + static_cast<size_t>(mt) * BK * 2);
}
constexpr size_t fixed_bytes() { return 1024 + BAR_BYTES; }
uint32_t tmem_cols_for(int w_tiles, int mt) {
    uint32_t c = 32;
    while (c < static_cast<uint32_t>(w_tiles * mt)) c *= 2;
    return c;
}
// The least shared memory of a CTA with that many TMEM columns (see the top).
size_t smem_floor(uint32_t cols) { return cols * SM_SMEM / 512 - 1024; }

std::mutex g_mu;

// Per device: the clusters of each size that fit at once, with one or two CTAs
// per SM (index 0, 1).  A GPC's SMs do not divide evenly into clusters: eight
// CTAs a cluster and one per SM leave more than ten SMs idle.
struct Device {
    bool ready = false;
    int clusters[2][MAX_SPLIT + 1] = {};
};
Device g_dev[64];

// Dynamic shared memory of a CTA when one or two are to share an SM.
constexpr size_t kBudget[2] = {227 * 1024, 113 * 1024};

int prepare_device(const Device **out) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_error(e, "cudaGetDevice");
    std::lock_guard<std::mutex> lk(g_mu);  // dev is in 0..63: the device check passed
    Device &d = g_dev[dev];
    if (!d.ready) {
        for (const void *fn : {reinterpret_cast<const void *>(product_split_kernel<false, 4>),
                               reinterpret_cast<const void *>(product_split_kernel<false, 8>),
                               reinterpret_cast<const void *>(product_split_kernel<true, 4>),
                               reinterpret_cast<const void *>(product_split_kernel<true, 8>),
                               reinterpret_cast<const void *>(occupancy_kernel)}) {
            e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
            if (e != cudaSuccess) return cuda_error(e, "cudaFuncSetAttribute(product_split_kernel)");
        }
        for (int two = 0; two < 2; ++two)
            for (int size = 1; size <= MAX_SPLIT; ++size) {
                cudaLaunchConfig_t cfg = {};
                cudaLaunchAttribute attr[1];
                attr[0].id = cudaLaunchAttributeClusterDimension;
                attr[0].val.clusterDim.x = static_cast<unsigned>(size);
                attr[0].val.clusterDim.y = 1;
                attr[0].val.clusterDim.z = 1;
                cfg.gridDim = dim3(static_cast<unsigned>(512 * size), 1, 1);
                cfg.blockDim = dim3(threads(8), 1, 1);
                cfg.dynamicSmemBytes = kBudget[two];
                cfg.attrs = attr;
                cfg.numAttrs = 1;
                e = cudaOccupancyMaxActiveClusters(&d.clusters[two][size], occupancy_kernel, &cfg);
                if (e != cudaSuccess) return cuda_error(e, "cudaOccupancyMaxActiveClusters");
            }
        d.ready = true;
    }
    *out = &d;
    return CUDAIR_OK;
}

// One way to cut a call.
struct Cut {
    int64_t tiles = 0, kb = 0;  // kb: k-blocks of the longest contraction
    int w_tiles = 1, mt = 0, rows = 0, split = 1;
    int two = 0;  // 1: the ring of two CTAs per SM
    double weight_bytes = 0.0;
};

// How long the kernel takes for one way to cut a call, in microseconds.  Fitted
// to 1800 timings of 82 shapes on B200 (1 to 1024 rows, 128 to 128256 columns,
// 64 to 14336 deep; tiles of 16 to 128 rows, split 1 to 8; 9 % rms).  What it
// says of the kernel:
//   * launch, set-up and the end are 3.8 us, 0.5 us more for each CTA per SM, and
//     0.65 us where some SMs get a second one; a further wave costs 2 us;
//   * a CTA's k-blocks follow one another in 0.32 us at best, at 89 GB/s into an
//     SM, and together no faster than HBM gives the weights: 5.9 TB/s to 112
//     CTAs, 6.4 to 224 (16 x 14336 x 4096: 24.1 and 23.1 us);
//   * a row of parts costs 13.6 ns on its way through shared memory, and 1.6 ns
//     more through the network between SMs.
double split_time(const Cut &c, const int (&clusters)[2][MAX_SPLIT + 1]) {
    const double sms = clusters[0][1];
    const double ctas = static_cast<double>(c.tiles) * c.split;
    const double places = static_cast<double>(clusters[c.two][c.split]) * c.split;
    const double waves = std::ceil(ctas / places), per_sm = std::max(1.0, std::min(ctas, places) / sms);
    const double run = std::ceil(static_cast<double>(c.kb) / c.split);
    const double stage = static_cast<double>(c.w_tiles) * W_TILE + c.mt * BK * 2;
    const double block = std::max(std::max(0.32, stage * per_sm / 89e3), 0.124 * c.w_tiles * c.mt / 128 * per_sm);
    const double hbm = 5.4e6 + 0.66e6 * std::min(ctas, places) / sms;  // bytes a microsecond
    const double stream = std::max(waves * run * block, c.weight_bytes / hbm);
    const double rows = static_cast<double>(c.rows) * c.w_tiles;
    const double joins = (0.0016 * (c.split - 1) / c.split + 0.0136) * rows * std::max(1.0, 0.36 * per_sm) * waves;
    return 3.8 + 0.49 * ctas / sms + (ctas > static_cast<double>(clusters[0][c.split]) * c.split ? 0.65 : 0.0) +
           2.0 * (waves - 1.0) + stream + joins;
}

}  // namespace
}  // namespace split

// The best way to cut a call: tiles of 16 to 128 rows, split 1, 2, 4 or 8, a
// ring for one or two CTAs per SM.  Several jobs share one grid and the split.
// Of two cuts that take the same, the ring of two CTAs per SM (a shorter first
// ring-full starts sooner: 1 x 256 x 8192 9.6 against 10.4 us), but a whole SM's
// where half of one holds three stages or fewer (128 x 4096 x 4096: 13.1 against 14.3 us).
int split_plan(const Product &p, SplitPlan *plan) {
    using namespace split;
    const Device *dev = nullptr;
    const int rc = prepare_device(&dev);
    if (rc != CUDAIR_OK) return rc;
    plan->time = 1e30;
    static constexpr int kRows[] = {16, 32, 48, 64, 96, 128};
    for (const int want : kRows) {
        Cut c;
        c.w_tiles = p.tiles_of_b();
        int mt[kMaxJobs] = {};
        bool whole = true, fits = true;  // whole: no job has more rows than this
        for (int i = 0; i < p.jobs; ++i) {
            const Job &j = p.job[i];
            // 64 rows at a time where A's rows run along memory.
            const int unit = j.a[0].mn ? 64 : 16;
            if (want % unit) fits = false;
            mt[i] = static_cast<int>(std::min<int64_t>(want, (j.M + unit - 1) / unit * unit));
            whole = whole && j.M <= want;
            c.tiles += (j.M + mt[i] - 1) / mt[i] * ((j.N + NT - 1) / NT);
            c.kb = std::max<int64_t>(c.kb, (j.K + BK - 1) / BK * j.parts);
            c.mt = std::max(c.mt, mt[i]);
            c.rows = std::max(c.rows, static_cast<int>(std::min<int64_t>(mt[i], j.M)));
            c.weight_bytes += static_cast<double>(j.N) * static_cast<double>(j.K) * j.parts * c.w_tiles * 2.0;
        }
        if (!fits) continue;
        const bool deep = c.w_tiles * static_cast<int>(W_TILE) + c.mt * BK * 2 > 28 * 1024;
        for (int k = 0; k < 2; ++k) {
            c.two = deep ? k : 1 - k;
            const int stages = std::min(
                MAX_STAGES, static_cast<int>((kBudget[c.two] - fixed_bytes()) / ring_bytes(c.w_tiles, c.mt, 1)));
            // The parts take the ring's place.
            if (ring_bytes(c.w_tiles, c.mt, stages) < static_cast<size_t>(c.w_tiles) * c.mt * NT * 4) continue;
            for (c.split = 1; c.split <= MAX_SPLIT; c.split *= 2) {
                if (c.split > std::max<int64_t>(c.kb, 1) || c.tiles * c.split > INT32_MAX) break;
                const double t = split_time(c, dev->clusters);
                if (t < plan->time) {
                    plan->time = t;
                    plan->split = c.split;
                    plan->stages = stages;
                    for (int i = 0; i < p.jobs; ++i) plan->mt[i] = mt[i];
                }
            }
        }
        if (whole) break;
    }
    return plan->time < 1e30 ? CUDAIR_OK : set_error(CUDAIR_ERR_INVALID, "cudair: linear: too many tiles");
}

int product_split_launch(const Product &p, const SplitPlan &plan, unsigned int *status, cudaStream_t stream) {
    using namespace split;
    const int w_tiles = p.tiles_of_b();
    alignas(64) split::Maps maps = {};
    split::Args args = {};
    int rc = CUDAIR_OK, tiles = 0, most_mt = 0;
    for (int i = 0; i < p.jobs; ++i) {
        const Job &j = p.job[i];
        split::JobArgs &o = args.job[i];
        o.M = static_cast<int>(j.M);
        o.N = static_cast<int>(j.N);
        o.num_kb = static_cast<int>((j.K + split::BK - 1) / split::BK);
        o.parts = j.parts;
        o.mt = plan.mt[i];
        o.m_tiles = static_cast<int>((j.M + o.mt - 1) / o.mt);
        o.first = tiles;
        o.run = o.num_kb * o.parts / plan.split;
        o.longer = o.num_kb * o.parts % plan.split;
        tiles += o.m_tiles * static_cast<int>((j.N + NT - 1) / NT);
        most_mt = std::max(most_mt, o.mt);
        o.w_mn = j.b[0].mn;
        o.x_mn = j.a[0].mn;
        o.idesc = idesc_f16_f32(NT, static_cast<uint32_t>(o.mt), j.b[0].mn, j.a[0].mn, p.bf16);
        o.w_early = j.b_weights && p.weights_early();
        o.d = mat_of(j.d);
        if (j.K == 0) continue;
        for (int k = 0; k < (p.gated ? 2 : j.parts); ++k)
            if ((rc = operand_map(&maps.w[i][k], j.b[k], j.N, j.K, NT, p.bf16)) != CUDAIR_OK) return rc;
        for (int k = 0; k < j.parts; ++k)
            if ((rc = operand_map(&maps.x[i][k], j.a[k], j.M, j.K, static_cast<uint32_t>(o.mt), p.bf16)) != CUDAIR_OK)
                return rc;
    }
    args.jobs = p.jobs;
    args.split = plan.split;
    args.stages = plan.stages;
    args.x_stage = static_cast<uint32_t>(most_mt) * split::BK * 2;
    args.tmem_cols = tmem_cols_for(w_tiles, most_mt);
    args.bf16 = p.bf16;
    args.act = p.act;
    for (int i = 0; i < 2; ++i) args.z[i] = mat_of(p.z[i]);
    args.residual = mat_of(p.residual);
    args.bias = p.bias;
    args.bias16 = p.bias16;
    args.status = status;
    // Up to 32 rows the join is short and four warps do it (eight cost 0.3 us
    // more, 1 x 4096 x 4096); above, eight (gated 64 x 14336 x 4096: 46.0 -> 45.2 us).
    const bool many = most_mt > 32;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    unsigned attrs = 0;
    if (plan.split > 1) {
        attr[attrs].id = cudaLaunchAttributeClusterDimension;
        attr[attrs].val.clusterDim.x = static_cast<unsigned>(plan.split);
        attr[attrs].val.clusterDim.y = 1;
        attr[attrs].val.clusterDim.z = 1;
        ++attrs;
    }
    if (p.pdl()) {
        attr[attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[attrs].val.programmaticStreamSerializationAllowed = 1;
        ++attrs;
    }
    cfg.gridDim = dim3(static_cast<unsigned>(tiles) * plan.split, 1, 1);
    cfg.blockDim = dim3(static_cast<unsigned>(threads(many ? 8 : 4)), 1, 1);
    cfg.dynamicSmemBytes =
        std::max(fixed_bytes() + ring_bytes(w_tiles, most_mt, plan.stages), smem_floor(args.tmem_cols));
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = attrs;
    const cudaError_t e = p.gated ? (many ? cudaLaunchKernelEx(&cfg, product_split_kernel<true, 8>, maps, args)
                                          : cudaLaunchKernelEx(&cfg, product_split_kernel<true, 4>, maps, args))
                                  : (many ? cudaLaunchKernelEx(&cfg, product_split_kernel<false, 8>, maps, args)
                                          : cudaLaunchKernelEx(&cfg, product_split_kernel<false, 4>, maps, args));
    return e == cudaSuccess ? CUDAIR_OK : cuda_error(e, "product_split_kernel launch");
}

}  // namespace ffn
}  // namespace cudair
