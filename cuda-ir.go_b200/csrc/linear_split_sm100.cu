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
// rank order, and runs the epilogue.  So there is no workspace, no counter and
// no atomic: the result does not depend on timing, and calls may overlap on
// any streams and in any graphs.
//   gated: two accumulators per CTA (Wg's and Wu's 128 columns), so G and U
//     of an element meet in the thread that adds its parts.
//
// What bounds it: the one pass over the weights through HBM (M <= 64), so what
// counts is bytes in flight on every SM: a TMA ring of about 96 KB per CTA, two
// CTAs per SM, one of which streams while the other joins its parts.
//
// Tensor memory and clusters: tcgen05.alloc blocks until columns are free, and a
// rank that holds columns waits for its cluster's other ranks.  Two clusters
// that each hold columns on one SM and wait for them on another would wait for good, so
// CTAs of this kernel never ask for more columns than an SM has: a CTA's
// shared memory is at least its share of the SM's in the proportion of its
// columns to 512 (smem_floor), whatever launches run side by side.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
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
    const int rank = static_cast<int>(blockIdx.x % p.split);
    int tile = static_cast<int>(blockIdx.x / p.split);
    int ji = 0;
    if (p.jobs > 1 && tile >= p.job[1].first) ji = p.jobs > 2 && tile >= p.job[2].first ? 2 : 1;
    const JobArgs job = ji == 0 ? p.job[0] : ji == 1 ? p.job[1] : p.job[2];  // fixed places: in registers
    tile -= job.first;
    const int mt = job.mt;
    const int m0 = tile % job.m_tiles * mt, n0 = tile / job.m_tiles * NT;
    const int rows = min(mt, job.M - m0);
    const int total_kb = job.num_kb * job.parts;
    const int kb0 = static_cast<int>(static_cast<long long>(total_kb) * rank / p.split);
    const int kb1 = static_cast<int>(static_cast<long long>(total_kb) * (rank + 1) / p.split);

    if (threadIdx.x == 64) grid_launch_dependents();  // cudair_set_gemm_pdl

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

    // The producer thread sets up its barriers and requests the first
    // ring-full at once: the rest of the set-up runs under the copies.  Its weights may be
    // requested before the preceding kernel ends (launch mode 2).
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
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
            if (mbar_wait(acc_full, 0, abort_flag, p.status, kSiteEpilogueAccFull)) {
                __syncwarp();
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

    // ---------------- the sums and the epilogue ----------------
    // Rank r takes rows r, r + split, ...; a warp takes whole rows of the tile,
    // four columns a lane.
    grid_dependency_wait();
    const int col = n0 + static_cast<int>(lane) * 4;
    if (col < job.N) {
        const bool bf16 = p.bf16 != 0;
        float bias[4] = {};
        if (p.bias) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < job.N)
                    bias[j] = p.bias16 ? from16(static_cast<const uint16_t *>(p.bias)[col + j], bf16)
                                       : static_cast<const float *>(p.bias)[col + j];
        }
        const uint32_t base = smem_u32(part) + lane * 16u;
        constexpr int BATCH = GATED ? 1 : 2;  // rows whose parts are requested together
        constexpr int WARPS = threads(EPI_WARPS) / 32;
        const int own = (rows - rank + p.split - 1) / p.split;  // rows of this rank
        for (int k0 = static_cast<int>(warp) * BATCH; k0 < own; k0 += WARPS * BATCH) {
            float4 t[BATCH * W_TILES][MAX_SPLIT];
            uint4 res[BATCH];
            if (p.residual.p) {
#pragma unroll
                for (int b = 0; b < BATCH; ++b)
                    res[b] = fetch4(p.residual, m0 + rank + min(k0 + b, own - 1) * p.split, col, job.N);
            }
#pragma unroll
            for (int r = 0; r < MAX_SPLIT; ++r)
                if (r < p.split) {
                    const uint32_t from = mapa_shared(base, r);
#pragma unroll
                    for (int b = 0; b < BATCH; ++b)
#pragma unroll
                        for (int i = 0; i < W_TILES; ++i) {
                            const int c = rank + min(k0 + b, own - 1) * p.split;
                            t[b * W_TILES + i][r] = ld_cluster_f4(from + (i * mt + c) * (NT * 4));
                        }
                }
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                if (k0 + b >= own) break;
                const int c = rank + (k0 + b) * p.split;
                float v[W_TILES][4] = {};
#pragma unroll
                for (int r = 0; r < MAX_SPLIT; ++r)
                    if (r < p.split) {
#pragma unroll
                        for (int i = 0; i < W_TILES; ++i) {
                            v[i][0] += t[b * W_TILES + i][r].x;
                            v[i][1] += t[b * W_TILES + i][r].y;
                            v[i][2] += t[b * W_TILES + i][r].z;
                            v[i][3] += t[b * W_TILES + i][r].w;
                        }
                    }
                const long long row = m0 + c;
                float out[4];
                if (GATED) {
                    if (p.z[0].p) {
                        store4(p.z[0], row, col, job.N, bf16, v[0]);
                        store4(p.z[1], row, col, job.N, bf16, v[W_TILES - 1]);
                    }
                    with_act(p.act, [&](auto tag) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            out[j] = act_value<decltype(tag)::value>(v[0][j]) * v[W_TILES - 1][j];
                    });
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[0][j] += bias[j];
                    if (p.z[0].p) store4(p.z[0], row, col, job.N, bf16, v[0]);
                    with_act(p.act, [&](auto tag) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) out[j] = act_value<decltype(tag)::value>(v[0][j]);
                    });
                    if (p.residual.p) add4(res[b], p.residual.f32, bf16, out);
                }
                store4(job.d, row, col, job.N, bf16, out);
            }
        }
    }
    __syncwarp();
    if (p.split > 1) cluster_sync();  // no rank leaves while its parts are being read
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, p.tmem_cols);
    }
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

}  // namespace
}  // namespace split

// When the split kernel runs, and how it is cut.  A cut is good when all its
// CTAs run at once: every further wave costs 4 to 5 us of set-up and join
// (16 x 14336 x 4096, 112 tiles: split in 2, 224 CTAs on 296 places 23.6 us;
// in 4, 448 CTAs, 28.2 us; in 8, 35.6 us).  So:
//   tile rows  M rounded up to 16 up to M = 128, else 128; 64 above M = 64 where
//              that still splits in four or more (256 x 1024 x 1024: 64 rows
//              and split 4 7.6 us, 128 rows and split 6 8.7 us).
//   split      the largest with one CTA per SM (512 x 512 x 512, 32 tiles: 4
//              6.6 us, 8 with two CTAs per SM 9.5 us).  Where that is 2 or less and
//              leaves a CTA 24 k-blocks or more, the largest with two per SM
//              (1 x 14336 x 4096: 27.0 us for 1, 24.4 us for 2; weight gradient
//              1024 x 1024 over 8192: 32.4 us for 2, 25.3 us for 4).
//   ring       that of two CTAs per SM (a shorter first ring-full starts
//              sooner: 1 x 256 x 8192 9.6 against 10.4 us), but a whole SM's where
//              half of one holds three stages or fewer (128 x 4096 x 4096: 14.4 against
//              15.5 us).
// Against the pair kernel: up to M = 128 the split kernel, unless its tiles
// exceed one wave above M = 96 (128 x 32768 x 2048: 36.6 against 32.6 us);
// above, where the tiles leave room to split at all (1024 x 1024 x 4096 18.0
// against 26.0 us; 1024 x 4096 x 4096, 256 tiles, 44.7 against 28.6 us).
// Several jobs (the gradients of a call) share one grid; they go to the pair
// kernel when one of them would alone.
int split_plan(const Product &p, SplitPlan *plan) {
    using namespace split;
    const Device *dev = nullptr;
    const int rc = prepare_device(&dev);
    if (rc != CUDAIR_OK) return rc;
    const int w_tiles = p.tiles_of_b();
    // The largest split whose clusters all fit, with one or two CTAs per SM (0: none).
    auto fits = [&](int64_t tiles, int64_t kb, int two) {
        for (int s = static_cast<int>(std::min<int64_t>(MAX_SPLIT, std::max<int64_t>(kb, 1))); s > 0; --s)
            if (tiles <= dev->clusters[two][s]) return s;
        return 0;
    };
    plan->split = 0;
    int64_t total = 0, most_kb = 0;
    int most_mt = 0;
    for (int i = 0; i < p.jobs; ++i) {
        const Job &j = p.job[i];
        const int64_t n_tiles = (j.N + NT - 1) / NT, kb = (j.K + BK - 1) / BK * j.parts;
        auto tiles = [&](int mt) { return (j.M + mt - 1) / mt * n_tiles; };
        const int unit = j.a[0].mn ? 64 : 16;
        int mt = static_cast<int>(std::min<int64_t>(128, (j.M + unit - 1) / unit * unit));
        const int one = fits(tiles(mt), kb, 0);
        if (j.M > 128 ? one < 2 : j.M > 96 && one < 1) return CUDAIR_OK;
        if (mt > 64 && p.jobs == 1 && fits(tiles(64), kb, 0) >= 4) mt = 64;
        plan->mt[i] = mt;
        most_mt = std::max(most_mt, mt);
        most_kb = std::max(most_kb, kb);
        total += tiles(mt);
    }
    const int one = fits(total, most_kb, 0);
    // A stage of which fewer than four fit half an SM.
    const bool deep = w_tiles * static_cast<int>(W_TILE) + most_mt * BK * 2 > 28 * 1024;
    const bool can_share = !(w_tiles == 2 && most_mt > 64);
    int split = std::max(one, 1), two = deep ? 0 : 1;
    // Where even whole tiles exceed one wave (wide N), two CTAs per SM overlap
    // one's join with the other's stream.
    if (can_share && (one == 0 || (one <= 2 && most_kb >= 24 * split))) {
        split = std::max(fits(total, most_kb, 1), 1);
        two = 1;
    }
    if (total * split > INT32_MAX)
        return set_error(CUDAIR_ERR_INVALID, "cudair: linear: %lld tiles are too many", (long long)total);
    plan->split = split;
    // Launch, set-up and join, then a CTA's k-blocks at the pace that its share
    // of an SM and of HBM allows (tiles of 128 rows: 16 k-blocks a CTA with 128 CTAs 13.7
    // us, with 256 CTAs 18.9 us).
    const double ctas = static_cast<double>(total * split), places = dev->clusters[two][split] * split;
    const double per_sm = std::min(ctas, places) / dev->clusters[0][1];
    plan->time = 5.5 + static_cast<double>((most_kb + split - 1) / split) * (0.3 + 0.29 * per_sm) *
                           std::max(1.0, ctas / places);
    plan->stages =
        std::min(MAX_STAGES, static_cast<int>((kBudget[two] - fixed_bytes()) / ring_bytes(w_tiles, most_mt, 1)));
    return CUDAIR_OK;
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
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(plan.split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(tiles) * plan.split, 1, 1);
    cfg.blockDim = dim3(static_cast<unsigned>(threads(many ? 8 : 4)), 1, 1);
    cfg.dynamicSmemBytes =
        std::max(fixed_bytes() + ring_bytes(w_tiles, most_mt, plan.stages), smem_floor(args.tmem_cols));
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = p.pdl() ? 2 : 1;
    const cudaError_t e = p.gated ? (many ? cudaLaunchKernelEx(&cfg, product_split_kernel<true, 8>, maps, args)
                                          : cudaLaunchKernelEx(&cfg, product_split_kernel<true, 4>, maps, args))
                                  : (many ? cudaLaunchKernelEx(&cfg, product_split_kernel<false, 8>, maps, args)
                                          : cudaLaunchKernelEx(&cfg, product_split_kernel<false, 4>, maps, args));
    return e == cudaSuccess ? CUDAIR_OK : cuda_error(e, "product_split_kernel launch");
}

}  // namespace ffn
}  // namespace cudair
