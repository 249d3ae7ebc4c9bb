// linear.cu - the entry points of the feed-forward operators (cudair_linear,
// cudair_gated and their gradients): argument rules, the products they are made of,
// and the element-wise step of the gradients.
//
// The gradients' element-wise step (act_grad_kernel):
//   linear  dZ = dY * act'(Z),  dbias[n] = sum_m dZ[m, n]
//   gated   dG = dH * U * act'(G),  dU = dH * act(G)
// dZ, dG and dU are then operands of two tensor-core products each, so they
// are rounded to 16 bits once here: doing it inside the products would repeat the
// activation for every tile that reads them.  Bound by HBM: 6 bytes an element
// (linear: two reads, one write), 10 (gated: three reads, two writes).  4096 x
// 14336: gated (silu) 94 us, 6.3 TB/s; linear (gelu_tanh) 55 to 60 us, 5.9 to
// 6.4 TB/s, with dbias 66 to 70 us.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <initializer_list>

#include "cudair_internal.h"
#include "linear_epilogue.cuh"
#include "linear_internal.h"
#include "sm100.cuh"

namespace cudair {
namespace ffn {

constexpr int EW_THREADS = 256;
constexpr int EW_COLS = 64;              // columns per block: 8 threads of 8 columns
constexpr int EW_ROWS = EW_THREADS / 8;  // rows per step of a block

struct EwArgs {
    int M, N;
    int chunks;       // blocks per strip of columns
    int rows;         // rows per block
    int act;
    const void *dy, *z, *u;  // gated: dH, G, U
    void *dz, *du;           // gated: dG, dU
    long long lddy, ldz, ldu, lddz, lddu;
    float *dbias;
};

// Eight columns of a row as they lie in memory: one 16-byte load of 16-bit
// values, two of fp32.  Not through the read-only path: an output may lie over
// the matrix.
struct Raw8 {
    uint4 lo, hi;
};
__device__ __forceinline__ Raw8 load_raw8(const void *base, long long ld, long long row, int col, bool f32) {
    Raw8 r;
    if (f32) {
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const float *>(base) + row * ld + col);
        r.lo = p[0];
        r.hi = p[1];
    } else {
        r.lo = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + row * ld + col);
        r.hi = r.lo;
    }
    return r;
}
__device__ __forceinline__ void convert8(const Raw8 &r, bool f32, bool bf16, float (&v)[8]) {
    if (f32) {
        const uint32_t w[8] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w, r.hi.x, r.hi.y, r.hi.z, r.hi.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    } else {
        const uint32_t w[4] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) unpack16(w[j], bf16, v[2 * j], v[2 * j + 1]);
    }
}
// The columns of a last block that ends inside the eight, one by one.
__device__ __forceinline__ void load8_edge(const void *base, long long ld, long long row, int col, int N, bool f32,
                                           bool bf16, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        v[j] = col + j >= N ? 0.0f
               : f32        ? (static_cast<const float *>(base) + row * ld + col)[j]
                            : from16((static_cast<const uint16_t *>(base) + row * ld + col)[j], bf16);
}
__device__ __forceinline__ void store8(void *base, long long ld, long long row, int col, int N, bool bf16,
                                       const float (&v)[8]) {
    uint16_t *p = static_cast<uint16_t *>(base) + row * ld + col;
    if (col + 8 <= N) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack16(v[2 * j], v[2 * j + 1], bf16);
        st_v4(p, w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (col + j < N) p[j] = to16(v[j], bf16);
    }
}

// A block takes `rows` rows of one strip of 64 columns, EW_ROWS x BATCH rows
// at a time.  A batch's loads are all issued before anything waits for one of
// them (a load and its conversion behind a row check each kept one load in
// flight per thread: 4096 x 14336 gated took 480 us), and an element is stored
// by the thread that loaded it, so the outputs may lie over the inputs.
//
// SUM (dbias): the blocks of a strip are one cluster of at most eight.  Each
// adds its rows in fp32 registers, then over its 32 row-threads in shared
// memory; the cluster's first block reads the others' sums and adds them in
// rank order.  No atomics and no workspace: the result does not depend on
// timing, and calls may overlap.
// The types are template parameters: chosen at run time, the conversions of both
// are computed and one kept, and with gelu_tanh the instructions, not the bytes,
// set the time.
template <bool GATED, bool F32>
struct EwCfg {
    static constexpr int BATCH = GATED || F32 ? 2 : 4;
    static constexpr int BLOCKS = GATED ? 3 : 4;  // per SM
};

template <bool GATED, bool SUM, bool bf16, bool f32>
__global__ void __launch_bounds__(EW_THREADS, (EwCfg<GATED, f32>::BLOCKS)) act_grad_kernel(const EwArgs p) {
    constexpr int BATCH = EwCfg<GATED, f32>::BATCH;
    __shared__ float part[EW_ROWS][EW_COLS];
    const int strips = (p.N + EW_COLS - 1) / EW_COLS;
    // A strip's blocks next to one another for the cluster; else row by row.
    const int strip = SUM ? static_cast<int>(blockIdx.x / p.chunks) : static_cast<int>(blockIdx.x % strips);
    const int chunk = SUM ? static_cast<int>(blockIdx.x % p.chunks) : static_cast<int>(blockIdx.x / strips);
    const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
    const int col = strip * EW_COLS + tx * 8;
    const long long first = static_cast<long long>(chunk) * p.rows;
    const long long last = min(first + p.rows, static_cast<long long>(p.M));
    const bool has_z = GATED || p.act != CUDAIR_ACT_NONE;
    float sum[8] = {};

    auto finish = [&](long long r, float (&dy)[8], const float (&z)[8], const float (&u)[8]) {
        if (GATED) {
            float dg[8], du[8];
            with_act(p.act, [&](auto tag) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float value, grad;
                    act_both<decltype(tag)::value>(z[j], value, grad);
                    dg[j] = dy[j] * u[j] * grad;
                    du[j] = dy[j] * value;
                }
            });
            store8(p.dz, p.lddz, r, col, p.N, bf16, dg);
            store8(p.du, p.lddu, r, col, p.N, bf16, du);
        } else {
            if (has_z)
                with_act(p.act, [&](auto tag) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float value, grad;
                        act_both<decltype(tag)::value>(z[j], value, grad);
                        dy[j] *= grad;
                    }
                });
            if (p.dz) store8(p.dz, p.lddz, r, col, p.N, bf16, dy);
            if (SUM) {
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] += dy[j];
            }
        }
    };

    grid_dependency_wait();
    // The products may set up, and request weights: after the wait, so that all
    // kernels before this one have ended.
    if (threadIdx.x == 0) grid_launch_dependents();
    if (col < p.N) {
        const bool whole = col + 8 <= p.N;
        long long r0 = first + ty;
        if (whole)
            for (; r0 + EW_ROWS * (BATCH - 1) < last; r0 += EW_ROWS * BATCH) {
                Raw8 dy[BATCH], z[BATCH], u[BATCH];
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                    const long long r = r0 + b * EW_ROWS;
                    dy[b] = load_raw8(p.dy, p.lddy, r, col, f32);
                    if (has_z) z[b] = load_raw8(p.z, p.ldz, r, col, false);
                    if (GATED) u[b] = load_raw8(p.u, p.ldu, r, col, false);
                }
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                    float fy[8], fz[8] = {}, fu[8] = {};
                    convert8(dy[b], f32, bf16, fy);
                    if (has_z) convert8(z[b], false, bf16, fz);
                    if (GATED) convert8(u[b], false, bf16, fu);
                    finish(r0 + b * EW_ROWS, fy, fz, fu);
                }
            }
        for (; r0 < last; r0 += EW_ROWS) {
            float fy[8], fz[8] = {}, fu[8] = {};
            if (whole) {
                const Raw8 dy = load_raw8(p.dy, p.lddy, r0, col, f32);
                Raw8 z = {}, u = {};
                if (has_z) z = load_raw8(p.z, p.ldz, r0, col, false);
                if (GATED) u = load_raw8(p.u, p.ldu, r0, col, false);
                convert8(dy, f32, bf16, fy);
                convert8(z, false, bf16, fz);
                convert8(u, false, bf16, fu);
            } else {
                load8_edge(p.dy, p.lddy, r0, col, p.N, f32, bf16, fy);
                if (has_z) load8_edge(p.z, p.ldz, r0, col, p.N, false, bf16, fz);
                if (GATED) load8_edge(p.u, p.ldu, r0, col, p.N, false, bf16, fu);
            }
            finish(r0, fy, fz, fu);
        }
    }
    if (SUM) {
#pragma unroll
        for (int j = 0; j < 8; ++j) part[ty][tx * 8 + j] = sum[j];
        __syncthreads();
        float s = 0.0f;
        if (threadIdx.x < EW_COLS) {
#pragma unroll
            for (int r = 0; r < EW_ROWS; ++r) s += part[r][threadIdx.x];
            part[0][threadIdx.x] = s;
        }
        cluster_sync();
        if (chunk == 0 && threadIdx.x < EW_COLS) {
            const uint32_t mine = smem_u32(&part[0][threadIdx.x]);
            for (int c = 1; c < p.chunks; ++c) {
                float other;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other) : "r"(mapa_shared(mine, c)) : "memory");
                s += other;
            }
            const int n = strip * EW_COLS + static_cast<int>(threadIdx.x);
            if (n < p.N) p.dbias[n] = s;
        }
        __syncwarp();
        cluster_sync();  // no block leaves while its sums are being read
    }
}

namespace {

template <bool GATED, bool SUM>
cudaError_t act_grad_start(const cudaLaunchConfig_t &cfg, const EwArgs &p, bool bf16, bool dy_f32) {
    if (!GATED && dy_f32)
        return bf16 ? cudaLaunchKernelEx(&cfg, act_grad_kernel<GATED, SUM, true, !GATED>, p)
                    : cudaLaunchKernelEx(&cfg, act_grad_kernel<GATED, SUM, false, !GATED>, p);
    return bf16 ? cudaLaunchKernelEx(&cfg, act_grad_kernel<GATED, SUM, true, false>, p)
                : cudaLaunchKernelEx(&cfg, act_grad_kernel<GATED, SUM, false, false>, p);
}

int act_grad_launch(EwArgs &p, bool gated, bool bf16, bool dy_f32, int pdl_mode, int sm_count, cudaStream_t stream) {
    const int64_t strips = (static_cast<int64_t>(p.N) + EW_COLS - 1) / EW_COLS;
    const bool sum = p.dbias != nullptr;
    const int64_t step = EW_ROWS * 4;  // whole batches
    const int64_t steps = (static_cast<int64_t>(p.M) + step - 1) / step;
    int64_t chunks = steps;
    if (sum) {
        // At most eight blocks (a portable cluster) share a strip; of those the
        // number whose last wave is fullest (224 strips on 592 places: 5 blocks
        // make 1.9 waves, 8 make 3.03).
        const int64_t places = static_cast<int64_t>(sm_count) * EwCfg<false, false>::BLOCKS;
        chunks = 1;
        double best = 1e30;
        for (int64_t c = 1; c <= 8 && c <= steps; ++c) {
            const double t = static_cast<double>((strips * c + places - 1) / places) *
                             static_cast<double>((steps + c - 1) / c);
            if (t <= best) {
                best = t;
                chunks = c;
            }
        }
    }
    p.chunks = static_cast<int>(chunks);
    p.rows = static_cast<int>((steps + chunks - 1) / chunks * step);
    if (strips * chunks > INT32_MAX)
        return set_error(CUDAIR_ERR_INVALID, "cudair: linear: M=%d x N=%d is too large", p.M, p.N);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(chunks);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(strips * chunks), 1, 1);
    cfg.blockDim = dim3(EW_THREADS, 1, 1);
    cfg.stream = stream;
    cfg.attrs = pdl_mode > 0 ? attr : attr + 1;
    cfg.numAttrs = (pdl_mode > 0 ? 1 : 0) + (sum ? 1 : 0);
    const cudaError_t e = gated ? act_grad_start<true, false>(cfg, p, bf16, dy_f32)
                          : sum ? act_grad_start<false, true>(cfg, p, bf16, dy_f32)
                                : act_grad_start<false, false>(cfg, p, bf16, dy_f32);
    return e == cudaSuccess ? CUDAIR_OK : cuda_error(e, "act_grad_kernel launch");
}

// ---- argument rules ------------------------------------------------------------------

constexpr int64_t kMaxSize = INT32_MAX - 1024;  // tile arithmetic is 32-bit

int check_sizes(const char *op, int64_t M, int64_t N, int64_t K) {
    if (M < 0 || N < 0 || K < 0)
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: negative size M=%lld N=%lld K=%lld", op, (long long)M,
                         (long long)N, (long long)K);
    if (M > kMaxSize || N > kMaxSize || K > kMaxSize)
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: sizes must be at most %lld", op, (long long)kMaxSize);
    return CUDAIR_OK;
}

// What one accumulator sums is bounded so that a tile's k-blocks take well under the
// two seconds after which a device wait gives up: 2^20 k-blocks of 0.73 us (tiles of
// two blocks, the slowest) are 0.77 s.  `parts` contractions go into one accumulator.
constexpr int64_t kMaxDepth = int64_t{1} << 26;
int check_depth(const char *op, int64_t depth, int parts = 1) {
    if (depth > kMaxDepth / parts)
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: a contraction over %lld is too long (at most %lld)", op,
                         (long long)depth, (long long)(kMaxDepth / parts));
    return CUDAIR_OK;
}

// The largest pitch, in elements: row * pitch stays far inside 64 bits.
constexpr int64_t kMaxPitch = INT64_MAX >> 34;

// Where a matrix lies, in bytes; no rows: nowhere.  (An operand that is given but not needed may
// have no such pitch: its first row counts.)
struct Extent {
    int64_t at = 0, pitch = 0, row = 0, rows = 0;
};
Extent extent(const void *p, int64_t ld, int64_t rows, int64_t cols, int elem) {
    Extent e;
    if (!p || rows == 0 || cols == 0) return e;
    e.at = static_cast<int64_t>(reinterpret_cast<uintptr_t>(p));
    e.row = cols * elem;
    e.rows = ld < cols || ld > kMaxPitch ? 1 : rows;
    e.pitch = e.rows > 1 ? ld * elem : e.row;
    return e;
}

// Whether two matrices of one pitch have a byte in common: rows i of a and j of b
// do if (i - j) pitch lies strictly between d - a.row and d + b.row, d = b.at - a.at.  (Views of
// one array, such as halves of its columns, interleave without that.)
bool rows_meet(const Extent &a, const Extent &b, int64_t pitch) {
    const int64_t d = b.at - a.at, low = d - a.row;
    int64_t k = low / pitch - (low % pitch < 0 ? 1 : 0) + 1;  // the least that is above low / pitch
    if (k < 1 - b.rows) k = 1 - b.rows;
    return k < a.rows && k * pitch < d + b.row;
}
bool overlap(const Extent &a, const Extent &b) {
    if (a.rows == 0 || b.rows == 0) return false;
    if (a.at + (a.rows - 1) * a.pitch + a.row <= b.at || b.at + (b.rows - 1) * b.pitch + b.row <= a.at) return false;
    if (a.rows == 1 || b.rows == 1 || a.pitch == b.pitch) {
        return rows_meet(a, b, a.rows > 1 ? a.pitch : b.pitch);
    }
    const Extent &few = a.rows < b.rows ? a : b, &many = a.rows < b.rows ? b : a;
    for (int64_t i = 0; i < few.rows; ++i) {
        Extent one = few;
        one.at += i * few.pitch;
        one.rows = 1;
        if (rows_meet(many, one, many.pitch)) return true;
    }
    return false;
}

// An output over an input or another output.
int check_distinct(const char *op, const char *name, const Extent &out, std::initializer_list<Extent> others) {
    for (const Extent &o : others)
        if (overlap(out, o))
            return set_error(CUDAIR_ERR_INVALID, "cudair: %s: %s lies over another matrix of the call", op, name);
    return CUDAIR_OK;
}
// An output that may be an input's own memory, element over element, but not else over it.
int check_in_place(const char *op, const char *name, const Extent &out, std::initializer_list<Extent> inputs) {
    for (const Extent &o : inputs)
        if (out.at != o.at) {
            const int rc = check_distinct(op, name, out, {o});
            if (rc != CUDAIR_OK) return rc;
        }
    return CUDAIR_OK;
}

int check_flags(const char *op, uint32_t flags, uint32_t known, uint32_t act) {
    if (flags & ~known) return set_error(CUDAIR_ERR_INVALID, "cudair: %s: unknown flags 0x%x", op, flags & ~known);
    if (act > CUDAIR_ACT_SILU)
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: unknown activation %u", op, act);
    return CUDAIR_OK;
}

// A rows x cols matrix: present, 16-byte aligned, rows of whole 16 bytes.
int check_mat(const char *op, const char *name, const void *p, int64_t ld, int64_t cols, int elem) {
    if (!p) return set_error(CUDAIR_ERR_INVALID, "cudair: %s: nil pointer (%s)", op, name);
    if (reinterpret_cast<uintptr_t>(p) & 15u)
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: %s must be 16-byte aligned", op, name);
    if (ld < cols)
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: pitch %lld of %s is below its %lld columns", op,
                         (long long)ld, name, (long long)cols);
    if (ld % (16 / elem))
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: pitch %lld of %s must be a multiple of %d (16-byte rows)",
                         op, (long long)ld, name, 16 / elem);
    if (ld > kMaxPitch)
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: pitch %lld of %s is too large", op, (long long)ld, name);
    return CUDAIR_OK;
}

#define CUDAIR_TRY(call)                        \
    do {                                        \
        const int rc_ = (call);                 \
        if (rc_ != CUDAIR_OK) return rc_;       \
    } while (0)

// cudair_set_linear_kernel: the kernel, and 16 bits further up the width.
std::atomic<int> g_kernel{0};

// A call's products, under the settings of the process as they are now.
Product new_product() {
    const int k = g_kernel.load();
    Product p;
    p.pdl_mode = gemm_pdl_mode();
    p.kernel = k & 0xFFFF;
    p.width = k >> 16;
    return p;
}

Operand operand(const void *p, int64_t ld, bool mn) {
    Operand o;
    o.p = p;
    o.ld = ld;
    o.mn = mn;
    return o;
}
OutMat out_mat(void *p, int64_t ld, bool f32) {
    OutMat m;
    m.p = p;
    m.ld = ld;
    m.f32 = f32;
    return m;
}

}  // namespace

namespace {

// What cudair_set_linear_kernel may choose.
constexpr int kSplit = 1, kPairs = 2;

// One launch, by the kernel that is the faster one by their estimates.  Up to
// 64 rows that is the split kernel: the pair kernel's 256-row tiles would read the
// weights at the pace of few SMs (gated 1 x 4672 x 7296: 124 against 26 us).
struct Launch {
    SplitPlan plan;
    bool split = true;
    double time = 0.0;
};
int plan_launch(const Product &p, int sm_count, Launch *l) {
    if (p.kernel != kPairs) {
        CUDAIR_TRY(split_plan(p, &l->plan));
        l->time = l->plan.time;
        bool few = true;
        for (int i = 0; i < p.jobs; ++i) few = few && p.job[i].M <= 64;
        if (few || p.kernel == kSplit) return CUDAIR_OK;
    }
    double pair = 0.0;
    CUDAIR_TRY(product_pair_time(p, sm_count, &pair));
    if (p.kernel == kPairs || pair < l->time) {
        l->split = false;
        l->time = pair;
    }
    return CUDAIR_OK;
}
int start(const Product &p, const Launch &l, int sm_count, unsigned int *status, cudaStream_t stream) {
    return l.split ? product_split_launch(p, l.plan, status, stream) : product_pair_launch(p, sm_count, status, stream);
}

}  // namespace

int product_launch(const Product &p, cudaStream_t stream) {
    unsigned int *status = nullptr;
    int sms = 0;
    CUDAIR_TRY(wait_status_current_device(&status));  // with the device and context checks
    CUDAIR_TRY(sm_count_current_device(&sms));
    Launch all;
    CUDAIR_TRY(plan_launch(p, sms, &all));
    constexpr double kTwoLaunches = 8.6;  // no two launches take less
    if (p.jobs > 1 && all.time > kTwoLaunches) {
        // A call's gradients share one launch (4096 x 14336 x 4096: linear 752 ->
        // 711 us, gated 1402 -> 1335 us; 301 x 515 x 1029 26 -> 15 us), unless the
        // first, whose contraction may be the longest, has few tiles that the
        // split kernel would cut: then it runs by itself, and the weights' gradients after it
        // (gated 203 x 1731 x 777: 46 us together, 25 us in two).
        Product first = p, rest = p;
        first.jobs = 1;
        rest.jobs = p.jobs - 1;
        for (int i = 0; i < rest.jobs; ++i) rest.job[i] = p.job[i + 1];
        rest.chained = true;
        Launch one, two;
        CUDAIR_TRY(plan_launch(first, sms, &one));
        CUDAIR_TRY(plan_launch(rest, sms, &two));
        if (one.time + two.time < all.time) {
            CUDAIR_TRY(start(first, one, sms, status, stream));
            return start(rest, two, sms, status, stream);
        }
    }
    return start(p, all, sms, status, stream);
}

}  // namespace ffn
}  // namespace cudair

using namespace cudair;
using namespace cudair::ffn;

CUDAIR_API int cudair_set_linear_kernel(int kernel, int width) {
    clear_error();
    if (kernel < 0 || kernel > 2)
        return set_error(CUDAIR_ERR_INVALID,
                         "cudair: linear kernel %d, want 0 (automatic), 1 (split) or 2 (CTA pairs)", kernel);
    bool known = width == 0;
    for (const int w : {192, 224, 256, 384, 448, 512}) known = known || (kernel == kPairs && width == w);
    if (!known)
        return set_error(CUDAIR_ERR_INVALID,
                         "cudair: linear tile width %d, want 0 (automatic) or, of CTA pairs, 192, 224, 256, 384, 448 or "
                         "512",
                         width);
    g_kernel.store(kernel | width << 16);
    return CUDAIR_OK;
}

CUDAIR_API int cudair_linear(const cudair_linear_args *q, void *stream) {
    clear_error();
    const char *op = "linear";
    if (!q) return set_error(CUDAIR_ERR_INVALID, "cudair: %s: nil arguments", op);
    CUDAIR_TRY(check_flags(op, q->flags,
                           CUDAIR_GEMM_BF16 | CUDAIR_GEMM_B_T | CUDAIR_LINEAR_D_F32 | CUDAIR_LINEAR_BIAS_16,
                           q->act));
    CUDAIR_TRY(check_sizes(op, q->M, q->N, q->K));
    if (q->M == 0 || q->N == 0) return CUDAIR_OK;
    const bool bt = q->flags & CUDAIR_GEMM_B_T, d_f32 = q->flags & CUDAIR_LINEAR_D_F32;
    const bool bias16 = q->flags & CUDAIR_LINEAR_BIAS_16;
    if (q->K > 0) {
        CUDAIR_TRY(check_mat(op, "a", q->a, q->lda, q->K, 2));
        CUDAIR_TRY(check_mat(op, "b", q->b, q->ldb, bt ? q->K : q->N, 2));
    }
    CUDAIR_TRY(check_mat(op, "d", q->d, q->ldd, q->N, d_f32 ? 4 : 2));
    if (q->residual) CUDAIR_TRY(check_mat(op, "residual", q->residual, q->ldres, q->N, d_f32 ? 4 : 2));
    if (q->z) CUDAIR_TRY(check_mat(op, "z", q->z, q->ldz, q->N, 2));
    if (q->bias && (reinterpret_cast<uintptr_t>(q->bias) & (bias16 ? 1u : 3u)))
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: bias must be aligned to its elements", op);
    CUDAIR_TRY(check_depth(op, q->K));
    const int d_size = d_f32 ? 4 : 2;
    const Extent a = extent(q->a, q->lda, q->M, q->K, 2), b = extent(q->b, q->ldb, bt ? q->N : q->K, bt ? q->K : q->N, 2);
    const Extent bias = extent(q->bias, q->N, 1, q->N, bias16 ? 2 : 4), z = extent(q->z, q->ldz, q->M, q->N, 2);
    const Extent d = extent(q->d, q->ldd, q->M, q->N, d_size), res = extent(q->residual, q->ldres, q->M, q->N, d_size);
    CUDAIR_TRY(check_distinct(op, "d", d, {a, b, bias, z}));
    CUDAIR_TRY(check_distinct(op, "z", z, {a, b, bias, res}));
    if (q->residual == q->d && q->residual && q->ldres != q->ldd)
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: a residual in D's memory needs D's pitch", op);
    CUDAIR_TRY(check_in_place(op, "d", d, {res}));
    Product p = new_product();
    p.jobs = 1;
    Job &j = p.job[0];
    j.M = q->M;
    j.N = q->N;
    j.K = q->K;
    j.a[0] = operand(q->a, q->lda, false);
    j.b[0] = operand(q->b, q->ldb, !bt);
    j.b_weights = true;
    j.d = out_mat(q->d, q->ldd, d_f32);
    p.z[0] = out_mat(q->z, q->ldz, false);
    p.residual = out_mat(const_cast<void *>(q->residual), q->ldres, d_f32);
    p.bias = q->bias;
    p.bias16 = bias16;
    p.act = static_cast<int>(q->act);
    p.bf16 = q->flags & CUDAIR_GEMM_BF16;
    return product_launch(p, static_cast<cudaStream_t>(stream));
}

CUDAIR_API int cudair_gated(const cudair_gated_args *q, void *stream) {
    clear_error();
    const char *op = "gated";
    if (!q) return set_error(CUDAIR_ERR_INVALID, "cudair: %s: nil arguments", op);
    CUDAIR_TRY(check_flags(op, q->flags, CUDAIR_GEMM_BF16 | CUDAIR_GEMM_B_T, q->act));
    CUDAIR_TRY(check_sizes(op, q->M, q->N, q->K));
    if (q->M == 0 || q->N == 0) return CUDAIR_OK;
    const bool bt = q->flags & CUDAIR_GEMM_B_T;
    if (q->K > 0) {
        CUDAIR_TRY(check_mat(op, "x", q->x, q->ldx, q->K, 2));
        CUDAIR_TRY(check_mat(op, "wg", q->wg, q->ldwg, bt ? q->K : q->N, 2));
        CUDAIR_TRY(check_mat(op, "wu", q->wu, q->ldwu, bt ? q->K : q->N, 2));
    }
    CUDAIR_TRY(check_mat(op, "h", q->h, q->ldh, q->N, 2));
    if (!q->g != !q->u) return set_error(CUDAIR_ERR_INVALID, "cudair: %s: g and u are given together", op);
    if (q->g) {
        CUDAIR_TRY(check_mat(op, "g", q->g, q->ldg, q->N, 2));
        CUDAIR_TRY(check_mat(op, "u", q->u, q->ldu, q->N, 2));
    }
    CUDAIR_TRY(check_depth(op, q->K));
    const int64_t wrows = bt ? q->N : q->K, wcols = bt ? q->K : q->N;
    const Extent x = extent(q->x, q->ldx, q->M, q->K, 2), h = extent(q->h, q->ldh, q->M, q->N, 2);
    const Extent wg = extent(q->wg, q->ldwg, wrows, wcols, 2), wu = extent(q->wu, q->ldwu, wrows, wcols, 2);
    const Extent g = extent(q->g, q->ldg, q->M, q->N, 2), u = extent(q->u, q->ldu, q->M, q->N, 2);
    CUDAIR_TRY(check_distinct(op, "h", h, {x, wg, wu, g, u}));
    CUDAIR_TRY(check_distinct(op, "g", g, {x, wg, wu, u}));
    CUDAIR_TRY(check_distinct(op, "u", u, {x, wg, wu}));
    Product p = new_product();
    if (p.width == 224 || p.width == 448)  // blocks of 224 columns: 112 of each product, not whole chunks of 32
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: tiles of %d columns do not take two weights", op, p.width);
    p.jobs = 1;
    p.gated = true;
    Job &j = p.job[0];
    j.M = q->M;
    j.N = q->N;
    j.K = q->K;
    j.a[0] = operand(q->x, q->ldx, false);
    j.b[0] = operand(q->wg, q->ldwg, !bt);
    j.b[1] = operand(q->wu, q->ldwu, !bt);
    j.b_weights = true;
    j.d = out_mat(q->h, q->ldh, false);
    p.z[0] = out_mat(q->g, q->ldg, false);
    p.z[1] = out_mat(q->u, q->ldu, false);
    p.act = static_cast<int>(q->act);
    p.bf16 = q->flags & CUDAIR_GEMM_BF16;
    return product_launch(p, static_cast<cudaStream_t>(stream));
}

CUDAIR_API int cudair_linear_backward(const cudair_linear_backward_args *q, void *stream) {
    clear_error();
    const char *op = "linear_backward";
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!q) return set_error(CUDAIR_ERR_INVALID, "cudair: %s: nil arguments", op);
    CUDAIR_TRY(check_flags(op, q->flags,
                           CUDAIR_GEMM_BF16 | CUDAIR_GEMM_B_T | CUDAIR_LINEAR_D_F32 | CUDAIR_LINEAR_DA_F32 |
                               CUDAIR_LINEAR_DB_F32,
                           q->act));
    CUDAIR_TRY(check_sizes(op, q->M, q->N, q->K));
    const bool bt = q->flags & CUDAIR_GEMM_B_T, dy_f32 = q->flags & CUDAIR_LINEAR_D_F32;
    const bool bf16 = q->flags & CUDAIR_GEMM_BF16, has_act = q->act != CUDAIR_ACT_NONE;
    const bool da_f32 = q->flags & CUDAIR_LINEAR_DA_F32, db_f32 = q->flags & CUDAIR_LINEAR_DB_F32;
    const bool own_dz = has_act || dy_f32;
    if (!own_dz && q->dz)
        return set_error(CUDAIR_ERR_INVALID,
                         "cudair: %s: without an activation a 16-bit dY is dZ itself: dz must be nil", op);
    if (q->M > 0 && q->N > 0) {
        CUDAIR_TRY(check_mat(op, "dy", q->dy, q->lddy, q->N, dy_f32 ? 4 : 2));
        if (has_act) CUDAIR_TRY(check_mat(op, "z", q->z, q->ldz, q->N, 2));
        if (own_dz) {
            CUDAIR_TRY(check_mat(op, "dz", q->dz, q->lddz, q->N, 2));
            if (q->dz == q->dy && (dy_f32 || q->lddz != q->lddy))
                return set_error(CUDAIR_ERR_INVALID, "cudair: %s: dz in dY's memory needs its type and pitch", op);
            if (q->dz == q->z && has_act && q->lddz != q->ldz)
                return set_error(CUDAIR_ERR_INVALID, "cudair: %s: dz in z's memory needs its pitch", op);
        }
    }
    const bool want_da = q->da && q->M > 0 && q->K > 0, want_db = q->db && q->N > 0 && q->K > 0;
    if (want_da) {
        CUDAIR_TRY(check_mat(op, "da", q->da, q->ldda, q->K, da_f32 ? 4 : 2));
        if (q->N > 0) CUDAIR_TRY(check_mat(op, "b", q->b, q->ldb, bt ? q->K : q->N, 2));
    }
    if (want_db) {
        CUDAIR_TRY(check_mat(op, "db", q->db, q->lddb, bt ? q->K : q->N, db_f32 ? 4 : 2));
        if (q->M > 0) CUDAIR_TRY(check_mat(op, "a", q->a, q->lda, q->K, 2));
    }
    if (q->dbias && (reinterpret_cast<uintptr_t>(q->dbias) & 3u))
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: dbias must be 4-byte aligned", op);
    if (want_da) CUDAIR_TRY(check_depth(op, q->N));
    if (want_db) CUDAIR_TRY(check_depth(op, q->M));
    const int64_t wrows = bt ? q->N : q->K, wcols = bt ? q->K : q->N;
    const Extent dy = extent(q->dy, q->lddy, q->M, q->N, dy_f32 ? 4 : 2);
    const Extent z = extent(q->z, q->ldz, q->M, q->N, 2);
    const Extent a = extent(q->a, q->lda, q->M, q->K, 2);
    const Extent b = extent(q->b, q->ldb, wrows, wcols, 2);
    const Extent edz = extent(q->dz, q->lddz, q->M, q->N, 2);
    const Extent da = extent(want_da ? q->da : nullptr, q->ldda, q->M, q->K, da_f32 ? 4 : 2);
    const Extent db = extent(want_db ? q->db : nullptr, q->lddb, wrows, wcols, db_f32 ? 4 : 2);
    const Extent dbias = extent(q->dbias, q->N, 1, q->N, 4);
    CUDAIR_TRY(check_in_place(op, "dz", edz, {dy, z}));
    CUDAIR_TRY(check_distinct(op, "dz", edz, {a, b, da, db}));
    CUDAIR_TRY(check_distinct(op, "da", da, {a, b, dy, z, db}));
    CUDAIR_TRY(check_distinct(op, "db", db, {a, b, dy, z}));
    CUDAIR_TRY(check_distinct(op, "dbias", dbias, {a, b, dy, z, edz, da, db}));

    int sms = 0;
    CUDAIR_TRY(sm_count_current_device(&sms));  // the device and context checks
    Product p = new_product();
    // dZ, and the bias's gradient from it (M = 0: its empty sums).
    const bool elementwise = q->N > 0 && ((own_dz && q->M > 0) || q->dbias);
    if (elementwise) {
        EwArgs e = {};
        e.M = static_cast<int>(q->M);
        e.N = static_cast<int>(q->N);
        e.act = static_cast<int>(q->act);
        e.dy = q->dy;
        e.z = has_act ? q->z : nullptr;
        e.dz = own_dz ? q->dz : nullptr;
        e.lddy = q->lddy;
        e.ldz = q->ldz;
        e.lddz = q->lddz;
        e.dbias = q->dbias;
        CUDAIR_TRY(act_grad_launch(e, false, bf16, dy_f32, p.pdl_mode, sms, s));
    }
    const void *dz = own_dz ? q->dz : q->dy;
    const int64_t lddz = own_dz ? q->lddz : q->lddy;
    p.bf16 = bf16;
    p.chained = elementwise;
    if (want_da) {
        Job &j = p.job[p.jobs++];
        j.M = q->M;
        j.N = q->K;
        j.K = q->N;
        j.a[0] = operand(dz, lddz, false);
        j.b[0] = operand(q->b, q->ldb, bt);  // the contraction runs over N
        j.b_weights = true;
        j.d = out_mat(q->da, q->ldda, da_f32);
    }
    if (want_db) {
        Job &j = p.job[p.jobs++];
        j.M = bt ? q->N : q->K;
        j.N = bt ? q->K : q->N;
        j.K = q->M;
        const Operand x = operand(q->a, q->lda, true), g = operand(dz, lddz, true);
        j.a[0] = bt ? g : x;
        j.b[0] = bt ? x : g;
        j.d = out_mat(q->db, q->lddb, db_f32);
    }
    return p.jobs ? product_launch(p, s) : CUDAIR_OK;
}

CUDAIR_API int cudair_gated_backward(const cudair_gated_backward_args *q, void *stream) {
    clear_error();
    const char *op = "gated_backward";
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!q) return set_error(CUDAIR_ERR_INVALID, "cudair: %s: nil arguments", op);
    CUDAIR_TRY(check_flags(op, q->flags,
                           CUDAIR_GEMM_BF16 | CUDAIR_GEMM_B_T | CUDAIR_LINEAR_DA_F32 | CUDAIR_LINEAR_DB_F32,
                           q->act));
    CUDAIR_TRY(check_sizes(op, q->M, q->N, q->K));
    const bool bt = q->flags & CUDAIR_GEMM_B_T, bf16 = q->flags & CUDAIR_GEMM_BF16;
    const bool dx_f32 = q->flags & CUDAIR_LINEAR_DA_F32, dw_f32 = q->flags & CUDAIR_LINEAR_DB_F32;
    if (!q->dwg != !q->dwu)
        return set_error(CUDAIR_ERR_INVALID, "cudair: %s: dwg and dwu are given together", op);
    if (q->M > 0 && q->N > 0) {
        CUDAIR_TRY(check_mat(op, "dh", q->dh, q->lddh, q->N, 2));
        CUDAIR_TRY(check_mat(op, "g", q->g, q->ldg, q->N, 2));
        CUDAIR_TRY(check_mat(op, "u", q->u, q->ldu, q->N, 2));
        CUDAIR_TRY(check_mat(op, "dg", q->dg, q->lddg, q->N, 2));
        CUDAIR_TRY(check_mat(op, "du", q->du, q->lddu, q->N, 2));
        if (q->dg == q->du) return set_error(CUDAIR_ERR_INVALID, "cudair: %s: dg and du share memory", op);
        const struct {
            const void *p;
            int64_t ld;
        } in[3] = {{q->dh, q->lddh}, {q->g, q->ldg}, {q->u, q->ldu}};
        for (const auto &m : in)
            if ((m.p == q->dg && m.ld != q->lddg) || (m.p == q->du && m.ld != q->lddu))
                return set_error(CUDAIR_ERR_INVALID, "cudair: %s: dg or du in an input's memory needs its pitch",
                                 op);
    }
    const bool want_dx = q->dx && q->M > 0 && q->K > 0, want_dw = q->dwg && q->N > 0 && q->K > 0;
    const int64_t wcols = bt ? q->K : q->N;
    if (want_dx) {
        CUDAIR_TRY(check_mat(op, "dx", q->dx, q->lddx, q->K, dx_f32 ? 4 : 2));
        if (q->N > 0) {
            CUDAIR_TRY(check_mat(op, "wg", q->wg, q->ldwg, wcols, 2));
            CUDAIR_TRY(check_mat(op, "wu", q->wu, q->ldwu, wcols, 2));
        }
    }
    if (want_dw) {
        CUDAIR_TRY(check_mat(op, "dwg", q->dwg, q->lddwg, wcols, dw_f32 ? 4 : 2));
        CUDAIR_TRY(check_mat(op, "dwu", q->dwu, q->lddwu, wcols, dw_f32 ? 4 : 2));
        if (q->M > 0) CUDAIR_TRY(check_mat(op, "x", q->x, q->ldx, q->K, 2));
    }
    if (want_dx) CUDAIR_TRY(check_depth(op, q->N, 2));
    if (want_dw) CUDAIR_TRY(check_depth(op, q->M));
    const int64_t wrows = bt ? q->N : q->K;
    const Extent dh = extent(q->dh, q->lddh, q->M, q->N, 2), g = extent(q->g, q->ldg, q->M, q->N, 2);
    const Extent u = extent(q->u, q->ldu, q->M, q->N, 2), dg = extent(q->dg, q->lddg, q->M, q->N, 2);
    const Extent du = extent(q->du, q->lddu, q->M, q->N, 2);
    const Extent x = extent(q->x, q->ldx, q->M, q->K, 2);
    const Extent wg = extent(q->wg, q->ldwg, wrows, wcols, 2);
    const Extent wu = extent(q->wu, q->ldwu, wrows, wcols, 2);
    const Extent dx = extent(want_dx ? q->dx : nullptr, q->lddx, q->M, q->K, dx_f32 ? 4 : 2);
    const Extent dwg = extent(want_dw ? q->dwg : nullptr, q->lddwg, wrows, wcols, dw_f32 ? 4 : 2);
    const Extent dwu = extent(want_dw ? q->dwu : nullptr, q->lddwu, wrows, wcols, dw_f32 ? 4 : 2);
    if (overlap(dg, du)) return set_error(CUDAIR_ERR_INVALID, "cudair: %s: dg and du share memory", op);
    CUDAIR_TRY(check_in_place(op, "dg", dg, {dh, g, u}));
    CUDAIR_TRY(check_in_place(op, "du", du, {dh, g, u}));
    CUDAIR_TRY(check_distinct(op, "dg", dg, {x, wg, wu, dx, dwg, dwu}));
    CUDAIR_TRY(check_distinct(op, "du", du, {x, wg, wu, dx, dwg, dwu}));
    CUDAIR_TRY(check_distinct(op, "dx", dx, {x, wg, wu, dh, g, u, dwg, dwu}));
    CUDAIR_TRY(check_distinct(op, "dwg", dwg, {x, wg, wu, dh, g, u, dwu}));
    CUDAIR_TRY(check_distinct(op, "dwu", dwu, {x, wg, wu, dh, g, u}));
    int sms = 0;
    CUDAIR_TRY(sm_count_current_device(&sms));  // the device and context checks
    Product p = new_product();
    const bool elementwise = q->M > 0 && q->N > 0;
    if (elementwise) {
        EwArgs e = {};
        e.M = static_cast<int>(q->M);
        e.N = static_cast<int>(q->N);
        e.act = static_cast<int>(q->act);
        e.dy = q->dh;
        e.z = q->g;
        e.u = q->u;
        e.dz = q->dg;
        e.du = q->du;
        e.lddy = q->lddh;
        e.ldz = q->ldg;
        e.ldu = q->ldu;
        e.lddz = q->lddg;
        e.lddu = q->lddu;
        CUDAIR_TRY(act_grad_launch(e, true, bf16, false, p.pdl_mode, sms, s));
    }
    p.bf16 = bf16;
    p.chained = elementwise;
    if (want_dx) {
        Job &j = p.job[p.jobs++];
        j.M = q->M;
        j.N = q->K;
        j.K = q->N;
        j.parts = 2;
        j.a[0] = operand(q->dg, q->lddg, false);
        j.a[1] = operand(q->du, q->lddu, false);
        j.b[0] = operand(q->wg, q->ldwg, bt);
        j.b[1] = operand(q->wu, q->ldwu, bt);
        j.b_weights = true;
        j.d = out_mat(q->dx, q->lddx, dx_f32);
    }
    if (want_dw) {
        const Operand x = operand(q->x, q->ldx, true);
        for (int i = 0; i < 2; ++i) {
            const Operand g = i ? operand(q->du, q->lddu, true) : operand(q->dg, q->lddg, true);
            Job &j = p.job[p.jobs++];
            j.M = bt ? q->N : q->K;
            j.N = bt ? q->K : q->N;
            j.K = q->M;
            j.a[0] = bt ? g : x;
            j.b[0] = bt ? x : g;
            j.d = i ? out_mat(q->dwu, q->lddwu, dw_f32) : out_mat(q->dwg, q->lddwg, dw_f32);
        }
    }
    return p.jobs ? product_launch(p, s) : CUDAIR_OK;
}
