// linear_internal.h - the products of one call of a feed-forward operator, as
// the entry points describe them to the kernels that run them.
#pragma once

#include "cudair_internal.h"

namespace cudair {
namespace ffn {

// A 16-bit operand: rows of the product (of A) or columns (of B) by the
// contraction.  As stored, either the contraction runs along memory (mn
// false) or the rows do (mn true).
struct Operand {
    const void *p = nullptr;
    int64_t ld = 0;
    bool mn = false;
};

struct OutMat {
    void *p = nullptr;
    int64_t ld = 0;
    bool f32 = false;
};

// D = sum over parts of A[i] . B[i], M x N, each contraction K long.  In a
// gated call (one job, one part) B[0] and B[1] are the two weights.
struct Job {
    int64_t M = 0, N = 0, K = 0;
    int parts = 1;
    Operand a[2], b[2];
    OutMat d;
    bool b_weights = false;  // B is a weight: no kernel of the same call writes it
};

constexpr int kMaxJobs = 3;

// The independent products that one launch computes: one with an epilogue
// (linear, gated), or the gradients of a call, which share the SMs so that the
// last wave of one is filled by the next.
struct Product {
    int jobs = 0;
    Job job[kMaxJobs];
    bool gated = false;
    const void *bias = nullptr;  // N values (linear)
    bool bias16 = false;
    OutMat residual;             // linear
    OutMat z[2];                 // linear: Z; gated: G and U
    int act = CUDAIR_ACT_NONE;
    bool bf16 = false;
    // Not the first kernel of its call: it may be launched while the one
    // before it ends (programmatic dependent launch), whatever the mode of
    // cudair_set_gemm_pdl.  It waits for that kernel before it reads what the
    // call computes.
    bool chained = false;
    // That mode, read once by the entry point: another thread may set it while
    // the call's kernels, which rely on one another's launches, are being set up.
    int pdl_mode = 0;
    // cudair_set_linear_kernel, read with it.
    int kernel = 0, width = 0;

    bool pdl() const { return chained || pdl_mode > 0; }
    // Whether weights may be requested before that wait: nothing that is still
    // running writes them.  A chained kernel's predecessors are the call's own,
    // unless the call's first kernel overlaps the caller's (mode 1).
    bool weights_early() const { return pdl_mode == 2 || (chained && pdl_mode == 0); }
    int tiles_of_b() const { return gated ? 2 : 1; }
};

// Runs the products on the current device.  Every job has M and N positive.
int product_launch(const Product &p, cudaStream_t stream);

// The persistent CTA-pair kernel (linear_sm100.cu), and an estimate of its time
// in microseconds.
int product_pair_launch(const Product &p, int sm_count, unsigned int *status, cudaStream_t stream);
int product_pair_time(const Product &p, int sm_count, double *us);

// The split kernel (linear_split_sm100.cu): tiles of mt rows x 128 columns,
// the contraction shared by `split` CTAs with a ring of `stages` each.
struct SplitPlan {
    int mt[kMaxJobs] = {}, split = 0, stages = 0;
    double time = 0.0;  // estimated, in microseconds
};
int split_plan(const Product &p, SplitPlan *plan);
int product_split_launch(const Product &p, const SplitPlan &plan, unsigned int *status, cudaStream_t stream);

// Shared by the two: an operand's tensor map, with boxes of 64 k x box_rows
// rows where k runs along memory, else of 64 rows x 64 k; 128-byte swizzle.
int operand_map(CUtensorMap *out, const Operand &o, int64_t rows, int64_t depth, uint32_t box_rows, bool bf16);

}  // namespace ffn
}  // namespace cudair
