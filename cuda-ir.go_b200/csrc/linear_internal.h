// linear_internal.h - one product of the feed-forward operators, as their
// entry points describe it to the kernels that run it.
#pragma once

#include "cudair_internal.h"

namespace cudair {
namespace ffn {

// A 16-bit operand: `rows` rows of the product (of A) or columns (of B) by
// `depth` of the contraction.  As stored, either the contraction runs along
// memory (mn false) or the rows do (mn true).
struct Operand {
    const void *p = nullptr;
    int64_t ld = 0;
    bool mn = false;
};

// D[i] = epilogue(A[i] . B[i]) for one or two problems of one shape:
//   plain    one problem
//   pair     two independent problems (the gradients of two weights)
//   sum      D[0] = epilogue(A[0].B[0] + A[1].B[1]) (the gradient of X)
//   gated    D[0] = act(A[0].B[0]) * (A[0].B[1])
enum class Form { plain, pair, sum, gated };

struct OutMat {
    void *p = nullptr;
    int64_t ld = 0;
    bool f32 = false;
};

struct Product {
    Form form = Form::plain;
    int64_t M = 0, N = 0, K = 0;
    Operand a[2], b[2];
    OutMat d[2];
    const void *bias = nullptr;  // N values (plain form)
    bool bias16 = false;
    OutMat residual;             // plain form
    OutMat z[2];                 // plain: Z in z[0]; gated: G and U
    int act = CUDAIR_ACT_NONE;
    bool bf16 = false;
    bool b_weights = false;      // B is a weight: no kernel of the same call writes it
    // Not the first kernel of its call: it may be launched while the one
    // before it ends (programmatic dependent launch), whatever the mode of
    // cudair_set_gemm_pdl.  It waits for that kernel before it reads what the
    // call computes.
    bool chained = false;

    bool pdl() const { return chained || gemm_pdl_mode() > 0; }
    // Whether the weights may be requested before that wait: nothing that is
    // still running writes them.  A chained kernel's predecessors are the call's own,
    // unless the call's first kernel overlaps the caller's (mode 1).
    bool weights_early() const { return b_weights && (gemm_pdl_mode() == 2 || (chained && gemm_pdl_mode() == 0)); }
};

// Runs the product on the current device: M and N positive, K >= 0.
int product_launch(const Product &p, cudaStream_t stream);

// The persistent CTA-pair kernel (linear_sm100.cu).
int product_pair_launch(const Product &p, int sm_count, unsigned int *status, cudaStream_t stream);

// The split kernel (linear_split_sm100.cu): tiles of mt rows x 128 columns,
// the contraction shared by `split` CTAs with a ring of `stages` each.
struct SplitPlan {
    int mt = 0, split = 0, stages = 0;
};
int product_split_launch(const Product &p, const SplitPlan &plan, unsigned int *status, cudaStream_t stream);
// How the split kernel should run this product; plan->split is 0 where the
// pair kernel is the faster one.
int split_plan(const Product &p, SplitPlan *plan);

// Shared by the two: an operand's tensor map, with boxes of 64 k x box_rows
// rows where k runs along memory, else of 64 rows x 64 k; 128-byte swizzle.
int operand_map(CUtensorMap *out, const Operand &o, int64_t rows, int64_t depth, uint32_t box_rows, bool bf16);

}  // namespace ffn
}  // namespace cudair
