// The entry points of linear.cu over fakes of everything below them, so that
// what one call launches can be read without a GPU.
//
//   launches CALL MODE [MODE...] [-- KERNEL WIDTH]
//
// CALL is linear, gated, linear_backward or gated_backward; the launch mode
// (cudair_set_gemm_pdl) reads as the MODEs one after the other, the last one
// from then on, as if another thread set it during the call.  KERNEL and WIDTH go
// to cudair_set_linear_kernel first.  Prints one line
// per launch: the element-wise kernel's attributes, and what a product launch
// would do about its own.
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "../../cuda-ir.go_b200/csrc/linear_internal.h"

static int g_modes[16], g_mode_count = 0, g_mode_reads = 0;

namespace cudair {
void clear_error() {}
int set_error(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vfprintf(stderr, fmt, ap);
    va_end(ap);
    fputc('\n', stderr);
    return code;
}
int cuda_error(cudaError_t, const char *op) { return set_error(CUDAIR_ERR_CUDA, "%s", op); }
int gemm_pdl_mode() {
    const int i = g_mode_reads < g_mode_count ? g_mode_reads : g_mode_count - 1;
    ++g_mode_reads;
    return g_modes[i];
}
int sm_count_current_device(int *count) {
    *count = 148;
    return CUDAIR_OK;
}
int wait_status_current_device(unsigned int **status) {
    static unsigned int word;
    *status = &word;
    return CUDAIR_OK;
}
namespace ffn {
// One launch of all jobs by the split kernel, whatever the sizes.
int split_plan(const Product &, SplitPlan *plan) {
    plan->time = 1.0;
    return CUDAIR_OK;
}
int product_pair_time(const Product &, int, double *us) {
    *us = 2.0;
    return CUDAIR_OK;
}
int product_pair_launch(const Product &p, int, unsigned int *, cudaStream_t) {
    printf("pairs jobs=%d programmatic=%d weights_early=%d width=%d\n", p.jobs, p.pdl(), p.weights_early(), p.width);
    return CUDAIR_OK;
}
int product_split_launch(const Product &p, const SplitPlan &, unsigned int *, cudaStream_t) {
    printf("product jobs=%d programmatic=%d weights_early=%d\n", p.jobs, p.pdl(), p.weights_early());
    return CUDAIR_OK;
}
}  // namespace ffn
}  // namespace cudair

// In place of the runtime's.
extern "C" cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t *cfg, const void *, void **) {
    int programmatic = 0, cluster = 0;
    for (unsigned i = 0; i < cfg->numAttrs; ++i) {
        if (cfg->attrs[i].id == cudaLaunchAttributeProgrammaticStreamSerialization) programmatic = 1;
        if (cfg->attrs[i].id == cudaLaunchAttributeClusterDimension)
            cluster = static_cast<int>(cfg->attrs[i].val.clusterDim.x);
    }
    printf("elementwise programmatic=%d cluster=%d\n", programmatic, cluster);
    return cudaSuccess;
}

int main(int argc, char **argv) {
    if (argc < 3) return 2;
    int i = 2;
    for (; i < argc && strcmp(argv[i], "--") && g_mode_count < 16; ++i) g_modes[g_mode_count++] = atoi(argv[i]);
    if (i + 2 < argc && cudair_set_linear_kernel(atoi(argv[i + 1]), atoi(argv[i + 2])) != CUDAIR_OK) return 3;
    const char *how = argv[1];
    // Sixteen separate arrays; nothing reads them.
    char *at[16];
    for (int i = 0; i < 16; ++i) at[i] = reinterpret_cast<char *>(0x7F0000000000ll + (static_cast<long long>(i) << 24));
    const int64_t M = 512, N = 256, K = 128;
    int rc = 2;
    if (!strcmp(how, "linear")) {
        cudair_linear_args q = {};
        q.a = at[0], q.b = at[1], q.d = at[2];
        q.M = M, q.N = N, q.K = K, q.lda = K, q.ldb = N, q.ldd = N;
        rc = cudair_linear(&q, nullptr);
    } else if (!strcmp(how, "gated")) {
        cudair_gated_args q = {};
        q.x = at[0], q.wg = at[1], q.wu = at[2], q.h = at[3];
        q.M = M, q.N = N, q.K = K, q.ldx = K, q.ldwg = N, q.ldwu = N, q.ldh = N;
        rc = cudair_gated(&q, nullptr);
    } else if (!strcmp(how, "linear_backward")) {
        cudair_linear_backward_args q = {};
        q.dy = at[0], q.a = at[1], q.b = at[2], q.z = at[3], q.dz = at[4], q.da = at[5], q.db = at[6];
        q.dbias = reinterpret_cast<float *>(at[7]);
        q.M = M, q.N = N, q.K = K, q.act = CUDAIR_ACT_SILU;
        q.lddy = q.ldz = q.lddz = N, q.lda = q.ldda = K, q.ldb = q.lddb = N;
        rc = cudair_linear_backward(&q, nullptr);
    } else if (!strcmp(how, "gated_backward")) {
        cudair_gated_backward_args q = {};
        q.dh = at[0], q.x = at[1], q.wg = at[2], q.wu = at[3], q.g = at[4], q.u = at[5], q.dg = at[6], q.du = at[7];
        q.dx = at[8], q.dwg = at[9], q.dwu = at[10];
        q.M = M, q.N = N, q.K = K, q.act = CUDAIR_ACT_SILU;
        q.lddh = q.ldg = q.ldu = q.lddg = q.lddu = N, q.ldx = q.lddx = K;
        q.ldwg = q.ldwu = q.lddwg = q.lddwu = N;
        rc = cudair_gated_backward(&q, nullptr);
    }
    return rc;
}
