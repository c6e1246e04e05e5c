/* fp4.c -- entry points of microscaled 4-bit floating point: quantisation and reading back, the plain
 * and the gated product, and the norms around a block whose result may leave quantised. Argument
 * checks are the launchers'; every function returns 0 or the CUDA error code that
 * fluke_last_error() then tells in words. */
#include <fluke/fluke.h>

#include "gpu_common.h"

size_t fluke_fp4_scale_bytes(int rows, int cols, int format) {
    size_t block = format == FLUKE_FP4_MX ? 32 : 16, tiles;
    if (rows <= 0 || cols <= 0 || cols % 32 != 0 || (format != FLUKE_FP4_MX && format != FLUKE_FP4_NV)) return 0;
    tiles = ((size_t)cols + 4 * block - 1) / (4 * block);
    return ((size_t)rows + 127) / 128 * tiles * 512;
}

int fluke_quant_mxfp4_gpu(const void *in, void *out, void *scale, int n_tokens, int hidden_dim, int dtype) {
    if (dtype != FLUKE_F16 && dtype != FLUKE_BF16) return fluke_host_note_error(1 /* cudaErrorInvalidValue */);
    return fluke_host_note_error(fluke_sm100_quant_fp4(in, out, scale, NULL, n_tokens, hidden_dim, FLUKE_SM100_FP4_MX,
                                                       dtype == FLUKE_BF16, fluke_host_stream()));
}

int fluke_quant_nvfp4_gpu(const void *in, void *out, void *scale, void *row_scale, int n_tokens, int hidden_dim,
                          int dtype) {
    if (dtype != FLUKE_F16 && dtype != FLUKE_BF16) return fluke_host_note_error(1);
    return fluke_host_note_error(fluke_sm100_quant_fp4(in, out, scale, row_scale, n_tokens, hidden_dim,
                                                       FLUKE_SM100_FP4_NV, dtype == FLUKE_BF16, fluke_host_stream()));
}

int fluke_dequant_mxfp4_gpu(const void *in, const void *scale, void *out, int n_tokens, int hidden_dim, int dtype) {
    if (dtype != FLUKE_F16 && dtype != FLUKE_BF16) return fluke_host_note_error(1);
    return fluke_host_note_error(fluke_sm100_dequant_fp4(in, scale, NULL, out, n_tokens, hidden_dim, FLUKE_SM100_FP4_MX,
                                                         dtype == FLUKE_BF16, fluke_host_stream()));
}

int fluke_dequant_nvfp4_gpu(const void *in, const void *scale, const void *row_scale, void *out, int n_tokens,
                            int hidden_dim, int dtype) {
    if (dtype != FLUKE_F16 && dtype != FLUKE_BF16) return fluke_host_note_error(1);
    return fluke_host_note_error(fluke_sm100_dequant_fp4(in, scale, row_scale, out, n_tokens, hidden_dim,
                                                         FLUKE_SM100_FP4_NV, dtype == FLUKE_BF16, fluke_host_stream()));
}

static int gemm(fluke_sm100_gemm_fp4_t *g, int M, int N, int K, int dtype) {
    if (dtype != FLUKE_F16 && dtype != FLUKE_BF16) return fluke_host_note_error(1);
    g->M = M; g->N = N; g->K = K;
    g->bf16 = dtype == FLUKE_BF16;
    return fluke_host_note_error(fluke_sm100_gemm_fp4(g, fluke_host_stream()));
}

int fluke_gemm_mxfp4_gpu(void *out, const void *a, const void *a_scale, const void *b, const void *b_scale, int M, int N,
                         int K, int dtype) {
    fluke_sm100_gemm_fp4_t g = {0};
    g.format = FLUKE_SM100_FP4_MX;
    g.out = out; g.a = a; g.a_scale = a_scale; g.b = b; g.b_scale = b_scale;
    return gemm(&g, M, N, K, dtype);
}

int fluke_gemm_nvfp4_gpu(void *out, const void *a, const void *a_scale, const void *a_row, const void *b,
                         const void *b_scale, const void *b_row, int M, int N, int K, int dtype) {
    fluke_sm100_gemm_fp4_t g = {0};
    g.format = FLUKE_SM100_FP4_NV;
    g.out = out; g.a = a; g.a_scale = a_scale; g.a_row = (const float *)a_row;
    g.b = b; g.b_scale = b_scale; g.b_row = (const float *)b_row;
    return gemm(&g, M, N, K, dtype);
}

int fluke_gated_mlp_mxfp4_gpu(void *out, const void *a, const void *a_scale, const void *gate, const void *gate_scale,
                              const void *up, const void *up_scale, int M, int N, int K, int dtype) {
    fluke_sm100_gemm_fp4_t g = {0};
    if (!up) return fluke_host_note_error(1);
    g.format = FLUKE_SM100_FP4_MX;
    g.out = out; g.a = a; g.a_scale = a_scale; g.b = gate; g.b_scale = gate_scale; g.b2 = up; g.b2_scale = up_scale;
    return gemm(&g, M, N, K, dtype);
}

int fluke_gated_mlp_nvfp4_gpu(void *out, const void *a, const void *a_scale, const void *a_row, const void *gate,
                              const void *gate_scale, const void *gate_row, const void *up, const void *up_scale,
                              const void *up_row, int M, int N, int K, int dtype) {
    fluke_sm100_gemm_fp4_t g = {0};
    if (!up) return fluke_host_note_error(1);
    g.format = FLUKE_SM100_FP4_NV;
    g.out = out; g.a = a; g.a_scale = a_scale; g.a_row = (const float *)a_row;
    g.b = gate; g.b_scale = gate_scale; g.b_row = (const float *)gate_row;
    g.b2 = up; g.b2_scale = up_scale; g.b2_row = (const float *)up_row;
    return gemm(&g, M, N, K, dtype);
}

int fluke_rmsnorm_block_gpu(const fluke_rmsnorm_block_t *b) {
    fluke_sm100_rmsnorm_block_t s = {0};
    if (!b || (b->dtype != FLUKE_F16 && b->dtype != FLUKE_BF16)) return fluke_host_note_error(1);
    s.rows = b->n_tokens; s.cols = b->hidden_dim; s.seqlen = b->seqlen;
    s.bf16 = b->dtype == FLUKE_BF16;
    /* without the second norm only the stream is written, whatever the format */
    s.out_format = b->pre_weight ? b->out_format : 3;
    if (b->out_format != 0 && b->out_format != FLUKE_FP4_MX && b->out_format != FLUKE_FP4_NV)
        return fluke_host_note_error(1);
    s.x = b->x; s.residual = b->residual; s.residual_out = b->residual_out;
    s.w_post = b->post_weight; s.gate = b->gate; s.w_pre = b->pre_weight;
    s.out = b->out; s.scale = b->scale; s.row_scale = (float *)b->row_scale;
    s.alpha = b->alpha; s.eps = b->eps;
    return fluke_host_note_error(fluke_sm100_rmsnorm_block(&s, fluke_host_stream()));
}
