/* linear.c -- entry points of the 16-bit product with its epilogue and of the gated linear recurrence.
 * Argument checks are the launchers'; every function returns 0 or the CUDA error code that
 * fluke_last_error() then tells in words. */
#include <fluke/fluke.h>

#include "gpu_common.h"

int fluke_linear_gpu(const fluke_linear_t *l) {
    fluke_sm100_linear_t g = {0};
    if (!l || (l->dtype != FLUKE_F16 && l->dtype != FLUKE_BF16)) return fluke_host_note_error(1 /* cudaErrorInvalidValue */);
    g.bf16 = l->dtype == FLUKE_BF16;
    g.activation = l->activation;
    g.M = l->M; g.N = l->N; g.K = l->K;
    g.x = l->x; g.w = l->weight; g.bias = l->bias; g.residual = l->residual; g.out = l->out;
    g.ld_x = l->ld_x; g.ld_residual = l->ld_residual; g.ld_out = l->ld_out;
    g.alpha = l->alpha;
    return fluke_host_note_error(fluke_sm100_linear(&g, fluke_host_stream()));
}

int fluke_linear_recurrence_gpu(const fluke_linear_recurrence_t *r) {
    fluke_sm100_recurrence_t s = {0};
    if (!r || (r->dtype != FLUKE_F16 && r->dtype != FLUKE_BF16)) return fluke_host_note_error(1);
    s.bf16 = r->dtype == FLUKE_BF16;
    s.T = r->T; s.B = r->B; s.H = r->H; s.reverse = r->reverse;
    s.gate = r->gate; s.value = r->value; s.out = r->out;
    s.gate_step = r->gate_step; s.gate_chunk = r->gate_chunk;
    s.value_step = r->value_step; s.value_chunk = r->value_chunk;
    s.out_step = r->out_step; s.out_chunk = r->out_chunk;
    s.lengths = (const int *)r->lengths;
    s.h0 = (const float *)r->h0; s.h_last = (float *)r->h_last; s.states = (float *)r->states;
    return fluke_host_note_error(fluke_sm100_recurrence(&s, 0, fluke_host_stream()));
}

int fluke_linear_recurrence_backward_gpu(const fluke_linear_recurrence_grad_t *r) {
    fluke_sm100_recurrence_t s = {0};
    if (!r || (r->dtype != FLUKE_F16 && r->dtype != FLUKE_BF16)) return fluke_host_note_error(1);
    s.bf16 = r->dtype == FLUKE_BF16;
    s.T = r->T; s.B = r->B; s.H = r->H; s.reverse = r->reverse;
    s.gate = r->gate; s.value = r->value; s.grad = r->grad; s.grad_gate = r->grad_gate; s.grad_value = r->grad_value;
    s.gate_step = r->gate_step; s.gate_chunk = r->gate_chunk;
    s.value_step = r->value_step; s.value_chunk = r->value_chunk;
    s.grad_step = r->grad_step; s.grad_chunk = r->grad_chunk;
    s.grad_gate_step = r->grad_gate_step; s.grad_gate_chunk = r->grad_gate_chunk;
    s.grad_value_step = r->grad_value_step; s.grad_value_chunk = r->grad_value_chunk;
    s.lengths = (const int *)r->lengths;
    s.states = (float *)r->states;   /* only read */
    s.grad_last = (const float *)r->grad_last; s.grad_h0 = (float *)r->grad_h0;
    return fluke_host_note_error(fluke_sm100_recurrence(&s, 1, fluke_host_stream()));
}
