// Requests of their own prompts stepped together (hipdec_requests_*): the rows of a step are the tokens and drafts of
// several sequences at positions of their own, with keys and values in the pages of one pool.  The products are the
// multi-row step's; rotary positions, the append and attention are the paged-cache operators, the decision about the
// drafts is the verification operator.  This file adds what lies between them.
#pragma once
#include "hipdec_prefill.h"

// rows[t][c] = (sum of the split planes) * channel scale (8-bit weights) * the row's norm factor: the step's queries,
// keys and values as fp32 rows, not yet turned
__global__ __launch_bounds__(256) void k_rq_qkv_rows(const float *__restrict__ P, int splits, size_t plane,
                                                     const float *__restrict__ wscale, float *__restrict__ rows,
                                                     const float *__restrict__ ssq, int nch, int D, int N) {
    const int t = blockIdx.y, c = 2 * (int)(blockIdx.x * blockDim.x + threadIdx.x);
    if (c >= N) return;
    float s[2] = {0.0f, 0.0f};
    pf_sum_planes<2>(P, splits, plane, (size_t)t * N + c, s);
    if (wscale) { s[0] *= wscale[c]; s[1] *= wscale[c + 1]; }
    const float inv = pf_row_inv(ssq, t, nch, D);
    *(float2 *)(rows + (size_t)t * N + c) = make_float2(s[0] * inv, s[1] * inv);
}

// attention output as the (hi, lo) pair of bf16 numbers the output projection takes
__global__ __launch_bounds__(256) void k_rq_pair(const float *__restrict__ x, uint16_t *__restrict__ hi, uint16_t *__restrict__ lo, int n) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) pf_split(x[i], hi[i], lo[i]);
}

// positions [0, len) of a layer's contiguous cache (rows of `row_bytes`, a multiple of 16) into a sequence's pages
__global__ __launch_bounds__(256) void k_rq_admit(const uint4 *__restrict__ from, uint4 *__restrict__ pool, const int *__restrict__ table,
                                                  int page_shift, int row_pieces, int len) {
    const int s = blockIdx.x;
    if (s >= len) return;
    const size_t row = ((size_t)table[s >> page_shift] << page_shift) + (s & ((1 << page_shift) - 1));
    for (int i = threadIdx.x; i < row_pieces; i += 256) pool[row * row_pieces + i] = from[(size_t)s * row_pieces + i];
}
