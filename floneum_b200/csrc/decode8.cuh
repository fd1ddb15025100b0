// Decode over the 8-bit paged KV cache: one query token per sequence, GQA.
//   s_j = scale 2^ke_j sum_d q_d kc_jd,   out = sum_j exp(s_j - m) 2^ve_j vc_j / sum_j exp(s_j - m)
#pragma once
#include "cache8.cuh"

namespace fusor {

struct Decode8Params {
    const void* q;
    int q_dtype;           // 0 f32, 1 bf16, 2 f16
    long long q_sb, q_sh;  // element strides of batch and head
    const int8_t* k_codes;
    const int8_t* v_codes;
    const uint8_t* scales;
    const int* page_table;
    int max_pages, num_pages;
    const int* end;    // [B] as in DecodeParams
    const int* front;  // [B]
    int B, Hkv, g;
    float scale_log2;
    int* err;
    DecodeOutput res;
};

// One CTA per (query head, sequence): a warp takes every fourth token, its lanes D / 32 elements each.
template <int D>
__global__ void __launch_bounds__(128) decode8_row_kernel(const __grid_constant__ Decode8Params P) {
    constexpr int E = D / 32;
    __shared__ float sh_o[4][D], sh_ml[4][2];
    const int h = blockIdx.x, b = blockIdx.y, hk = h / P.g;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int end = P.end[b];
    float q[E], o[E] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = ld_as_float(P.q, P.q_dtype, b * P.q_sb + h * P.q_sh + lane * E + e);
    for (int at = P.front[b] + warp; at < end; at += 4) {
        int page = P.page_table[(long long)b * P.max_pages + at / DEC_PT];
        if (page < 0 || page >= P.num_pages) {  // record and read page 0 instead
            atomicExch(P.err, kErrBadPage);
            page = 0;
        }
        const long long tile = (long long)page * P.Hkv + hk, row = (tile * DEC_PT + at % DEC_PT) * D + lane * E;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += q[e] * (float)P.k_codes[row + e];
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= row8_step(P.scales[tile * 2 * DEC_PT + at % DEC_PT]) * P.scale_log2;
        const float m_new = fmaxf(m, s), a = exp2f(m - m_new), p = exp2f(s - m_new);
        const float w = p * row8_step(P.scales[(tile * 2 + 1) * DEC_PT + at % DEC_PT]);
        m = m_new;
        l = l * a + p;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * (float)P.v_codes[row + e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sh_o[warp][lane * E + e] = o[e];
    if (lane == 0) {
        sh_ml[warp][0] = m;
        sh_ml[warp][1] = l;
    }
    __syncthreads();
    const int dg = threadIdx.x;
    if (dg >= D / 4) return;
    float M = fmaxf(fmaxf(sh_ml[0][0], sh_ml[1][0]), fmaxf(sh_ml[2][0], sh_ml[3][0])), L = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int w = 0; w < 4; ++w) {
        if (sh_ml[w][1] == 0.0f) continue;
        const float a = exp2f(sh_ml[w][0] - M);
        const float4 x = *reinterpret_cast<const float4*>(&sh_o[w][dg * 4]);
        acc.x += a * x.x; acc.y += a * x.y; acc.z += a * x.z; acc.w += a * x.w;
        L += a * sh_ml[w][1];
    }
    decode_emit(P.res, D, P.g, b, hk, h % P.g, dg, M, L, acc);
}

}  // namespace fusor
