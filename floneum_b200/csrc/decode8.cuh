// Decode over the 8-bit paged KV cache: one query token per sequence, GQA.
//   s_j = scale 2^ke_j sum_d q_d kc_jd,   out = sum_j exp(s_j - m) 2^ve_j vc_j / sum_j exp(s_j - m)
// HBM-bound: D + 1 bytes per cached row, each read once and shared by the g query heads of its kv head.
//
// A warp takes pages of 16 tokens, copies them by cp.async into slots of its own two pages ahead, and works on them with warp-level
// MMAs whose rows are tokens (S^T = K Q^T) and dims (O^T = V^T P^T), so the eight columns are the query heads and none of
// the 16 rows is padding.  Against f32 arithmetic on the values nothing is given up that the result would show:
//  * scores are 8-bit MMAs on the codes as they lie: q, times a power of two per head, is a whole number of 22 to 23 bits, three digits
//    of base 256, whose products with the codes are summed exactly; a score is scaled by its row's step in f32;
//  * the weight of a value row is exp(s) 2^ve in one exponential, against a running reference of its own, so that rows whose steps
//    lie far apart weigh in f16 as they do in the result: a factor of 2^6 and two terms, 22 bits down to 2^-31 of the reference.
//    The value codes become f16 by setting the exponent of 1024 over the byte and subtracting: exact;
//  * the tensor core cuts f32 sums off towards zero: each page's products go to accumulators of their own, which are then added to the
//    running output in f32.
// The references (of the sum and of the output) follow the maxima lazily: a page whose scores exceed them by less than 2^8 leaves them.
#pragma once
#include <cfloat>

#include "attn_mma16.cuh"
#include "cache8.cuh"

namespace fusor {

constexpr int D8_NW = 8;      // warps of a CTA
constexpr int D8_SLOTS = 3;   // pages of a warp: one in use, two on their way
constexpr int D8_CTAS = 2;    // CTAs per SM
constexpr int D8_THREADS = D8_NW * 32;
constexpr float D8_SHIFT = 6.0f;  // log2 of the factor the weights of value rows carry: with a page 2^8 above its reference 2^14

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
    float* part_o;     // records as in DecodeParams
    float* part_ml;
    int* err;
    DecodeOutput res;
};

template <int D>
struct Decode8Smem {
    static constexpr int TILE = DEC_PT * D;      // bytes of a page's K or V codes
    static constexpr int SLOT = 2 * TILE;
    static constexpr int WARP = D8_SLOTS * SLOT;
    static constexpr int SCALES = D8_NW * WARP;  // offset of [warp][slot][32]
    static constexpr int META = SCALES + D8_NW * D8_SLOTS * 32;  // [warp][DEC_GP] float4, see Decode8State::store
    static constexpr int bytes = META + D8_NW * DEC_GP * 16;
    static_assert(SLOT >= DEC_GP * D * 4, "a warp's output fits the slot it has just used");
};

__device__ __forceinline__ void cp_async16(uint32_t smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// c (16x8, f32) = a (16x16, f16, row) * b (16x8, f16, col)
__device__ __forceinline__ void mma_f16_fresh(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// c (16x8, s32) += a (16x32, s8, row) * b (32x8, s8, col)
__device__ __forceinline__ void mma_s8_16832(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Bytes 0 and 2 (of w >> 8: 1 and 3) of four int8 as two f16: the byte with its sign bit flipped over the exponent of 1024.
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
    const uint32_t x = (w & 0x00ff00ffu) ^ 0x64806480u;
    const uint32_t bias = 0x64806480u;  // 1024 + 128
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&y);
}

// Where a warp stands in a stream of pages: pages [0, n) of the stream are the pages of (b, hk) from 0 (the first: any) on, then
// those of the next (b, hk) and so on.
struct Decode8Walk {
    int b, hk;
    int np;   // pages of sequence b
    int off;  // stream index of page 0 of (b, hk); negative in the first when the stream begins behind it
    // to the (b, hk) that stream index i, inside the stream, belongs to
    __device__ __forceinline__ void seek(const Decode8Params& P, int i) {
        while (i >= off + np) {
            off += np;
            if (++hk < P.Hkv) continue;
            hk = 0;
            do {
                ++b;
                np = (__ldg(P.end + b) + DEC_PT - 1) / DEC_PT;
            } while (np == 0);
        }
    }
};

// The pages of the stream a warp is about to copy, their table entries read two pages ahead of the copy.
struct Decode8Feed {
    Decode8Walk w;
    int i, n, step;  // next stream index to look up, length of the stream, every which page of it
    int page[2], hk[2];  // hk < 0: none
    __device__ __forceinline__ void look(const Decode8Params& P, int k) {
        hk[k] = -1;
        if (i < n) {
            w.seek(P, i);
            hk[k] = w.hk;
            page[k] = __ldg(P.page_table + (long long)w.b * P.max_pages + (i - w.off));  // first used by its copy
            i += step;
        }
    }
    __device__ __forceinline__ void init(const Decode8Params& P, const Decode8Walk& start, int first, int length, int every) {
        w = start;
        i = first;
        n = length;
        step = every;
        page[0] = page[1] = 0;
        look(P, 0);
        look(P, 1);
    }
};

// Rows of 128 bytes: chunk c of row r lies at c ^ (r & 7); of 64: at c ^ (r / 2 & 3).  ldmatrix then meets no bank conflict.
template <int D>
__device__ __forceinline__ int d8_swizzle(int row) { return D == 128 ? row & 7 : (row >> 1) & 3; }

// The next page of the feed into a slot, as a group of its own (an empty one when there is none).
template <int D>
__device__ __forceinline__ void d8_copy(const Decode8Params& P, Decode8Feed& F, uint32_t slot, uint32_t scale_slot, int lane) {
    constexpr int CH = D / 16;  // 16-byte chunks of a row
    if (F.hk[0] >= 0) {
        int page = F.page[0];
        if ((unsigned)page >= (unsigned)P.num_pages) {  // record and read page 0 instead
            if (lane == 0) atomicExch(P.err, kErrBadPage);
            page = 0;
        }
        const long long tile = (long long)page * P.Hkv + F.hk[0];
        const int8_t* k = P.k_codes + tile * (DEC_PT * D) + lane * 16;
        const int8_t* v = P.v_codes + tile * (DEC_PT * D) + lane * 16;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const int row = lane / CH + j * (32 / CH);
            const uint32_t dst = slot + row * D + ((lane % CH) ^ d8_swizzle<D>(row)) * 16;
            cp_async16(dst, k + j * 512);
            cp_async16(dst + DEC_PT * D, v + j * 512);
        }
        if (lane < 2) cp_async16(scale_slot + lane * 16, P.scales + tile * 32 + lane * 16);
    }
    cp_async_commit();
    F.page[0] = F.page[1];
    F.hk[0] = F.hk[1];
    F.look(P, 1);
}

// A warp's state over one (sequence, kv head).  A lane holds columns (query heads) 2 (lane % 4) and the next.
template <int D>
struct Decode8State {
    uint32_t q[3][D / 32][2];  // B fragments of Q^T, column lane / 4: the digits of the query, base 256, largest first
    float qs[2];               // what turns a sum of digits times codes into a score in log2 units, but for the row's step
    float top[2];              // largest score so far
    float m[2], mv[2];         // references of the sum and of the output
    float l[2];
    float o[D / 16][4];        // [dims 16 c + 2 (lane / 4), next][columns]: (d, col), (d, col + 1), (d + 1, col), (d + 1, col + 1)

    __device__ __forceinline__ void load_q(const Decode8Params& P, int b, int hk, int lane) {
        const int h = lane >> 2, t = lane & 3;
        float x[D / 16][4];
        uint32_t big = 0;
        const long long at = b * P.q_sb + (long long)(hk * P.g + h) * P.q_sh + 4 * t;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            if (P.q_dtype == 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[c][e] = h < P.g ? __ldg(static_cast<const float*>(P.q) + at + 16 * c + e) : 0.0f;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const uint32_t u = h < P.g ? __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(P.q) + at + 16 * c + e)) : 0;
                    const float2 f = P.q_dtype == 1 ? make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u))
                                                    : __half22float2(*reinterpret_cast<const __half2*>(&u));
                    x[c][e] = f.x;
                    x[c][e + 1] = f.y;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) big = max(big, abs_bits(x[c][e]));
        }
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // 2^up q is at most 126 * 2^16 (up at most 100: the factor back stays a normal number)
        const int up = min(16 + 133 - (int)((big + 0x20000u) >> 23), 100);
        const float factor = __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            uint32_t u[4];  // with 128 added to each digit they are the bytes; flipping the top bit takes it off again
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = (uint32_t)(__float2int_rn(x[c][e] * factor) + 0x808080);
            const uint32_t lo01 = __byte_perm(u[0], u[1], 0x5140), lo23 = __byte_perm(u[2], u[3], 0x5140);
            q[2][c >> 1][c & 1] = __byte_perm(lo01, lo23, 0x5410) ^ 0x80808080u;
            q[1][c >> 1][c & 1] = __byte_perm(lo01, lo23, 0x7632) ^ 0x80808080u;
            q[0][c >> 1][c & 1] = __byte_perm(__byte_perm(u[0], u[1], 0x0062), __byte_perm(u[2], u[3], 0x0062), 0x5410) ^ 0x80808080u;
        }
        // a query that is not finite: NaN in every place of its head's result
        const float back = h >= P.g ? 0.0f : big >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : P.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
        qs[0] = __shfl_sync(0xffffffffu, back, 8 * t);
        qs[1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            top[j] = -INFINITY;
            m[j] = mv[j] = -FLT_MAX;  // (finite: -inf - m is -inf)
            l[j] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < D / 16; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.0f;
    }

    // One page in shared memory, tokens tok0 .. tok0 + 15 of which 0 .. len - 1 exist.  Whole warp.
    __device__ __forceinline__ void page(uint32_t slot, uint32_t scale_slot, int tok0, int len, int lane) {
        constexpr int TILE = DEC_PT * D;
        const int row = lane & 15, gl = lane >> 2;
        const uint32_t kb = slot + row * D, sw = d8_swizzle<D>(row), half = lane >> 4;
        // ---- the page's scales, one per lane: steps of K, exponents of V
        uint32_t byte;
        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(byte) : "r"(scale_slot + lane) : "memory");
        // ---- S^T = K Q^T: rows gl and gl + 8 (tokens), this lane's two columns
        int acc[3][4] = {};
#pragma unroll
        for (int c = 0; c < D / 16; c += 2) {
            uint32_t a[4];
            ldmatrix_x4(a, kb + (((c + half) ^ sw) << 4));
#pragma unroll
            for (int k = 0; k < 3; ++k) mma_s8_16832(acc[k], a, q[k][c >> 1][0], q[k][c >> 1][1]);
        }
        const float scale = byte == kRowNaN ? __uint_as_float(0x7fc00000u) : lane < DEC_PT ? __uint_as_float(byte << 23) : (float)((int)byte - 127);
        float s[4], sv[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float step = __shfl_sync(0xffffffffu, scale, gl + 8 * i), ve = __shfl_sync(0xffffffffu, scale, gl + 8 * i + DEC_PT);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int e = 2 * i + j;
                s[e] = fmaf((float)acc[0][e], 65536.0f, (float)(acc[1][e] * 256 + acc[2][e])) * (step * qs[j]);
                sv[e] = s[e] + ve;
            }
        }
        if (tok0 < 0 || tok0 + DEC_PT > len) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if ((unsigned)(tok0 + gl + 8 * i) >= (unsigned)len) s[2 * i] = s[2 * i + 1] = sv[2 * i] = sv[2 * i + 1] = -INFINITY;
        }
        // ---- references
        constexpr float LAZY = 8.0f;
        float d[4], dv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            d[e] = s[e] - m[e & 1];
            dv[e] = sv[e] - mv[e & 1];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) top[j] = fmax3(top[j], s[j], s[2 + j]);
        if (__any_sync(0xffffffffu, fmax3(fmax3(d[0], d[1], d[2]), fmax3(d[3], dv[0], dv[1]), fmaxf(dv[2], dv[3])) > LAZY)) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float hi = fmaxf(s[j], s[2 + j]), hiv = fmaxf(sv[j], sv[2 + j]);
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, x));
                    hiv = fmaxf(hiv, __shfl_xor_sync(0xffffffffu, hiv, x));
                }
                hi = fmaxf(m[j], hi);
                hiv = fmaxf(mv[j], hiv);
                l[j] *= fast_exp2(m[j] - hi);
                const float a = fast_exp2(mv[j] - hiv);
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    o[c][j] *= a;
                    o[c][2 + j] *= a;
                }
                m[j] = hi;
                mv[j] = hiv;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                d[e] = s[e] - m[e & 1];
                dv[e] = sv[e] - mv[e & 1];
            }
        }
        // ---- weights: of the sum, and of the value rows' codes
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            l[e & 1] += fast_exp2(d[e]);
            w[e] = fast_exp2(dv[e] + D8_SHIFT);
        }
        const uint32_t h0 = movmatrix_trans(split_pair<true>(w[0], w[1])), h1 = movmatrix_trans(split_pair<true>(w[2], w[3]));
        const uint32_t l0 = movmatrix_trans(split_pair<true>(w[0], w[1])), l1 = movmatrix_trans(split_pair<true>(w[2], w[3]));
        // ---- O^T += V^T P^T
#pragma unroll
        for (int c = 0; c < D / 16; c += 2) {
            uint32_t v[4];
            ldmatrix_x4_trans(v, kb + TILE + (((c + half) ^ sw) << 4));
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t a[4] = {codes_f16(v[2 * u]), codes_f16(v[2 * u] >> 8), codes_f16(v[2 * u + 1]), codes_f16(v[2 * u + 1] >> 8)};
                float x[4];
                mma_f16_fresh(x, a, l0, l1);
                mma_16816<true>(x, a, h0, h1);
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float2 y = fadd2(make_float2(o[c + u][e], o[c + u][e + 1]), make_float2(x[e], x[e + 1]));
                    o[c + u][e] = y.x;
                    o[c + u][e + 1] = y.y;
                }
            }
        }
    }

    // Sums over the lanes that share a column; m becomes the largest score.
    __device__ __forceinline__ void reduce() {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                l[j] += __shfl_xor_sync(0xffffffffu, l[j], x);
                top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], x));
            }
            if (top[j] != -INFINITY) l[j] *= fast_exp2(m[j] - top[j]);
            if (l[j] != l[j]) top[j] = 0.0f;  // a NaN that no merge may leave out
            m[j] = top[j];
        }
    }

    // The reduced state to shared memory: O [DEC_GP][D] and per column {largest score, sum, reference of the output, -}.
    __device__ __forceinline__ void store(float* out, float4* meta, int lane) const {
        const int gl = lane >> 2, t = lane & 3;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (gl == 0) meta[2 * t + j] = make_float4(m[j], l[j], mv[j] - D8_SHIFT, 0.0f);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) *reinterpret_cast<float2*>(out + (2 * t + j) * D + 16 * c + 2 * gl) = make_float2(o[c][j], o[c][2 + j]);
        }
    }

    // The reduced state as the result of (b, hk), as decode_emit writes it, or as record `rec`.
    __device__ __forceinline__ void emit(const Decode8Params& P, int b, int hk, bool whole, long long rec, int lane) const {
        const int gl = lane >> 2, t = lane & 3;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int rr = 2 * t + j, h = hk * P.g + rr;
            if (rr >= P.g) continue;
            float a = fast_exp2(mv[j] - D8_SHIFT - m[j]);
            if (l[j] == 0.0f) a = 0.0f;
            if (!whole) {
                float* po = P.part_o + (rec * DEC_GP + rr) * D + 2 * gl;
#pragma unroll
                for (int c = 0; c < D / 16; ++c) *reinterpret_cast<float2*>(po + 16 * c) = make_float2(a * o[c][j], a * o[c][2 + j]);
                if (gl == 0) *reinterpret_cast<float2*>(P.part_ml + (rec * DEC_GP + rr) * 2) = make_float2(m[j], l[j]);
            } else if (P.res.mode == 0) {
                if (l[j] > 0.0f) a /= l[j];
                const long long at = (long long)b * P.res.o_sb + (long long)h * P.res.o_sh + 2 * gl;
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    if (P.res.out_dtype == 0)
                        *reinterpret_cast<float2*>(static_cast<float*>(P.res.out) + at + 16 * c) = make_float2(a * o[c][j], a * o[c][2 + j]);
                    else
                        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(P.res.out) + at + 16 * c) = pack_16(P.res.out_dtype, a * o[c][j], a * o[c][2 + j]);
                }
            } else {
                float* r = static_cast<float*>(P.res.out) + ((long long)b * P.res.Hq + h) * (D + 2);
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    r[2 + 16 * c + 2 * gl] = a * o[c][j];
                    r[3 + 16 * c + 2 * gl] = a * o[c][2 + j];
                }
                if (gl == 0) {
                    r[0] = m[j] * 0.6931471805599453f;
                    r[1] = l[j];
                }
            }
        }
    }
};

// The warps' states merged, for query head rr of the group and dims 4 dg .. 4 dg + 3.  out(w): a warp's O.
template <int D, class Out>
__device__ __forceinline__ void d8_merge(const float4* meta, Out out, int rr, int dg, float& M, float& L, float4& acc) {
    M = -INFINITY;
    L = 0.0f;
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < D8_NW; ++w) M = fmaxf(M, meta[w * DEC_GP + rr].x);
#pragma unroll
    for (int w = 0; w < D8_NW; ++w) {
        const float4 x = meta[w * DEC_GP + rr];
        if (x.y == 0.0f) continue;  // no page
        const float a = fast_exp2(x.z - M);
        const float4 o = *reinterpret_cast<const float4*>(out(w) + rr * D + dg * 4);
        acc.x += a * o.x; acc.y += a * o.y; acc.z += a * o.z; acc.w += a * o.w;
        L += x.y * fast_exp2(x.x - M);
    }
}

// The pages of all (sequence, kv head) pairs, numbered as in decode_splitkv_kernel, are dealt evenly to `shares` warps, each a run of
// its own: warps meet nobody on the way, copies run on over the ends of sequences, and what a warp has of a (sequence, kv head) goes
// from its registers to the result, when it is all of it, or to a record for decode_combine_kernel (to which a share is what
// a CTA is there).  Only the warps of a CTA that lies inside one (sequence, kv head) merge their states first and write one record, the
// first warp's, so that a long sequence has a record per CTA.
template <int D>
__global__ void __launch_bounds__(D8_THREADS, D8_CTAS) decode8_splitkv_kernel(const __grid_constant__ Decode8Params P, const int shares) {
    using Smem = Decode8Smem<D>;
    extern __shared__ __align__(128) uint8_t d8_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cta0 = (int)blockIdx.x * D8_NW, share = cta0 + warp;
    // T pages in all
    int sum = 0;
    for (int b0 = 0; b0 < P.B; b0 += 32) sum += __reduce_add_sync(0xffffffffu, b0 + lane < P.B ? (P.end[b0 + lane] + DEC_PT - 1) / DEC_PT : 0);
    const int T = sum * P.Hkv;
    const auto bound = [&](int c) { return (int)((long long)min(c, shares) * T / shares); };
    const int cta_first = bound(cta0), cta_end = bound(cta0 + D8_NW);
    const int first = min(bound(share), cta_end - 1), n = bound(share + 1) - bound(share);  // (a share has a page at least; warps past the last: n = 0)
    // the sequence that holds the warp's first page, and the pages (per kv head) before it
    Decode8Walk w;
    for (int b0 = 0, cum = 0;; b0 += 32) {
        const int pages = b0 + lane < P.B ? (P.end[b0 + lane] + DEC_PT - 1) / DEC_PT : 0;
        int upto = pages;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, x);
            if (lane >= x) upto += y;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, (cum + upto) * P.Hkv > first);
        if (hit) {
            const int at = __ffs(hit) - 1;
            w.b = b0 + at;
            w.np = __shfl_sync(0xffffffffu, pages, at);
            const int rel = first - (cum + __shfl_sync(0xffffffffu, upto, at) - w.np) * P.Hkv;
            w.hk = rel / w.np;
            w.off = w.hk * w.np - rel;
            break;
        }
        cum += __shfl_sync(0xffffffffu, upto, 31);
    }
    const bool together = cta_first >= first + w.off && cta_end <= first + w.off + w.np && shares - cta0 > 1;
    if (n == 0 && !together) return;
    const uint32_t ring = smem_u32(d8_smem) + warp * Smem::WARP, scales = smem_u32(d8_smem) + Smem::SCALES + warp * D8_SLOTS * 32;
    Decode8Feed feed;
    feed.init(P, w, 0, n, 1);
    d8_copy<D>(P, feed, ring, scales, lane);
    d8_copy<D>(P, feed, ring + Smem::SLOT, scales + 32, lane);

    Decode8State<D> st;
    int i = 0, slot = 0, free_slot = 2;  // the next page, its slot, and the one that holds nothing that is still needed
    do {
        if (n > 0) w.seek(P, i);
        const int seg_end = min(n, w.off + w.np);
        const int front = __ldg(P.front + w.b), len = __ldg(P.end + w.b) - front;
        st.load_q(P, w.b, w.hk, lane);
        for (; i < seg_end; ++i) {
            cp_async_wait<1>();
            __syncwarp();  // the page is there, and every lane is done with the slot before it
            d8_copy<D>(P, feed, ring + free_slot * Smem::SLOT, scales + free_slot * 32, lane);
            st.page(ring + slot * Smem::SLOT, scales + slot * 32, (i - w.off) * DEC_PT - front, len, lane);
            free_slot = slot;
            slot = slot == D8_SLOTS - 1 ? 0 : slot + 1;
        }
        st.reduce();
        if (!together)
            st.emit(P, w.b, w.hk, w.off >= 0 && w.off + w.np <= n && P.res.mode != 2, (long long)w.b * P.Hkv + w.hk + share, lane);
    } while (i < n);
    if (!together) return;

    cp_async_wait<0>();
    __syncwarp();
    float4* meta = reinterpret_cast<float4*>(d8_smem + Smem::META);
    const auto out = [&](int k) { return reinterpret_cast<float*>(d8_smem + k * Smem::WARP); };  // nothing is on its way any more
    st.store(out(warp), meta + warp * DEC_GP, lane);
    __syncthreads();
    const long long rec = (long long)w.b * P.Hkv + w.hk + cta0;
    for (int item = tid; item < P.g * (D / 4); item += D8_THREADS) {
        const int rr = item / (D / 4), dg = item % (D / 4);
        float M, L;
        float4 acc;
        d8_merge<D>(meta, out, rr, dg, M, L, acc);
        *reinterpret_cast<float4*>(P.part_o + (rec * DEC_GP + rr) * D + dg * 4) = acc;
        if (dg == 0) {
            *reinterpret_cast<float2*>(P.part_ml + (rec * DEC_GP + rr) * 2) = make_float2(M, L);
            for (int k = 1; k < D8_NW && cta0 + k < shares; ++k)  // the other warps' records: empty
                *reinterpret_cast<float2*>(P.part_ml + ((rec + k) * DEC_GP + rr) * 2) = make_float2(-INFINITY, 0.0f);
        }
    }
}

// One block per (query head, sequence), whose records may be hundreds, most of them empty: the weights of all records first, in two
// rounds of loads whatever their number, then the sums, a run of records per warp and no load of an empty one.  A head whose pages all went to one warp has been written by that warp.
constexpr int D8_MERGE = 256;  // threads
template <int D>
__global__ void __launch_bounds__(D8_MERGE) decode8_combine_kernel(const __grid_constant__ CombineParams P) {
    extern __shared__ __align__(16) float d8_weight[];  // [records], then [warps][D]
    __shared__ int red[66];
    __shared__ float part[2][D8_MERGE / 32];
    const int h = blockIdx.x, b = blockIdx.y, hk = h / P.g, rr = h % P.g, tid = threadIdx.x, warp = tid >> 5;
    int first, n;
    decode_head_records(P.end, P.B, P.Hkv, P.grid, b, hk, red, first, n);
    if (n == 1) return;
    float2 ml[4];  // this thread's records, where four a thread are enough; else they are read again
    float M = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int s = tid + k * D8_MERGE;
        ml[k] = s < n ? *reinterpret_cast<const float2*>(P.part_ml + ((long long)(first + s) * DEC_GP + rr) * 2) : make_float2(-INFINITY, 0.0f);
        M = fmaxf(M, ml[k].x);
    }
    for (int s = tid + 4 * D8_MERGE; s < n; s += D8_MERGE) M = fmaxf(M, P.part_ml[((long long)(first + s) * DEC_GP + rr) * 2]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    if ((tid & 31) == 0) part[0][warp] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < D8_MERGE / 32; ++w) M = fmaxf(M, part[0][w]);
    float L = 0.0f;
    const auto weigh = [&](int s, float2 x) {
        const float a = x.y == 0.0f ? 0.0f : fast_exp2(x.x - M);
        d8_weight[s] = a;
        if (x.y != 0.0f) L += a * x.y;
    };
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (tid + k * D8_MERGE < n) weigh(tid + k * D8_MERGE, ml[k]);
    for (int s = tid + 4 * D8_MERGE; s < n; s += D8_MERGE) weigh(s, *reinterpret_cast<const float2*>(P.part_ml + ((long long)(first + s) * DEC_GP + rr) * 2));
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
    if ((tid & 31) == 0) part[1][warp] = L;
    __syncthreads();
    L = 0.0f;
#pragma unroll
    for (int w = 0; w < D8_MERGE / 32; ++w) L += part[1][w];
    // a run of records per warp, the loads of four that are not empty at a time
    constexpr int NW = D8_MERGE / 32, E = D / 32;
    const int lane = tid & 31, end = (int)((long long)n * (warp + 1) / NW);
    float acc[E] = {};
    const float* po = P.part_o + ((long long)first * DEC_GP + rr) * D + lane * E;
    for (int s0 = (int)((long long)n * warp / NW); s0 < end; s0 += 32) {
        unsigned some = __ballot_sync(0xffffffffu, s0 + lane < end && d8_weight[s0 + lane] != 0.0f);
        while (some) {
            float a[4], o[4][E];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int s = s0 + __ffs(some) - 1;
                a[k] = some ? d8_weight[s] : 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) o[k][e] = some ? po[(long long)s * (DEC_GP * D) + e] : 0.0f;
                some &= some - 1;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += a[k] * o[k][e];
        }
    }
    float* sum = d8_weight + (n + 3) / 4 * 4;  // [warp][D]
#pragma unroll
    for (int e = 0; e < E; ++e) sum[warp * D + lane * E + e] = acc[e];
    __syncthreads();
    if (tid >= D / 4) return;
    float4 all = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float4 o = *reinterpret_cast<const float4*>(sum + w * D + tid * 4);
        all.x += o.x; all.y += o.y; all.z += o.z; all.w += o.w;
    }
    decode_emit(P.res, D, P.g, b, hk, rr, tid, M, L, all);
}

// Few pages: a cluster of C CTAs per (sequence, kv head), as decode_cluster_kernel: one launch, the CTAs' states meet in shared
// memory over the cluster.
template <int D>
struct Decode8ClusterSmem {
    static constexpr int SLOT_F4 = DEC_GP * D / 4 + DCL_MAX;  // column groups pushed here by all CTAs (rounded up per source)
    static constexpr int PUSH = Decode8Smem<D>::bytes;
    static constexpr int bytes = PUSH + SLOT_F4 * 16 + DCL_MAX * DEC_GP * 8;
};

template <int D>
__global__ void __launch_bounds__(D8_THREADS, D8_CTAS) decode8_cluster_kernel(const __grid_constant__ Decode8Params P, const int C) {
    using Smem = Decode8Smem<D>;
    constexpr int DG = D / 4;
    extern __shared__ __align__(128) uint8_t d8_smem[];
    float4* meta = reinterpret_cast<float4*>(d8_smem + Smem::META);
    float4* push = reinterpret_cast<float4*>(d8_smem + Decode8ClusterSmem<D>::PUSH);       // [source CTA][column group of this CTA]
    float2* push_ml = reinterpret_cast<float2*>(push + Decode8ClusterSmem<D>::SLOT_F4);    // [source CTA][GP]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = C > 1 ? (int)cluster_cta_rank() : 0;
    const int head = (int)blockIdx.x / C, b = head / P.Hkv, hk = head % P.Hkv;
    const int end = __ldg(P.end + b), front = __ldg(P.front + b), pages = (end + DEC_PT - 1) / DEC_PT;
    const int p_begin = (int)((long long)pages * rank / C), n = (int)((long long)pages * (rank + 1) / C) - p_begin;
    if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for before the first push

    const uint32_t ring = smem_u32(d8_smem) + warp * Smem::WARP, scales = smem_u32(d8_smem) + Smem::SCALES + warp * D8_SLOTS * 32;
    const Decode8Walk start{b, hk, pages, -p_begin};
    Decode8Feed feed;
    feed.init(P, start, warp, n, D8_NW);
    d8_copy<D>(P, feed, ring, scales, lane);
    d8_copy<D>(P, feed, ring + Smem::SLOT, scales + 32, lane);
    Decode8State<D> st;
    st.load_q(P, b, hk, lane);
    int slot = 0, free_slot = 2;
    for (int i = warp; i < n; i += D8_NW) {
        cp_async_wait<1>();
        __syncwarp();  // the page is there, and every lane is done with the slot before it
        d8_copy<D>(P, feed, ring + free_slot * Smem::SLOT, scales + free_slot * 32, lane);
        st.page(ring + slot * Smem::SLOT, scales + slot * 32, (p_begin + i) * DEC_PT - front, end - front, lane);
        free_slot = slot;
        slot = slot == D8_SLOTS - 1 ? 0 : slot + 1;
    }
    cp_async_wait<0>();
    __syncwarp();
    auto out = [&](int w) { return reinterpret_cast<float*>(d8_smem + w * Smem::WARP); };  // nothing is on its way any more
    st.reduce();
    st.store(out(warp), meta + warp * DEC_GP, lane);
    __syncthreads();
    if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA of the cluster has started
    const int items = P.g * DG, per = (items + C - 1) / C;  // CTA k finishes column groups [k per, (k + 1) per)
    for (int item = tid; item < items; item += D8_THREADS) {
        const int rr = item / DG, dg = item % DG;
        float M, L;
        float4 acc;
        d8_merge<D>(meta, out, rr, dg, M, L, acc);
        if (C == 1) {
            decode_emit(P.res, D, P.g, b, hk, rr, dg, M, L, acc);
        } else {
            const int to = item / per;
            st_cluster_f4(map_to_cta(push + rank * per + (item - to * per), (uint32_t)to), acc);
            if (dg < C) st_cluster_f2(map_to_cta(push_ml + rank * DEC_GP + rr, (uint32_t)dg), make_float2(M, L));
        }
    }
    if (C == 1) return;
    __syncwarp();
    cluster_sync();  // everything pushed here has arrived
    for (int item = rank * per + tid; item < min(items, (rank + 1) * per); item += D8_THREADS) {
        const int rr = item / DG, dg = item % DG;
        float M = -INFINITY, L = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < C; ++k) M = fmaxf(M, push_ml[k * DEC_GP + rr].x);
        for (int k = 0; k < C; ++k) {
            const float2 ml = push_ml[k * DEC_GP + rr];
            if (ml.y == 0.0f) continue;  // no page
            const float a = fast_exp2(ml.x - M);
            const float4 o = push[k * per + item - rank * per];
            acc.x += a * o.x; acc.y += a * o.y; acc.z += a * o.z; acc.w += a * o.w;
            L += a * ml.y;
        }
        decode_emit(P.res, D, P.g, b, hk, rr, dg, M, L, acc);
    }
}

}  // namespace fusor
