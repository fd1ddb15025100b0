// Decode over the 8-bit paged KV cache: one query token per sequence, GQA.
//   s_j = scale 2^ke_j sum_d q_d kc_jd,   out = sum_j exp(s_j - m) 2^ve_j vc_j / sum_j exp(s_j - m)
// HBM-bound: D + 1 bytes per cached row, each read once and shared by the g query heads of its kv head.
//
// A warp takes pages of 16 tokens, copies them by cp.async into slots of its own two pages ahead, and works on them with warp-level
// MMAs whose rows are tokens (S^T = K Q^T) and dims (O^T = V^T P^T), so the eight columns are the query heads and none of
// the 16 rows is padding.  Codes become f16 by setting the exponent of 1024 over the byte and subtracting: exact.  Against f32
// arithmetic on the values nothing is given up that the result would show:
//  * q, times a power of two per head that brings its largest element to 2^14, is one f16 term for 16-bit queries (what lies below
//    2^-24 is 2^-38 of the largest) and two for f32 (22 bits);
//  * a score is scaled by its row's step in f32, after the sum;
//  * the weight of a value row is exp(s) 2^ve in one exponential, against a running reference of its own, so that rows whose steps
//    lie far apart weigh in f16 as they do in the result: a factor of 2^6 and two terms, 22 bits down to 2^-31 of the reference;
//  * the tensor core cuts sums off towards zero: scores are summed in two halves, each page's products in accumulators of their own,
//    added to the running output in f32.
// The references (of the sum and of the output) follow the maxima lazily: a page whose scores exceed them by less than 2^8 leaves them.
#pragma once
#include "attn_mma16.cuh"
#include "cache8.cuh"

namespace fusor {

constexpr int D8_NW = 8;      // warps of a CTA
constexpr int D8_SLOTS = 3;   // pages of a warp: one in use, two on their way
constexpr int D8_CTAS = 2;    // CTAs per SM
constexpr int D8_THREADS = D8_NW * 32;

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
// Bytes 0 and 2 (of w >> 8: 1 and 3) of four int8 as two f16: the byte with its sign bit flipped over the exponent of 1024.
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
    const uint32_t x = (w & 0x00ff00ffu) ^ 0x64806480u;
    const uint32_t bias = 0x64806480u;  // 1024 + 128
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&y);
}

// Where a warp stands in a CTA's stream of pages: pages [0, n) of the stream are the pages of (b, hk) from 0 (the first: any) on, then
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

// The pages a warp is about to copy: every D8_NW-th of the stream, their table entries read two pages ahead of the copy.
struct Decode8Feed {
    Decode8Walk w;
    int i, n;  // next stream index to look up, length of the stream
    int page[2], hk[2];  // hk < 0: none
    __device__ __forceinline__ void look(const Decode8Params& P, int k) {
        hk[k] = -1;
        if (i < n) {
            w.seek(P, i);
            hk[k] = w.hk;
            page[k] = __ldg(P.page_table + (long long)w.b * P.max_pages + (i - w.off));  // first used by its copy
            i += D8_NW;
        }
    }
    __device__ __forceinline__ void init(const Decode8Params& P, const Decode8Walk& start, int first, int length) {
        w = start;
        i = first;
        n = length;
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
template <int D, int TERMS>
struct Decode8State {
    uint32_t q[TERMS][D / 16][2];  // B fragments of Q^T, column lane / 4
    float qs[2];                   // what turns a sum of q codes into a score in log2 units, but for the row's step
    float top[2];                  // largest score so far
    float m[2], mv[2];             // references of the sum and of the output
    float l[2];
    float o[D / 16][4];            // [dims 16 c + 2 (lane / 4), next][columns]: (d, col), (d, col + 1), (d + 1, col), (d + 1, col + 1)

    __device__ __forceinline__ void load_q(const Decode8Params& P, int b, int hk, int lane) {
        const int h = lane >> 2, t = lane & 3;
        float x[D / 16][4];
        uint32_t big = 0;
        const long long at = b * P.q_sb + (long long)(hk * P.g + h) * P.q_sh + 4 * t;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            if (TERMS == 2) {
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
        // 2^14 over the exponent of the largest element (at most 2^100: the factor back stays a normal number)
        const int up = min(14 + 127 - (int)(big >> 23), 100);
        const float factor = __uint_as_float((uint32_t)(127 + up) << 23);
        const bool bad = big >= 0x7f800000u;  // not finite: the head's result is NaN
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float y0 = x[c][e] * factor, y1 = x[c][e + 2] * factor;
#pragma unroll
                for (int term = 0; term < TERMS; ++term) {
                    q[term][c][e] = split_pair<true>(y0, y1);
                    if (bad) q[term][c][e] = 0x7e007e00u;
                }
            }
        const float back = h < P.g ? P.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23) : 0.0f;
        qs[0] = __shfl_sync(0xffffffffu, back, 8 * t);
        qs[1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            top[j] = m[j] = mv[j] = -INFINITY;
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
        // ---- S^T = K Q^T: rows gl and gl + 8 (tokens), this lane's two columns
        float acc[2][4] = {}, low[4] = {};
#pragma unroll
        for (int c = 0; c < D / 16; c += 2) {
            uint32_t w[4];
            ldmatrix_x4(w, kb + (((c + half) ^ sw) << 4));
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t a[4] = {codes_f16(w[2 * u]), codes_f16(w[2 * u + 1]), codes_f16(w[2 * u] >> 8), codes_f16(w[2 * u + 1] >> 8)};
                mma_16816<true>(acc[u], a, q[0][c + u][0], q[0][c + u][1]);
                if (TERMS == 2) mma_16816<true>(low, a, q[TERMS - 1][c + u][0], q[TERMS - 1][c + u][1]);
            }
        }
        uint32_t kbyte[2], vbyte[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            asm volatile("ld.shared.u8 %0, [%1];" : "=r"(kbyte[i]) : "r"(scale_slot + gl + 8 * i));
            asm volatile("ld.shared.u8 %0, [%1];" : "=r"(vbyte[i]) : "r"(scale_slot + 16 + gl + 8 * i));
        }
        float s[4], sv[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float step = row8_step(kbyte[i]);
            const float ve = vbyte[i] == kRowNaN ? __uint_as_float(0x7fc00000u) : (float)((int)vbyte[i] - 127);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float x = acc[0][2 * i + j] + acc[1][2 * i + j];
                if (TERMS == 2) x += low[2 * i + j];
                s[2 * i + j] = x * (step * qs[j]);
                sv[2 * i + j] = s[2 * i + j] + ve;
            }
        }
        if (tok0 < 0 || tok0 + DEC_PT > len) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if ((unsigned)(tok0 + gl + 8 * i) >= (unsigned)len) s[2 * i] = s[2 * i + 1] = sv[2 * i] = sv[2 * i + 1] = -INFINITY;
        }
        // ---- references
        constexpr float LAZY = 8.0f, SHIFT = 6.0f;
        float hi[2], hiv[2];
        bool up = false;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            hi[j] = fmaxf(s[j], s[2 + j]);
            hiv[j] = fmaxf(sv[j], sv[2 + j]);
            top[j] = fmaxf(top[j], hi[j]);
            up = up || hi[j] > m[j] + LAZY || hiv[j] > mv[j] + LAZY;
        }
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    hi[j] = fmaxf(hi[j], __shfl_xor_sync(0xffffffffu, hi[j], x));
                    hiv[j] = fmaxf(hiv[j], __shfl_xor_sync(0xffffffffu, hiv[j], x));
                }
                const float m1 = fmaxf(m[j], hi[j]), mv1 = fmaxf(mv[j], hiv[j]);
                l[j] *= m1 == -INFINITY ? 1.0f : fast_exp2(m[j] - m1);
                const float a = mv1 == -INFINITY ? 1.0f : fast_exp2(mv[j] - mv1);
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    o[c][j] *= a;
                    o[c][2 + j] *= a;
                }
                m[j] = m1;
                mv[j] = mv1;
            }
        }
        // ---- weights: of the sum, and of the value rows' codes
        float w[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float sub = m[j] == -INFINITY ? 0.0f : m[j], subv = (mv[j] == -INFINITY ? 0.0f : mv[j]) - SHIFT;
            l[j] += fast_exp2(s[j] - sub) + fast_exp2(s[2 + j] - sub);
            w[j] = fast_exp2(sv[j] - subv);
            w[2 + j] = fast_exp2(sv[2 + j] - subv);
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

    // The state to shared memory: O [DEC_GP][D] and per column {largest score, sum, reference of the output, a tag}.
    __device__ __forceinline__ void store(float* out, float4* meta, int tag, int lane) {
        constexpr float SHIFT = 6.0f;
        const int gl = lane >> 2, t = lane & 3;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                l[j] += __shfl_xor_sync(0xffffffffu, l[j], x);
                top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], x));
            }
            if (top[j] != -INFINITY) l[j] *= fast_exp2(m[j] - top[j]);
            if (l[j] != l[j]) top[j] = 0.0f;  // a NaN that no merge may leave out
            if (gl == 0) meta[2 * t + j] = make_float4(top[j], l[j], mv[j] - SHIFT, __int_as_float(tag));
#pragma unroll
            for (int c = 0; c < D / 16; ++c) *reinterpret_cast<float2*>(out + (2 * t + j) * D + 16 * c + 2 * gl) = make_float2(o[c][j], o[c][2 + j]);
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
        if (x.y == 0.0f) continue;  // no page of this segment
        const float a = fast_exp2(x.z - M);
        const float4 o = *reinterpret_cast<const float4*>(out(w) + rr * D + dg * 4);
        acc.x += a * o.x; acc.y += a * o.y; acc.z += a * o.z; acc.w += a * o.w;
        L += x.y * fast_exp2(x.x - M);
    }
}

// The pages of all (sequence, kv head) pairs are dealt evenly to the CTAs as in decode_splitkv_kernel, page i of a CTA's share to warp
// i % 8.  Copies run on over the ends of segments; at an end the warps put their states into the slots they have just used and
// merge them into a record, or into the result where the CTA has all pages of the pair.
template <int D, int TERMS>
__global__ void __launch_bounds__(D8_THREADS, D8_CTAS) decode8_splitkv_kernel(const __grid_constant__ Decode8Params P) {
    using Smem = Decode8Smem<D>;
    extern __shared__ __align__(128) uint8_t d8_smem[];
    float4* meta = reinterpret_cast<float4*>(d8_smem + Smem::META);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // T pages in all; the sequence that holds this CTA's first one, and the pages (per kv head) before it
    int sum = 0;
    for (int b0 = 0; b0 < P.B; b0 += 32) sum += __reduce_add_sync(0xffffffffu, b0 + lane < P.B ? (P.end[b0 + lane] + DEC_PT - 1) / DEC_PT : 0);
    const int T = sum * P.Hkv;
    const int first = (int)((long long)blockIdx.x * T / gridDim.x), n = (int)((long long)(blockIdx.x + 1) * T / gridDim.x) - first;
    if (n == 0) return;
    Decode8Walk start;
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
            start.b = b0 + at;
            start.np = __shfl_sync(0xffffffffu, pages, at);
            const int rel = first - (cum + __shfl_sync(0xffffffffu, upto, at) - start.np) * P.Hkv;
            start.hk = rel / start.np;
            start.off = start.hk * start.np - rel;
            break;
        }
        cum += __shfl_sync(0xffffffffu, upto, 31);
    }
    const uint32_t ring = smem_u32(d8_smem) + warp * Smem::WARP, scales = smem_u32(d8_smem) + Smem::SCALES + warp * D8_SLOTS * 32;
    Decode8Feed feed;
    feed.init(P, start, warp, n);
    d8_copy<D>(P, feed, ring, scales, lane);
    d8_copy<D>(P, feed, ring + Smem::SLOT, scales + 32, lane);

    int i = warp, slot = 0, free_slot = 2;  // this warp's next page, its slot, and the one that holds nothing that is still needed
    for (int pos = 0; pos < n;) {
        start.seek(P, pos);
        const int seg_end = min(n, start.off + start.np);
        const int b = start.b, hk = start.hk;
        const int front = __ldg(P.front + b), len = __ldg(P.end + b) - front;
        Decode8State<D, TERMS> st;
        st.load_q(P, b, hk, lane);
        for (; i < seg_end; i += D8_NW) {
            cp_async_wait<1>();
            __syncwarp();  // the page is there, and every lane is done with the slot before it
            d8_copy<D>(P, feed, ring + free_slot * Smem::SLOT, scales + free_slot * 32, lane);
            st.page(ring + slot * Smem::SLOT, scales + slot * 32, (i - start.off) * DEC_PT - front, len, lane);
            free_slot = slot;
            slot = slot == D8_SLOTS - 1 ? 0 : slot + 1;
        }
        __syncwarp();
        float* mine = reinterpret_cast<float*>(d8_smem + warp * Smem::WARP + free_slot * Smem::SLOT);
        st.store(mine, meta + warp * DEC_GP, free_slot, lane);
        __syncthreads();
        const bool whole = start.off >= 0 && start.off + start.np <= n && P.res.mode != 2;
        const long long rec = (long long)(b * P.Hkv + hk) + blockIdx.x;
        for (int item = tid; item < P.g * (D / 4); item += D8_THREADS) {
            const int rr = item / (D / 4), dg = item % (D / 4);
            float M, L;
            float4 acc;
            d8_merge<D>(meta, [&](int w) {
                return reinterpret_cast<const float*>(d8_smem + w * Smem::WARP + __float_as_int(meta[w * DEC_GP].w) * Smem::SLOT);
            }, rr, dg, M, L, acc);
            if (whole) {
                decode_emit(P.res, D, P.g, b, hk, rr, dg, M, L, acc);
            } else {
                *reinterpret_cast<float4*>(P.part_o + (rec * DEC_GP + rr) * D + dg * 4) = acc;
                if (dg == 0) *reinterpret_cast<float2*>(P.part_ml + (rec * DEC_GP + rr) * 2) = make_float2(M, L);
            }
        }
        __syncthreads();  // the slots may be filled again
        pos = seg_end;
    }
}

// Few pages: a cluster of C CTAs per (sequence, kv head), as decode_cluster_kernel: one launch, the CTAs' states meet in shared
// memory over the cluster.
template <int D>
struct Decode8ClusterSmem {
    static constexpr int SLOT_F4 = DEC_GP * D / 4 + DCL_MAX;  // column groups pushed here by all CTAs (rounded up per source)
    static constexpr int PUSH = Decode8Smem<D>::bytes;
    static constexpr int bytes = PUSH + SLOT_F4 * 16 + DCL_MAX * DEC_GP * 8;
};

template <int D, int TERMS>
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
    feed.init(P, start, warp, n);
    d8_copy<D>(P, feed, ring, scales, lane);
    d8_copy<D>(P, feed, ring + Smem::SLOT, scales + 32, lane);
    Decode8State<D, TERMS> st;
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
    st.store(out(warp), meta + warp * DEC_GP, 0, lane);
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
