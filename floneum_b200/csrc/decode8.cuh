// Decode over the 8-bit paged KV cache: one query token per sequence, GQA.
//   s_j = scale 2^ke_j sum_d q_d kc_jd,   out = sum_j exp(s_j - m) 2^ve_j vc_j / sum_j exp(s_j - m)
// HBM-bound: D + 1 bytes per cached row, each read once and shared by the g query heads of its kv head.
//
// A warp takes pages of 16 tokens, copies them by cp.async into slots of its own two pages ahead, and works on them with warp-level
// MMAs whose rows are tokens (S^T = K Q^T) and dims (O^T = V^T P^T), so the eight columns are the query heads and none of
// the 16 rows is padding.  Against f32 arithmetic on the values nothing is given up that the result would show:
//  * scores are 8-bit MMAs on the codes as they lie: q, times a power of two per head, is a whole number of 22 to 23 bits, three digits
//    of base 256, whose products with the codes are summed exactly; a score is scaled by its row's step in f32.  f32 queries have three
//    digits more for what is left, 45 bits together; of 16-bit ones an element below 2^-14 (f16: 2^-11) of its head's largest is off by up to
//    2^-23 of that;
//  * the weight of a value row is exp(s) 2^ve in one exponential, against a running reference of its own, so that rows whose steps
//    lie far apart weigh in f16 as they do in the result: a factor of 2^6 and two terms, off by 2^-22 of the weight or, from 2^-9 of the
//    reference on down, by 2^-31 of the reference.  The value codes become f16 by setting the exponent of 1024 over the byte and
//    subtracting: exact;
//  * the tensor core cuts f32 sums off towards zero: each page's products go to accumulators of their own, which are then added to the
//    running output in f32.
// The references (of the sum and of the output) follow the maxima lazily: a page whose scores exceed them by less than 2^8 leaves them.
// Error of an f32 result against 64 bits: 2.4e-7 to 3.5e-7 (2-norm), that of f32 arithmetic in torch 4.5e-7 to 1.1e-6.
//
// B64 kv 1024-8192 H32/8 D128, 610 MB: 109 to 112 us in graphs = 5.5 TB/s, with f32 queries 119 to 121; the bf16 cache's kernels take 193 us for
// these sequences.  Time stamps (without the overlap with the launch before): dealt 1.5 us, first copies 4, first page used 6.5; pages
// done on average at 90, the last at 100; the last CTA ends at 108.  610 MB in those 84 us are 7.2 TB/s: HBM is the bound in between, and
// the ends are latencies and the spread of the warps, which a deal at run time would even out at the price of results that depend on it.
// 401 warp instructions a page with all ends (ALU 44 % busy, the tensor pipe 32 %).  16-bit MMAs on converted keys took 519 a page and
// 130 us, 8-bit ones before each warp had a run of pages 135, with it and a second launch for the merge 118.
#pragma once
#include <cfloat>

#include "attn_mma16.cuh"
#include "cache8.cuh"

namespace fusor {

constexpr int D8_NW = 16;     // warps of a CTA (most)
constexpr int D8_SLOTS = 3;   // pages of a warp: one in use, two on their way
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
    int* done;         // [B * Hkv] pages whose records are written, zero between launches
    int* err;
    DecodeOutput res;
};

// LEVELS: of the query's digits, 2 for f32 queries, 1 for 16-bit ones.  At D = 128 those take 24 registers more: fewer warps, with 168 each
// instead of 128.
template <int D, int LEVELS>
constexpr int d8_warps = LEVELS > 1 && D == 128 ? 12 : D8_NW;

template <int D, int NW = D8_NW>
struct Decode8Smem {
    static constexpr int TILE = DEC_PT * D;      // bytes of a page's K or V codes
    static constexpr int SLOT = 2 * TILE + 128;  // K, V, 32 scales and padding: rows of K and V start on multiples of 64 or 128
    static constexpr int WARP = D8_SLOTS * SLOT;
    static constexpr int META = NW * WARP;    // [warp][DEC_GP] float4, see Decode8State::store
    static constexpr int WEIGHTS = META + NW * DEC_GP * 16;  // the same: {of O, of the sum, largest score of the group, -}
    static constexpr int bytes = WEIGHTS + NW * DEC_GP * 16;
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

// A place in the pages of all (sequence, kv head) pairs, numbered in (b, hk, page) order and counted from where a warp's run begins.
struct Decode8Walk {
    int b, hk;
    int np;   // pages of sequence b
    int off;  // place of page 0 of (b, hk); negative when the run begins behind it
    __device__ __forceinline__ void next(const Decode8Params& P) {  // the next pair that has pages (there is one)
        off += np;
        if (++hk < P.Hkv) return;
        hk = 0;
        do {
            ++b;
            np = (P.end[b] + DEC_PT - 1) / DEC_PT;
        } while (np == 0);
    }
};

// The pages a warp is about to copy: every `step`-th of its run, their table entries read two pages ahead of the copy.
struct Decode8Feed {
    Decode8Walk w;
    int i, n, step, seg_end;  // next page to look up, length of the run, where (b, hk) or the run ends
    const int* entry;         // its place in the page table
    int page[2], hk[2];       // hk < 0: none
    __device__ __forceinline__ void seek(const Decode8Params& P) {
        seg_end = min(n, w.off + w.np);
        entry = P.page_table + (long long)w.b * P.max_pages + (i - w.off);
    }
    __device__ __forceinline__ void look(const Decode8Params& P, int k) {
        hk[k] = -1;
        if (i >= seg_end) {
            if (i >= n) return;
            w.next(P);
            seek(P);
        }
        hk[k] = w.hk;
        page[k] = *entry;  // first used by its copy
        entry += step;
        i += step;
    }
    __device__ __forceinline__ void init(const Decode8Params& P, const Decode8Walk& start, int first, int length, int every) {
        w = start;
        i = first;
        n = length;
        step = every;
        page[0] = page[1] = 0;
        seek(P);
        look(P, 0);
        look(P, 1);
    }
};

// Rows of 128 bytes: chunk c of row r lies at c ^ (r & 7); of 64: at c ^ (r / 2 & 3).  ldmatrix then meets no bank conflict.
template <int D>
__device__ __forceinline__ int d8_swizzle(int row) { return D == 128 ? row & 7 : (row >> 1) & 3; }

// Where a lane reads fragments of a tile (of chunks 0 and 1; chunk pair c is the place ^ 16 c) and writes its chunks (the first; the next
// is 512 bytes on, its chunk the first's ^ 4 for rows of 128 bytes, the same for rows of 64).
template <int D>
__device__ __forceinline__ uint32_t d8_frag(int lane) { return (lane & 15) * D + (((lane >> 4) ^ d8_swizzle<D>(lane & 15)) << 4); }
template <int D>
__device__ __forceinline__ uint32_t d8_place(int lane) {
    constexpr int CH = D / 16;  // 16-byte chunks of a row
    return lane / CH * D + (((lane % CH) ^ d8_swizzle<D>(lane / CH)) << 4);
}

// The next page of the feed into a slot, as a group of its own (an empty one when there is none).  place: slot + d8_place.
template <int D>
__device__ __forceinline__ void d8_copy(const Decode8Params& P, Decode8Feed& F, uint32_t place, uint32_t scale_slot, int lane) {
    constexpr int TILE = DEC_PT * D;
    if (F.hk[0] >= 0) {
        int page = F.page[0];
        if ((unsigned)page >= (unsigned)P.num_pages) {  // record and read page 0 instead
            if (lane == 0) atomicExch(P.err, kErrBadPage);
            page = 0;
        }
        const uint32_t tile = (uint32_t)page * (uint32_t)P.Hkv + (uint32_t)F.hk[0];  // (the pool has fewer than 2^31 rows of 16)
        const unsigned long long at = (unsigned long long)tile * TILE + lane * 16;
        const int8_t *k = P.k_codes + at, *v = P.v_codes + at;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const uint32_t dst = (D == 128 && (j & 1) ? place ^ 64 : place) + j * 512;
            cp_async16(dst, k + j * 512);
            cp_async16(dst + TILE, v + j * 512);
        }
        if (lane < 2) cp_async16(scale_slot + lane * 16, P.scales + (unsigned long long)tile * 32 + lane * 16);
    }
    cp_async_commit();
    F.page[0] = F.page[1];
    F.hk[0] = F.hk[1];
    F.look(P, 1);
}

// The query heads of a (sequence, kv head) as digits, [digit][head][ROW] words of four dims, then what turns a sum of digits times codes
// into a score in log2 units, but for the row's step, per head.  (Padded rows: the fragments' reads meet no bank conflict.)
template <int D>
struct Decode8Digits {
    static constexpr int ROW = D / 4 + 4, WORDS = 3 * DEC_GP * ROW + DEC_GP;
    static_assert(WORDS * 4 <= Decode8Smem<D>::SLOT, "they fit a slot");
};

// The query's lines to L2 while the memory is idle: its loads come behind those of the first pages.
template <int D>
__device__ __forceinline__ void d8_prefetch_q(const Decode8Params& P, int b, int hk, int lane) {
    const int h = lane >> 2, size = P.q_dtype == 0 ? 4 : 2, at = (lane & 3) * 128;
    if (h >= P.g || at >= D * size) return;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(P.q) + (b * P.q_sb + (long long)(hk * P.g + h) * P.q_sh) * size + at));
}

// Query heads first, first + step, .. of the group into `digits`, a warp; D = 64: two at a time.  Heads past the last: factor 0, and
// whatever lies there as digits (whole numbers, so their scores are zeros).  LOW: the three digits behind those, of what is left of an
// element without them, times 2^23.  f32 arithmetic keeps 24 bits of every element however far apart they lie.  With 22 bits of the largest
// alone, one element r times the others, where the keys are zero, puts the result off by 1.1e-6 for r = 30 and 3.6e-5 for r = 1000; with both
// levels by 6e-12 at most up to r = 30000 and by 1.5e-9 for 10^6.
template <int D, bool LOW = false>
__device__ __forceinline__ void d8_digits(const Decode8Params& P, int b, int hk, int first, int step, uint32_t* digits, int lane) {
    constexpr int PER = 128 / D, ROW = Decode8Digits<D>::ROW;  // heads at a time
    const int word = lane % (D / 4), sub = lane / (D / 4);
    const unsigned mates = D == 128 ? 0xffffffffu : 0xffffu << (16 * sub);
    if (first == 0 && lane >= P.g && lane < DEC_GP) digits[3 * DEC_GP * ROW + lane] = 0u;
    for (int h0 = first * PER; h0 < P.g; h0 += 2 * step * PER) {
        uint32_t raw[2][4] = {};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int h = h0 + u * step * PER + sub;
            if (h >= P.g) continue;
            const long long at = b * P.q_sb + (long long)(hk * P.g + h) * P.q_sh + 4 * word;
            if (P.q_dtype == 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) raw[u][e] = static_cast<const uint32_t*>(P.q)[at + e];
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) raw[u][e] = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(P.q) + at)[e];
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int h = h0 + u * step * PER + sub;
            if (h0 + u * step * PER >= P.g) break;
            float x[4];
            if (P.q_dtype == 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(raw[u][e]);
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float2 f = P.q_dtype == 1 ? make_float2(__uint_as_float(raw[u][e] << 16), __uint_as_float(raw[u][e] & 0xffff0000u))
                                                    : __half22float2(*reinterpret_cast<const __half2*>(&raw[u][e]));
                    x[2 * e] = f.x;
                    x[2 * e + 1] = f.y;
                }
            }
            const uint32_t big = __reduce_max_sync(mates, max(max(abs_bits(x[0]), abs_bits(x[1])), max(abs_bits(x[2]), abs_bits(x[3]))));
            // 2^up q is below 127 * 2^16 (up at most 100: the factor back stays a normal number)
            const int up = min(16 + 133 - (int)((big + 0x20000u) >> 23), 100);
            const float factor = __uint_as_float((uint32_t)(127 + up) << 23);
            uint32_t n[4];  // with 128 added to each digit they are the bytes; flipping the top bit takes it off again
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float y = x[e] * factor;
                const int whole = __float2int_rn(y);  // (below 2^23: y - whole is exact, at most a half)
                n[e] = (uint32_t)((LOW ? __float2int_rn((y - (float)whole) * 0x1p23f) : whole) + 0x808080);
            }
            const uint32_t lo01 = __byte_perm(n[0], n[1], 0x5140), lo23 = __byte_perm(n[2], n[3], 0x5140);
            const uint32_t hi = __byte_perm(__byte_perm(n[0], n[1], 0x0062), __byte_perm(n[2], n[3], 0x0062), 0x5410);
            uint32_t* out = digits + h * ROW + word;
            out[0] = hi ^ 0x80808080u;
            out[DEC_GP * ROW] = __byte_perm(lo01, lo23, 0x7632) ^ 0x80808080u;
            out[2 * DEC_GP * ROW] = __byte_perm(lo01, lo23, 0x5410) ^ 0x80808080u;
            // a query that is not finite: NaN in every place of its head's result
            const float back = big >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : P.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
            if (word == 0 && h < P.g) digits[3 * DEC_GP * ROW + h] = __float_as_uint(back);
        }
    }
}

// A warp's state over one (sequence, kv head).  A lane holds columns (query heads) 2 (lane % 4) and the next.
template <int D, int LEVELS>
struct Decode8State {
    uint32_t q[3 * LEVELS][D / 32][2];  // B fragments of Q^T, column lane / 4: the digits of the query, base 256, largest first
    float qs[2];               // what turns a sum of digits times codes into a score in log2 units, but for the row's step
    float top[2];              // largest score so far
    float m[2], mv[2];         // references of the sum and of the output
    float l[2];
    float o[D / 16][4];        // [dims 16 c + 2 (lane / 4), next][columns]: (d, col), (d, col + 1), (d + 1, col), (d + 1, col + 1)

    // A level of digits from what d8_digits has left in shared memory.
    __device__ __forceinline__ void load(const uint32_t* digits, int level, int lane) {
        constexpr int ROW = Decode8Digits<D>::ROW;
#pragma unroll
        for (int k = 0; k < 3; ++k)
#pragma unroll
            for (int c = 0; c < D / 16; ++c) q[3 * level + k][c >> 1][c & 1] = digits[(k * DEC_GP + (lane >> 2)) * ROW + 4 * c + (lane & 3)];
    }

    // The first level with its factors, and the state before the first page.
    __device__ __forceinline__ void start(const uint32_t* digits, int lane) {
        constexpr int ROW = Decode8Digits<D>::ROW;
        const int t = lane & 3;
        load(digits, 0, lane);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            qs[j] = __uint_as_float(digits[3 * DEC_GP * ROW + 2 * t + j]);
            top[j] = -INFINITY;
            m[j] = mv[j] = -FLT_MAX;  // (finite: -inf - m is -inf)
            l[j] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < D / 16; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.0f;
    }

    // A level's digits times the codes, tokens gl and gl + 8 and this lane's columns: whole numbers, rounded to f32.
    __device__ __forceinline__ void products(float (&x)[4], uint32_t frag, int level) const {
        int acc[3][4] = {};
#pragma unroll
        for (int c = 0; c < D / 16; c += 2) {
            uint32_t a[4];
            ldmatrix_x4(a, frag ^ (c << 4));
#pragma unroll
            for (int k = 0; k < 3; ++k) mma_s8_16832(acc[k], a, q[3 * level + k][c >> 1][0], q[3 * level + k][c >> 1][1]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fmaf((float)acc[0][e], 65536.0f, (float)(acc[1][e] * 256 + acc[2][e]));
    }

    // One page in shared memory, tokens tok0 .. tok0 + 15 of which 0 .. len - 1 exist.  Whole warp.
    // frag: slot + d8_frag.
    __device__ __forceinline__ void page(uint32_t frag, uint32_t scale_slot, int tok0, int len, int lane) {
        constexpr int TILE = DEC_PT * D;
        const int gl = lane >> 2;
        // ---- the page's scales, one per lane: steps of K, exponents of V
        uint32_t byte;
        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(byte) : "r"(scale_slot + lane) : "memory");
        // ---- S^T = K Q^T: rows gl and gl + 8 (tokens), this lane's two columns
        float x[4];
        products(x, frag, 0);
        if (LEVELS > 1) {  // (both in one loop, with six accumulators: 121 against 120 us, D = 64 77 against 74.5)
            float y[4];
            products(y, frag, LEVELS - 1);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = fmaf(y[e], 0x1p-23f, x[e]);
        }
        const float scale = byte == kRowNaN ? __uint_as_float(0x7fc00000u) : lane < DEC_PT ? __uint_as_float(byte << 23) : (float)((int)byte - 127);
        float s[4], sv[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float step = __shfl_sync(0xffffffffu, scale, gl + 8 * i), ve = __shfl_sync(0xffffffffu, scale, gl + 8 * i + DEC_PT);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int e = 2 * i + j;
                s[e] = x[e] * (step * qs[j]);
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
            ldmatrix_x4_trans(v, (frag ^ (c << 4)) + TILE);
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

    // The reduced state to shared memory, over the warp's slots: O [DEC_GP][D] and per column {largest score, sum, reference of the output, -}.
    __device__ __forceinline__ void store(uint8_t* smem, int warp, int lane) const {
        const int gl = lane >> 2, t = lane & 3;
        float* out = reinterpret_cast<float*>(smem + warp * Decode8Smem<D>::WARP);
        float4* meta = reinterpret_cast<float4*>(smem + Decode8Smem<D, d8_warps<D, LEVELS>>::META) + warp * DEC_GP;
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

// T pages dealt to `shares` as [c T / shares, (c + 1) T / shares): decode_walk_init's and decode_page_owner's numbers without 64-bit
// divisions (a few hundred cycles each, at both ends of a kernel of some microseconds).
struct Decode8Deal {
    int T, shares, each, rest;
    __device__ __forceinline__ Decode8Deal(int pages, int n) : T(pages), shares(n), each(pages / n), rest(pages % n) {}
    __device__ __forceinline__ int bound(int c) const {  // first page of share c; rest < shares < 2^12
        c = min(c, shares);
        return c * each + (int)((unsigned)(c * rest) / (unsigned)shares);
    }
    __device__ __forceinline__ int owner(int page) const {  // floor(((page + 1) shares - 1) / T): an estimate, off by one at most
        const long long x = (long long)(page + 1) * shares - 1;
        int q = (int)((float)(page + 1) * (float)shares / (float)T);
        long long r = x - (long long)q * T;
        while (r < 0) { --q; r += T; }
        while (r >= T) { ++q; r -= T; }
        return q;
    }
};

// A warp's slots: pages come in turn, two ahead of the one in use.
template <int D>
struct Decode8Ring {
    static constexpr uint32_t SLOT = Decode8Smem<D>::SLOT, LAST = (D8_SLOTS - 1) * SLOT;
    uint32_t base, frag, place;  // of slot 0
    uint32_t now, spare;         // offsets of the slot of the next page, and of the one that holds nothing that is still needed
    __device__ __forceinline__ Decode8Ring(const void* smem, int warp, int lane)
        : base(smem_u32(smem) + warp * Decode8Smem<D>::WARP), frag(base + d8_frag<D>(lane)), place(base + d8_place<D>(lane)), now(0), spare(LAST) {}
    __device__ __forceinline__ void fill(const Decode8Params& P, Decode8Feed& feed, int lane) {
#pragma unroll
        for (uint32_t at = 0; at < LAST; at += SLOT) d8_copy<D>(P, feed, place + at, base + at + 2 * DEC_PT * D, lane);
    }
    template <int LEVELS>
    __device__ __forceinline__ void page(const Decode8Params& P, Decode8Feed& feed, Decode8State<D, LEVELS>& st, int tok0, int len, int lane) {
        cp_async_wait<D8_SLOTS - 2>();
        __syncwarp();  // the page is there, and every lane is done with the slot before it
        d8_copy<D>(P, feed, place + spare, base + spare + 2 * DEC_PT * D, lane);
        st.page(frag + now, base + now + 2 * DEC_PT * D, tok0, len, lane);
        spare = now;
        now = now == LAST ? 0 : now + SLOT;
    }
};

// The CTA's merge of its warps' states (Decode8State::store has put them at smem + w * WARP and to meta).  ends_with[w]: which warps belong
// together, neighbours; < 0: none.  First every (warp, head) its weight next to its group's largest score, then the sums, where nothing
// waits for anything.  done(w0, group size, rr, dg, M, L, acc) gets the group's first warp and the sums of dims 4 dg .. 4 dg + 3.
template <int D, int NW, class Done>
__device__ __forceinline__ void d8_merge_warps(uint8_t* smem, const int* ends_with, int g, Done done) {
    float4* meta = reinterpret_cast<float4*>(smem + Decode8Smem<D, NW>::META);
    float4* weights = reinterpret_cast<float4*>(smem + Decode8Smem<D, NW>::WEIGHTS);
    const int tid = threadIdx.x, lane = tid & 31;
    __syncthreads();
    const int pair = lane < NW ? ends_with[lane] : -1, before = __shfl_up_sync(0xffffffffu, pair, 1);
    const unsigned joins = __ballot_sync(0xffffffffu, lane > 0 && pair >= 0 && pair == before);  // warps that go with the one before
    const unsigned leads = __ballot_sync(0xffffffffu, pair >= 0) & ~joins;
    const auto size_of = [&](int w0) { return __ffs(~(joins >> (w0 + 1))); };
    if (tid < NW * DEC_GP) {
        const int w = tid / DEC_GP, rr = tid % DEC_GP;
        const unsigned upto = leads & ((2u << w) - 1);  // the last of them is this warp's group's, if it has one
        const int w0 = 31 - __clz(upto | 1);
        if (rr < g && upto && w < w0 + size_of(w0)) {
            const float4 mine = meta[w * DEC_GP + rr];
            float M = -INFINITY;
            for (int k = w0; k < w0 + size_of(w0); ++k) M = fmaxf(M, meta[k * DEC_GP + rr].x);
            const bool none = mine.y == 0.0f;  // no page
            weights[w * DEC_GP + rr] = make_float4(none ? 0.0f : fast_exp2(mine.z - M), none ? 0.0f : mine.y * fast_exp2(mine.x - M), M, 0.0f);
        }
    }
    __syncthreads();
    const int items = __popc(leads) * g * (D / 4);
    for (int item = tid; item < items; item += NW * 32) {
        const int dg = item % (D / 4), row = item / (D / 4), rr = row % g;
        unsigned from = leads;
        for (int k = row / g; k > 0; --k) from &= from - 1;
        const int w0 = __ffs(from) - 1, size = size_of(w0);
        const uint8_t* state = smem + w0 * Decode8Smem<D>::WARP + (rr * D + dg * 4) * 4;
        const float4* weight = weights + w0 * DEC_GP + rr;
        const float M = weight->z;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float L = 0.0f;
        for (int k = 0; k < size; k += 4) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int at = min(k + u, size - 1);
                const float2 x = k + u < size ? *reinterpret_cast<const float2*>(weight + at * DEC_GP) : make_float2(0.0f, 0.0f);
                const float4 o = *reinterpret_cast<const float4*>(state + at * Decode8Smem<D>::WARP);
                L += x.y;
                acc.x += x.x * o.x; acc.y += x.x * o.y; acc.z += x.x * o.z; acc.w += x.x * o.w;
            }
        }
        done(w0, size, rr, dg, M, L, acc);
    }
}

// The records of a (sequence, kv head) whose pages are [page0, page0 + np) of T, when more than one share has pages of it: one for each
// CTA in which it is what shares end with, in the slot of the first of them, and one of the share that it ends inside of, if any.
template <int NW>
struct Decode8Records {
    int c_first, c_last;  // its shares
    int cta, groups, n;   // CTA of the first share; CTAs with a record of their shares; records
    Decode8Records() = default;
    __device__ __forceinline__ Decode8Records(const Decode8Deal& deal, int page0, int np) {
        c_first = deal.owner(page0);
        c_last = deal.owner(page0 + np - 1);
        const int inside = deal.bound(c_last + 1) > page0 + np;
        cta = c_first / NW;
        groups = (c_last - inside) / NW - cta + 1;
        n = groups + inside;
    }
    __device__ __forceinline__ int share(int i) const { return i == 0 ? c_first : i < groups ? (cta + i) * NW : c_last; }
};

// One query head's records merged to its result, by a warp; other CTAs have written them, so nothing of them is read from L1.  The loads
// of eight records do not wait for their weights.
template <int D, int NW>
__device__ __forceinline__ void d8_merge_records(const Decode8Params& P, const Decode8Records<NW>& R, int pair, int rr, int lane) {
    constexpr int E = D / 32, BATCH = 8;
    const int b = pair / P.Hkv, hk = pair % P.Hkv;
    float M = -INFINITY, L = 0.0f, acc[E] = {};
    for (int i0 = 0; i0 < R.n; i0 += BATCH) {
        const int here = min(BATCH, R.n - i0);
        const long long row = (long long)(pair + R.share(i0 + min(lane, here - 1))) * DEC_GP + rr;
        const float2 x = lane < here ? __ldcg(reinterpret_cast<const float2*>(P.part_ml) + row) : make_float2(-INFINITY, 0.0f);
        float o[BATCH][E];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const float* from = P.part_o + __shfl_sync(0xffffffffu, row, k) * D + lane * E;  // (past the last record: the last one's)
            if (k < here) {
                if (E == 4) {
                    const float4 y = __ldcg(reinterpret_cast<const float4*>(from));
                    o[k][0] = y.x; o[k][1] = y.y; o[k][E - 2] = y.z; o[k][E - 1] = y.w;
                } else {
                    const float2 y = __ldcg(reinterpret_cast<const float2*>(from));
                    o[k][0] = y.x; o[k][1] = y.y;
                }
            }
        }
        float top = x.x;
#pragma unroll
        for (int z = 16; z > 0; z >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, z));
        top = fmaxf(M, top);
        const float weight = x.y == 0.0f ? 0.0f : fast_exp2(x.x - top), before = M == -INFINITY ? 0.0f : fast_exp2(M - top);
        M = top;
        L = L * before + (x.y == 0.0f ? 0.0f : weight * x.y);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= before;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            // (a weight that is zero next to the largest score keeps a record's NaN; only a record without keys counts for nothing)
            const float a = __shfl_sync(0xffffffffu, weight, k), sum = __shfl_sync(0xffffffffu, x.y, k);
            if (k < here && sum != 0.0f) {
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += a * o[k][e];
            }
        }
    }
#pragma unroll
    for (int z = 16; z > 0; z >>= 1) L += __shfl_xor_sync(0xffffffffu, L, z);
    if (E == 4) {
        decode_emit(P.res, D, P.g, b, hk, rr, lane, M, L, make_float4(acc[0], acc[1], acc[E - 2], acc[E - 1]));
    } else {
        const float z = __shfl_down_sync(0xffffffffu, acc[0], 1), w = __shfl_down_sync(0xffffffffu, acc[1], 1);
        if (!(lane & 1)) decode_emit(P.res, D, P.g, b, hk, rr, lane >> 1, M, L, make_float4(acc[0], acc[1], z, w));
    }
}

// The pages of all (sequence, kv head) pairs, numbered as in decode_splitkv_kernel, are dealt evenly to `shares` warps, each a run of
// its own: warps meet nobody on the way, copies run on over the ends of sequences, and a pair that a warp has all pages of goes from
// its registers to the result.  What a warp ends with is merged with the warps of the CTA that end with the same pair, to one
// record, or to the result when the CTA has all of it.  Of the pairs that it shares with other CTAs it adds the pages it had to a counter,
// and merges the records of those that are complete with it: no second launch, and no order of arrival in a result.
template <int D, int LEVELS>
__global__ void __launch_bounds__(d8_warps<D, LEVELS> * 32, 1) decode8_splitkv_kernel(const __grid_constant__ Decode8Params P, const int shares) {
    constexpr int NW = d8_warps<D, LEVELS>;
    using Smem = Decode8Smem<D, NW>;
    extern __shared__ __align__(128) uint8_t d8_smem[];
    __shared__ int ends_with[NW];     // the pair that a warp's last pages belong to, -1 when there is nothing to merge
    __shared__ int4 parts[2 * NW];    // what a warp begins and ends with, when it has not all of it: {pair, first page of it, pages here, pages}
    __shared__ struct { int pair; Decode8Records<NW> records; } complete[2 * NW];
    __shared__ int n_complete;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cta0 = (int)blockIdx.x * NW, share = cta0 + warp;
    after_previous_launch();
    // T pages in all
    int sum = 0;
    for (int b0 = 0; b0 < P.B; b0 += 32) sum += __reduce_add_sync(0xffffffffu, b0 + lane < P.B ? (P.end[b0 + lane] + DEC_PT - 1) / DEC_PT : 0);
    const int T = sum * P.Hkv;
    // `shares` is from the launch.  A captured one may meet shorter sequences: as many shares as pages then, since Decode8Records looks for
    // a record in the first share of a CTA.  (In mode 2 the merge goes by the launch's number; shares with no page write empty records.)
    const bool merged_later = P.res.mode == 2;
    const Decode8Deal deal(T, merged_later ? shares : max(1, min(shares, T)));
    const int first = deal.bound(share), n = deal.bound(share + 1) - first;  // (a share has a page at least; warps past the last: none)
    // the sequence that holds the warp's first page, and the pages (per kv head) before it
    Decode8Walk w{};
    const bool nothing = merged_later && n == 0 && share < shares && first < T;
    for (int b0 = 0, cum = 0; n > 0 || nothing; b0 += 32) {
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
    if (nothing && lane < P.g)
        *reinterpret_cast<float2*>(P.part_ml + ((long long)(w.b * P.Hkv + w.hk + share) * DEC_GP + lane) * 2) = make_float2(-INFINITY, 0.0f);
    Decode8Ring<D> ring(d8_smem, warp, lane);
    Decode8Feed feed;
    feed.init(P, w, 0, n, 1);
    if (n > 0) d8_prefetch_q<D>(P, w.b, w.hk, lane);
    ring.fill(P, feed, lane);

    if (P.res.mode != 2)  // sequences without pages (mode 0: in a replay only): empty records, zeros
        for (int row = (int)blockIdx.x * NW * 32 + tid; row < P.B * P.res.Hq; row += gridDim.x * NW * 32)
            if (P.end[row / P.res.Hq] == 0) {
                const int b = row / P.res.Hq, h = row % P.res.Hq;
                for (int dg = 0; dg < D / 4; ++dg)
                    decode_emit(P.res, D, P.g, b, h / P.g, h % P.g, dg, -INFINITY, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
            }
    if (tid == 0) n_complete = 0;
    if (lane < 2) parts[2 * warp + lane] = make_int4(0, 0, 0, 0);
    Decode8State<D, LEVELS> st;
    int open = -1;
    for (int i = 0; i < n; w.next(P)) {
        const int seg_end = min(n, w.off + w.np);
        const int front = P.front[w.b], len = P.end[w.b] - front;
        uint32_t* digits = reinterpret_cast<uint32_t*>(d8_smem + warp * Smem::WARP + ring.spare);
        __syncwarp();  // every lane is done with the slot
        d8_digits<D>(P, w.b, w.hk, 0, 1, digits, lane);
        __syncwarp();
        st.start(digits, lane);
        if (LEVELS > 1) {
            __syncwarp();
            d8_digits<D, true>(P, w.b, w.hk, 0, 1, digits, lane);
            __syncwarp();
            st.load(digits, LEVELS - 1, lane);
        }
        for (int tok0 = (i - w.off) * DEC_PT - front; i < seg_end; ++i, tok0 += DEC_PT) ring.page(P, feed, st, tok0, len, lane);
        st.reduce();
        const int pair = w.b * P.Hkv + w.hk;
        const bool whole = w.off >= 0 && w.off + w.np <= n && P.res.mode != 2;
        if (!whole && lane == 0) parts[2 * warp + (i >= n)] = make_int4(pair, first + w.off, seg_end - max(0, w.off), w.np);
        if (whole || i < n) {
            st.emit(P, w.b, w.hk, whole, (long long)pair + share, lane);
        } else {
            cp_async_wait<0>();
            __syncwarp();  // nothing is on its way to the slots any more
            st.store(d8_smem, warp, lane);
            open = pair;
        }
        if (i >= n) break;
    }
    if (lane == 0) ends_with[warp] = open;
    const int cta_first = deal.bound(cta0), cta_end = deal.bound(cta0 + NW);
    const auto inside = [&](int4 part) { return part.y >= cta_first && part.y + part.w <= cta_end && P.res.mode != 2; };  // all its pages are this CTA's
    d8_merge_warps<D, NW>(d8_smem, ends_with, P.g, [&](int w0, int size, int rr, int dg, float M, float L, float4 acc) {
        const int pair = ends_with[w0];
        const long long rec = ((long long)pair + cta0 + w0) * DEC_GP + rr;
        if (inside(parts[2 * w0 + 1])) {
            if (w0 + size < NW && parts[2 * (w0 + size)].z > 0 && parts[2 * (w0 + size)].x == pair) {  // and the record of the warp that it ends inside of
                const float2 ml = *reinterpret_cast<const float2*>(P.part_ml + (rec + size * DEC_GP) * 2);
                const float4 o = *reinterpret_cast<const float4*>(P.part_o + (rec + size * DEC_GP) * D + dg * 4);
                const float top = fmaxf(M, ml.x), a0 = L == 0.0f ? 0.0f : fast_exp2(M - top), a1 = ml.y == 0.0f ? 0.0f : fast_exp2(ml.x - top);
                acc.x = acc.x * a0 + o.x * a1; acc.y = acc.y * a0 + o.y * a1; acc.z = acc.z * a0 + o.z * a1; acc.w = acc.w * a0 + o.w * a1;
                L = L * a0 + ml.y * a1;
                M = top;
            }
            decode_emit(P.res, D, P.g, pair / P.Hkv, pair % P.Hkv, rr, dg, M, L, acc);
            return;
        }
        *reinterpret_cast<float4*>(P.part_o + rec * D + dg * 4) = acc;
        if (dg == 0) {
            *reinterpret_cast<float2*>(P.part_ml + rec * 2) = make_float2(M, L);
            if (P.res.mode == 2)  // its merge looks at a record of every share
                for (int k = 1; k < size; ++k) *reinterpret_cast<float2*>(P.part_ml + (rec + k * DEC_GP) * 2) = make_float2(-INFINITY, 0.0f);
        }
    });
    if (P.res.mode == 2) return;

    // ---- the pairs that are complete with this CTA's pages
    __threadfence();
    __syncthreads();  // this CTA's records can be seen everywhere
    if (tid < 2 * NW && parts[tid].z > 0 && !inside(parts[tid])) {
        const int4 part = parts[tid];
        const int pair = part.x, before = atomicAdd(P.done + pair, part.z);
        const Decode8Records<NW> R(deal, part.y, part.w);
        if (before + part.z == part.w) {
            P.done[pair] = 0;
            complete[atomicAdd(&n_complete, 1)] = {pair, R};
        }
    }
    __threadfence();
    __syncthreads();
    for (int item = warp; item < n_complete * P.g; item += NW)
        d8_merge_records<D, NW>(P, complete[item / P.g].records, complete[item / P.g].pair, item % P.g, lane);
}

// Few pages: a cluster of C CTAs per (sequence, kv head), as decode_cluster_kernel: one launch, the CTAs' states meet in shared
// memory over the cluster.  Bound by latencies: of 6.6 us for 1411 tokens (H32/8 D128, medians of time stamps, without the overlap with the launch before) 1.4 go to the
// lengths, 0.5 to the page table, 0.6 to the query's digits, 1.4 to the pages, 1.4 to the CTA's merge, 1.2 to the cluster's.  Back to back in
// graphs 7.5 to 7.6, where the bf16 cache takes 6.4: so few pages gain nothing from being half as long.
template <int D, int NW>
struct Decode8ClusterSmem {
    static constexpr int SLOT_F4 = DEC_GP * D / 4 + DCL_MAX;  // column groups pushed here by all CTAs (rounded up per source)
    static constexpr int PUSH = Decode8Smem<D, NW>::bytes;
    static constexpr int bytes = PUSH + SLOT_F4 * 16 + DCL_MAX * DEC_GP * 8;
};

template <int D, int LEVELS>
__global__ void __launch_bounds__(d8_warps<D, LEVELS> * 32, 1) decode8_cluster_kernel(const __grid_constant__ Decode8Params P, const int C) {
    constexpr int DG = D / 4, NW = d8_warps<D, LEVELS>;
    extern __shared__ __align__(128) uint8_t d8_smem[];
    __shared__ int ends_with[NW];
    float4* push = reinterpret_cast<float4*>(d8_smem + Decode8ClusterSmem<D, NW>::PUSH);       // [source CTA][column group of this CTA]
    float2* push_ml = reinterpret_cast<float2*>(push + Decode8ClusterSmem<D, NW>::SLOT_F4);    // [source CTA][GP]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = C > 1 ? (int)cluster_cta_rank() : 0;
    after_previous_launch();
    const int head = (int)blockIdx.x / C, b = head / P.Hkv, hk = head % P.Hkv;
    const int end = P.end[b], front = P.front[b], pages = (end + DEC_PT - 1) / DEC_PT;
    const int p_begin = (int)((long long)pages * rank / C), n = (int)((long long)pages * (rank + 1) / C) - p_begin;
    if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for before the first push

    Decode8Ring<D> ring(d8_smem, warp, lane);
    const Decode8Walk start{b, hk, pages, -p_begin};
    Decode8Feed feed;
    feed.init(P, start, warp, n, NW);
    ring.fill(P, feed, lane);
    uint32_t* digits = reinterpret_cast<uint32_t*>(d8_smem + ring.spare);  // warp 0's, of the second level warp 1's
    uint32_t* low_digits = reinterpret_cast<uint32_t*>(d8_smem + Decode8Smem<D>::WARP + ring.spare);
    constexpr int MAKERS = DEC_GP * D / 128 * LEVELS > NW ? NW / LEVELS : DEC_GP * D / 128;  // warps that make a level
    if (warp < MAKERS) d8_digits<D>(P, b, hk, warp, MAKERS, digits, lane);
    else if (LEVELS > 1 && warp < 2 * MAKERS) d8_digits<D, true>(P, b, hk, warp - MAKERS, MAKERS, low_digits, lane);
    __syncthreads();
    Decode8State<D, LEVELS> st;
    st.start(digits, lane);
    if (LEVELS > 1) st.load(low_digits, LEVELS - 1, lane);
    __syncthreads();
    for (int i = warp; i < n; i += NW) ring.page(P, feed, st, (p_begin + i) * DEC_PT - front, end - front, lane);
    cp_async_wait<0>();
    __syncwarp();  // nothing is on its way to the slots any more
    st.reduce();
    st.store(d8_smem, warp, lane);
    if (lane == 0) ends_with[warp] = 0;
    if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA of the cluster has started
    const int items = P.g * DG, per = (items + C - 1) / C;  // CTA k finishes column groups [k per, (k + 1) per)
    d8_merge_warps<D, NW>(d8_smem, ends_with, P.g, [&](int, int, int rr, int dg, float M, float L, float4 acc) {
        if (C == 1) {
            decode_emit(P.res, D, P.g, b, hk, rr, dg, M, L, acc);
        } else {
            const int item = rr * DG + dg, to = item / per;
            st_cluster_f4(map_to_cta(push + rank * per + (item - to * per), (uint32_t)to), acc);
            if (dg < C) st_cluster_f2(map_to_cta(push_ml + rank * DEC_GP + rr, (uint32_t)dg), make_float2(M, L));
        }
    });
    if (C == 1) return;
    __syncwarp();
    cluster_sync();  // everything pushed here has arrived
    for (int item = rank * per + tid; item < min(items, (rank + 1) * per); item += NW * 32) {
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

// The two kernels of a head_dim and a type of query, as the host launches them
struct Decode8Kernels {
    void (*deal)(Decode8Params, int);
    void (*cluster)(Decode8Params, int);
    int warps, deal_smem, cluster_smem;
};
template <int D, int LEVELS>
Decode8Kernels decode8_kernels_of() {
    constexpr int NW = d8_warps<D, LEVELS>;
    return {decode8_splitkv_kernel<D, LEVELS>, decode8_cluster_kernel<D, LEVELS>, NW, Decode8Smem<D, NW>::bytes, Decode8ClusterSmem<D, NW>::bytes};
}
inline Decode8Kernels decode8_kernels(int D, bool f32) {
    if (D == 128) return f32 ? decode8_kernels_of<128, 2>() : decode8_kernels_of<128, 1>();
    return f32 ? decode8_kernels_of<64, 2>() : decode8_kernels_of<64, 1>();
}

}  // namespace fusor
