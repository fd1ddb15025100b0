// The 8-bit paged KV cache: its format, the kernel that writes rows to either cache (rotated on the way if asked for), the
// dense read-back and the eviction of rows.
//
// A row is one token of one kv head, D elements x (f32 after a rotation).  Its step is a power of two, 2^e with e the smallest
// whole number, at least -126 and at most 121, for which max |x| < 127.5 * 2^e, and it is held as codes rint(x / 2^e) in -127 .. 127
// (ties to even) and one byte e + 127.  (Beyond 127.5 * 2^121, 0.8 % below the largest float, codes end at 127: 64 * 2^122 is infinite.)  x / 2^e and code * 2^e are exact, so every value the cache stands for is a bf16 number: the decode that
// reads codes and an attention over the dense bf16 read-back see the same keys and values, bit for bit, and a row that is
// read back and written again has the same codes.  Against steps of max |x| / 127 this costs up to one bit of the eight.
// The step belongs to one token: rows come one at a time, and a step shared by several tokens would have to grow, and the rows
// before it to be rounded again, when a larger one arrives.  A row with an element that is not finite stands for NaN in all
// its places (byte 255).
//   k_codes, v_codes : int8 [num_pages][Hkv][16][D],   scales : uint8 [num_pages][Hkv][2][16]  (K, V)
#pragma once
#include "decode_splitkv.cuh"
#include "rope_append.cuh"

namespace fusor {

constexpr int kRowNaN = 255;  // scale byte of a row that is not finite
constexpr int kRowTop = 121 + 127;

// Scale byte of a row from max |x|: the mantissa of 127.5 is 0x7f0000, so adding 0x10000 carries into the exponent from there on.
__device__ __forceinline__ int row8_byte(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    if (bits >= 0x7f800000u) return kRowNaN;
    return min(max(1, (int)((bits + 0x10000u) >> 23) - 6), kRowTop);
}
// 2^(127 - byte), what x is multiplied by (byte from 1 to 248: the power is a normal number)
__device__ __forceinline__ float row8_inverse(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }
// 2^(byte - 127), or NaN
__device__ __forceinline__ float row8_step(int byte) { return byte == kRowNaN ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)byte << 23); }
__device__ __forceinline__ int row8_code(float x, float inverse) { return max(-127, min(127, __float2int_rn(x * inverse))); }

// max |x| of a row's elements that keeps a NaN: the largest bit pattern of |x|
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Rows to place: q [B][Hq][n][D] -> q_out, k_new and v_new [B][Hkv][n][D] -> pages, q and k rotated on the way when there are tables.
struct PlaceParams {
    const void* q;  // with Hq = 0: none
    void* q_out;
    int q_dtype, qo_dtype;
    long long qs[3], qos[3];
    int Hq;
    const void* k_new;
    const void* v_new;
    int k_dtype, v_dtype;
    long long ks[3], vs[3];
    int pages;  // where k and v go: 0 nowhere, 1 bf16 pages, 2 8-bit pages
    void* k_pages;
    void* v_pages;
    uint8_t* scales;
    const int* page_table;
    KvLens lens;
    int max_pages, Hkv;
    const float* cos_t;  // [context][D / 2]; null: nothing is rotated
    const float* sin_t;
    int context;
    int B, n, D;
    int interleaved;
    int start_pos;              // without `pos`: table row of token 0; < 0: each sequence's length before this append
    const uint32_t* pos;        // table rows [axis][B][n], the last axis contiguous
    long long pos_axis, pos_b;  // strides
    uint8_t axis[256];          // of each pair
    int* err;
};

// Table row of pair i of token t of sequence b.  Rows outside the table are recorded and read as row 0.
__device__ __forceinline__ int place_row(const PlaceParams& P, int b, int t, int i) {
    if (!P.pos) return (P.start_pos >= 0 ? P.start_pos : P.lens.before(b) - P.lens.evicted(b)) + t;
    const uint32_t row = __ldg(P.pos + P.axis[i] * P.pos_axis + b * P.pos_b + t);
    if (row < (uint32_t)P.context) return (int)row;
    atomicExch(P.err, kErrBadPosition);
    return 0;
}

// One warp per row of q, k or v.
__global__ void __launch_bounds__(256) place_rows_kernel(const __grid_constant__ PlaceParams P) {
    if (P.pages) P.lens.publish();
    const int lane = threadIdx.x & 31, half = P.D >> 1;
    const int heads = P.Hq + (P.pages ? 2 * P.Hkv : 0);
    const long long rows = (long long)P.B * heads * P.n;
    for (long long r = (blockIdx.x * (long long)blockDim.x + threadIdx.x) >> 5; r < rows; r += ((long long)gridDim.x * blockDim.x) >> 5) {
        const int t = (int)(r % P.n);
        const int h = (int)(r / P.n % heads), b = (int)(r / P.n / heads);
        const bool is_q = h < P.Hq, is_k = !is_q && h < P.Hq + P.Hkv;
        const int hk = is_q ? h : is_k ? h - P.Hq : h - P.Hq - P.Hkv;
        const void* x = is_q ? P.q : is_k ? P.k_new : P.v_new;
        const int dtype = is_q ? P.q_dtype : is_k ? P.k_dtype : P.v_dtype;
        const long long* st = is_q ? P.qs : is_k ? P.ks : P.vs;
        const long long src = b * st[0] + hk * st[1] + t * st[2];
        const bool turn = P.cos_t && (is_q || is_k);
        auto value = [&](int d) {
            const float a = ld_as_float(x, dtype, src + d);
            if (!turn) return a;
            const int i = P.interleaved ? d >> 1 : d % half, first = P.interleaved ? !(d & 1) : d < half;
            const int partner = P.interleaved ? d ^ 1 : first ? d + half : d - half;
            const long long at = (long long)place_row(P, b, t, i) * half + i;
            const float z = ld_as_float(x, dtype, src + partner), c = __ldg(P.cos_t + at), s = __ldg(P.sin_t + at);
            float ya, yb;
            rope_pair(first ? a : z, first ? z : a, c, s, P.interleaved, ya, yb);
            return first ? ya : yb;
        };
        if (is_q) {
            const long long dst = b * P.qos[0] + hk * P.qos[1] + t * P.qos[2];
            for (int d = lane; d < P.D; d += 32) st_from_float(P.q_out, P.qo_dtype, dst + d, value(d));
            continue;
        }
        const int at = P.lens.before(b) + t;
        const long long tile = (long long)P.page_table[(long long)b * P.max_pages + at / DEC_PT] * P.Hkv + hk;
        const long long dst = (tile * DEC_PT + at % DEC_PT) * P.D;
        if (P.pages == 1) {
            for (int d = lane; d < P.D; d += 32) static_cast<__nv_bfloat16*>(is_k ? P.k_pages : P.v_pages)[dst + d] = __float2bfloat16_rn(value(d));
            continue;
        }
        uint32_t top = 0;
        for (int d = lane; d < P.D; d += 32) top = max(top, abs_bits(value(d)));
        const int byte = row8_byte(__uint_as_float(__reduce_max_sync(0xffffffffu, top)));
        for (int d = lane; d < P.D; d += 32)
            static_cast<int8_t*>(is_k ? P.k_pages : P.v_pages)[dst + d] = byte == kRowNaN ? 0 : (int8_t)row8_code(value(d), row8_inverse(byte));
        if (lane == 0) P.scales[(tile * 2 + (is_k ? 0 : 1)) * DEC_PT + at % DEC_PT] = (uint8_t)byte;
    }
}

// Dense export of 8-bit pages, as kvcache_gather_kernel: out [B][Hkv][len][D] (strided), rows past a sequence's length are zero.
struct Gather8Params {
    void* k_out;
    void* v_out;
    int k_dtype, v_dtype;
    long long ks[3], vs[3];
    const int8_t* k_codes;
    const int8_t* v_codes;
    const uint8_t* scales;
    const int* page_table;
    const int* end;    // [B]
    const int* front;  // [B]
    int max_pages, Hkv, D, len, B;
};

__global__ void __launch_bounds__(256) kvcache8_gather_kernel(const __grid_constant__ Gather8Params P) {
    const long long total = (long long)P.B * P.Hkv * P.len * P.D;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const int d = (int)(i % P.D);
        const int t = (int)((i / P.D) % P.len);
        const int hk = (int)((i / ((long long)P.D * P.len)) % P.Hkv);
        const int b = (int)(i / ((long long)P.D * P.len * P.Hkv));
        float kf = 0.0f, vf = 0.0f;
        const int at = P.front[b] + t;
        if (at < P.end[b]) {
            const long long tile = (long long)P.page_table[(long long)b * P.max_pages + at / DEC_PT] * P.Hkv + hk;
            const long long src = (tile * DEC_PT + at % DEC_PT) * P.D + d;
            kf = row8_step(P.scales[tile * 2 * DEC_PT + at % DEC_PT]) * (float)P.k_codes[src];
            vf = row8_step(P.scales[(tile * 2 + 1) * DEC_PT + at % DEC_PT]) * (float)P.v_codes[src];
        }
        st_from_float(P.k_out, P.k_dtype, b * P.ks[0] + hk * P.ks[1] + t * P.ks[2] + d, kf);
        st_from_float(P.v_out, P.v_dtype, b * P.vs[0] + hk * P.vs[1] + t * P.vs[2] + d, vf);
    }
}

// kvcache_shift_kernel for 8-bit pages: rows [drop, drop + keep) of a sequence -> staging (to_pages = 0), staging -> rows [0, keep).
// Staging: codes [K, V][Hkv][keep][D], then bytes [K, V][Hkv][keep].  One thread per 16 codes; the first of a row moves its byte.
struct Shift8Params {
    int8_t* pages[2];  // K, V
    uint8_t* scales;
    const int* row;  // the sequence's page-table row on the device
    int8_t* codes;
    uint8_t* bytes;
    int Hkv, D, keep, drop;
    int to_pages;
};

__global__ void __launch_bounds__(256) kvcache8_shift_kernel(const __grid_constant__ Shift8Params P) {
    const int vec = P.D / 16;
    const long long total = 2ll * P.Hkv * P.keep * vec;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const int c = (int)(i % vec);
        const long long dense = i / vec;
        const int t = (int)(dense % P.keep);
        const int hk = (int)(dense / P.keep % P.Hkv), which = (int)(dense / P.keep / P.Hkv);
        const int at = P.to_pages ? t : t + P.drop;
        const long long tile = (long long)P.row[at / DEC_PT] * P.Hkv + hk;
        int4* paged = reinterpret_cast<int4*>(P.pages[which] + (tile * DEC_PT + at % DEC_PT) * P.D) + c;
        int4* stage = reinterpret_cast<int4*>(P.codes + dense * P.D) + c;
        uint8_t* byte = P.scales + (tile * 2 + which) * DEC_PT + at % DEC_PT;
        if (P.to_pages) {
            *paged = *stage;
            if (c == 0) *byte = P.bytes[dense];
        } else {
            *stage = *paged;
            if (c == 0) P.bytes[dense] = *byte;
        }
    }
}

}  // namespace fusor
