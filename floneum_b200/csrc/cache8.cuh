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
#include <type_traits>

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
// Without pages k_new (where Hkv > 0) goes to a dense tensor too: k_pages, of type v_dtype and strides vs.
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
    const uint32_t row = P.pos[P.axis[i] * P.pos_axis + b * P.pos_b + t];
    if (row < (uint32_t)P.context) return (int)row;
    atomicExch(P.err, kErrBadPosition);
    return 0;
}

// ---------------------------------------------------------------------------------------------------------------
// The vector form, for D a multiple of 16, tensors of one type and 16-byte aligned rows: a thread takes 16 elements of a row, 8 pairs with
// their cos / sin values, and walks heads with them.  HBM-bound, so the loads of two query heads (or of a kv head's k and v) are issued
// together and three blocks lie on an SM: with twice the loads a thread 128 registers leave two blocks, 24.8 against 24.6 us
// (each then a launch of its own), and 26.7 without the cheaper maximum below; one warp per row took 345 us with the read-back, 52 now.  The D / 16 threads of a row are neighbours in
// a warp and find its largest element by shuffles.  B4 H8 S4096 D128 bf16, k and v 24.8 us (4.1 TB/s); with q of 32 heads rotated 64.4;
// on three axes 66.0 (graphs).
template <int T>
struct PlaceType {
    static constexpr int ES = T == 0 ? 4 : 2, U4 = ES / 2;  // bytes of an element; 16-byte vectors of 8 of them
};

// Eight elements from `base + at`, in flight until place_floats
template <int T>
__device__ __forceinline__ void place_fetch(const void* base, long long at, uint4 (&raw)[PlaceType<T>::U4]) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + at * PlaceType<T>::ES);
#pragma unroll
    for (int j = 0; j < PlaceType<T>::U4; ++j) raw[j] = ld_stream(p + j);
}
template <int T>
__device__ __forceinline__ void place_floats(const uint4 (&raw)[PlaceType<T>::U4], float (&f)[8]) {
    if (T == 0) {
        const uint4 a = raw[0], b = raw[PlaceType<T>::U4 - 1];
        f[0] = __uint_as_float(a.x); f[1] = __uint_as_float(a.y); f[2] = __uint_as_float(a.z); f[3] = __uint_as_float(a.w);
        f[4] = __uint_as_float(b.x); f[5] = __uint_as_float(b.y); f[6] = __uint_as_float(b.z); f[7] = __uint_as_float(b.w);
    } else {
        rope_unpack16<T == 2>(raw[0], f);
    }
}

// Eight values of a table, by loads that stay behind after_previous_launch() (as do all of this kernel: the launch before may have written
// positions and tables too).
__device__ __forceinline__ void place_table8(const float* t, long long at, float (&f)[8]) {
    const float4* v = reinterpret_cast<const float4*>(t + at);
    const float4 a = v[0], b = v[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// cos and sin of pairs i0 .. i0 + 7 of token t of sequence b
__device__ __forceinline__ void place_angles(const PlaceParams& P, int b, int t, int i0, float (&c)[8], float (&s)[8]) {
    const int half = P.D >> 1;
    bool one = !P.pos;  // one axis for all eight: vector loads
    if (!one) {
        const uint2 axes = *reinterpret_cast<const uint2*>(P.axis + i0);
        one = axes.x == axes.y && axes.x == (axes.x & 0xffu) * 0x01010101u;
    }
    if (one) {
        const long long at = (long long)place_row(P, b, t, i0) * half + i0;
        place_table8(P.cos_t, at, c);
        place_table8(P.sin_t, at, s);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const long long at = (long long)place_row(P, b, t, i0 + j) * half + i0 + j;
        c[j] = P.cos_t[at];
        s[j] = P.sin_t[at];
    }
}

__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 16 elements of a row, this thread's, as codes in cv (the first eight, the others) and the row's byte.  GROUP threads share the row.
// x / 2^e + 1.5 * 2^23 rounds to the code, ties to even, and has it in its low byte.
template <int GROUP>
__device__ __forceinline__ int place_codes(float (&a)[8], float (&z)[8], uint2 (&cv)[2]) {
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = fmax3_nan(most, fabsf(a[j]), fabsf(z[j]));
    uint32_t top = __float_as_uint(most);
#pragma unroll
    for (int x = 1; x < GROUP; x <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, x));
    const int byte = row8_byte(__uint_as_float(top));
    const float inverse = row8_inverse(min(byte, kRowTop));
    if (byte >= kRowTop) {  // seldom: values beyond the last step end at 127, rows that are not finite have codes of 0
        most = byte == kRowTop ? 127.0f * row8_step(kRowTop) : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            a[j] = fmaxf(fminf(a[j], most), -most);
            z[j] = fmaxf(fminf(z[j], most), -most);
        }
    }
    constexpr float MAGIC = 12582912.0f;
    const auto pack = [&](const float* x) {
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = __float_as_uint(fmaf(x[j], inverse, MAGIC));
        return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
    };
    cv[0] = make_uint2(pack(a), pack(a + 4));
    cv[1] = make_uint2(pack(z), pack(z + 4));
    return byte;
}

// PAGES: 0 q alone, 1 bf16 pages, 2 8-bit pages.  ROT: 0 none (no q), 1 halves, 2 adjacent pairs.  T: type of all tensors.  blockIdx.y:
// sequence, and a group of query heads or, from q_groups on, of kv heads.
template <int PAGES, int ROT, int T, int D>
__global__ void __launch_bounds__(256, 3) place_vec_kernel(const __grid_constant__ PlaceParams P, const unsigned q_groups, const unsigned per_thread) {
    after_previous_launch();
    if (PAGES && blockIdx.y == 0) P.lens.publish();
    constexpr int U4 = PlaceType<T>::U4, U = T == 0 ? 1 : 2;  // query heads whose loads are in flight (of k and v: one head's)
    const int d = D ? D : P.D, half = d >> 1;
    const unsigned chunks = (unsigned)d >> 4;
    const unsigned kv_groups = gridDim.y / (unsigned)P.B - q_groups;
    const unsigned b = blockIdx.y / (q_groups + kv_groups), group = blockIdx.y % (q_groups + kv_groups);
    const bool is_q = group < q_groups;
    const bool dense = is_q || PAGES == 0;  // (k beside q)
    const unsigned heads = (unsigned)(is_q ? P.Hq : P.Hkv), per = dense ? per_thread : max(1u, per_thread / 2);
    unsigned idx = blockIdx.x * blockDim.x + threadIdx.x;
    const bool live = idx < (unsigned)P.n * chunks;  // (the others stay for the shuffles)
    if (!live) idx = (unsigned)P.n * chunks - 1;
    const unsigned ch = idx % chunks, t = idx / chunks;
    const unsigned h_begin = (is_q ? group : group - q_groups) * per, h_end = live ? min(heads, h_begin + per) : 0;
    const int i0 = (int)ch * 8;
    const int offa = ROT == 1 ? i0 : 2 * i0, offz = ROT == 1 ? i0 + half : 2 * i0 + 8;
    float c[8], s[8];
    if (dense) {
        const void* x = is_q ? P.q : P.k_new;
        void* out = is_q ? P.q_out : P.k_pages;
        const long long *xs = is_q ? P.qs : P.ks, *os = is_q ? P.qos : P.vs;
        const long long src = b * xs[0] + t * xs[2], dst = b * os[0] + t * os[2];
        for (unsigned h0 = h_begin; h0 < h_end; h0 += U) {
            uint4 a[U][U4], z[U][U4];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (h0 + u < h_end) {
                    place_fetch<T>(x, src + (h0 + u) * xs[1] + offa, a[u]);
                    place_fetch<T>(x, src + (h0 + u) * xs[1] + offz, z[u]);
                }
            if (h0 == h_begin) place_angles(P, (int)b, (int)t, i0, c, s);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (h0 + u < h_end) {
                    float xa[8], xz[8];
                    place_floats<T>(a[u], xa);
                    place_floats<T>(z[u], xz);
                    rope_rotate8<ROT == 2>(xa, xz, c, s);
                    rope_store8(out, T, dst + (h0 + u) * os[1] + offa, xa);
                    rope_store8(out, T, dst + (h0 + u) * os[1] + offz, xz);
                }
        }
        return;
    }
    if (PAGES == 0) return;
    const int at = P.lens.before((int)b) + (int)t;
    const int page = P.page_table[(long long)b * P.max_pages + at / DEC_PT];
    const long long ksrc = b * P.ks[0] + t * P.ks[2], vsrc = b * P.vs[0] + t * P.vs[2];
    for (unsigned k = 0; k < per; ++k) {
        const unsigned h = h_begin + k;
        const bool here = h < h_end;
        uint4 a[U4], z[U4], va[U4], vz[U4];
        if (here) {
            place_fetch<T>(P.k_new, ksrc + h * P.ks[1] + offa, a);
            place_fetch<T>(P.k_new, ksrc + h * P.ks[1] + offz, z);
            place_fetch<T>(P.v_new, vsrc + h * P.vs[1] + 2 * i0, va);
            place_fetch<T>(P.v_new, vsrc + h * P.vs[1] + 2 * i0 + 8, vz);
        }
        if (ROT && k == 0) place_angles(P, (int)b, (int)t, i0, c, s);
        float xa[8] = {}, xz[8] = {}, ya[8] = {}, yz[8] = {};
        if (here) {
            place_floats<T>(a, xa);
            place_floats<T>(z, xz);
            place_floats<T>(va, ya);
            place_floats<T>(vz, yz);
            if (ROT) rope_rotate8<ROT == 2>(xa, xz, c, s);
        }
        const long long tile = (long long)page * P.Hkv + h, dst = (tile * DEC_PT + at % DEC_PT) * d;
        if (PAGES == 1) {
            if (here) {
                rope_store8(P.k_pages, 1, dst + offa, xa);
                rope_store8(P.k_pages, 1, dst + offz, xz);
                rope_store8(P.v_pages, 1, dst + 2 * i0, ya);
                rope_store8(P.v_pages, 1, dst + 2 * i0 + 8, yz);
            }
        } else {
            constexpr int GROUP = D ? D / 16 : 1;
            uint2 kc[2], vc[2];
            const int kb = place_codes<GROUP>(xa, xz, kc), vb = place_codes<GROUP>(ya, yz, vc);
            if (here) {
                uint8_t* kp = static_cast<uint8_t*>(P.k_pages) + dst;
                if (ROT == 1) {
                    *reinterpret_cast<uint2*>(kp + offa) = kc[0];
                    *reinterpret_cast<uint2*>(kp + offz) = kc[1];
                } else {
                    *reinterpret_cast<uint4*>(kp + 2 * i0) = make_uint4(kc[0].x, kc[0].y, kc[1].x, kc[1].y);
                }
                *reinterpret_cast<uint4*>(static_cast<uint8_t*>(P.v_pages) + dst + 2 * i0) = make_uint4(vc[0].x, vc[0].y, vc[1].x, vc[1].y);
                if (ch == 0) {
                    uint8_t* scale = P.scales + tile * 2 * DEC_PT + at % DEC_PT;
                    scale[0] = (uint8_t)kb;
                    scale[DEC_PT] = (uint8_t)vb;
                }
            }
        }
    }
}

// What the vector form does not take: one warp per row of q, k or v.
__global__ void __launch_bounds__(256) place_rows_kernel(const __grid_constant__ PlaceParams P) {
    if (P.pages) P.lens.publish();
    const int lane = threadIdx.x & 31, half = P.D >> 1;
    const int heads = P.Hq + (P.pages ? 2 : 1) * P.Hkv;
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
        // the two values of pair i, at da and db; whoever reads them writes them, so a dense row may be rotated where it lies
        const auto pair = [&](int i, int& da, int& db, float& ya, float& yb) {
            da = P.interleaved ? 2 * i : i;
            db = P.interleaved ? 2 * i + 1 : i + half;
            ya = ld_as_float(x, dtype, src + da);
            yb = ld_as_float(x, dtype, src + db);
            if (!turn) return;
            const long long at = (long long)place_row(P, b, t, i) * half + i;
            rope_pair(ya, yb, __ldg(P.cos_t + at), __ldg(P.sin_t + at), P.interleaved, ya, yb);
        };
        int da, db;
        float ya, yb;
        if (is_q || !P.pages) {
            const long long* os = is_q ? P.qos : P.vs;
            const long long dst = b * os[0] + hk * os[1] + t * os[2];
            for (int i = lane; i < half; i += 32) {
                pair(i, da, db, ya, yb);
                st_from_float(is_q ? P.q_out : P.k_pages, is_q ? P.qo_dtype : P.v_dtype, dst + da, ya);
                st_from_float(is_q ? P.q_out : P.k_pages, is_q ? P.qo_dtype : P.v_dtype, dst + db, yb);
            }
            continue;
        }
        const int at = P.lens.before(b) + t;
        const long long tile = (long long)P.page_table[(long long)b * P.max_pages + at / DEC_PT] * P.Hkv + hk;
        const long long dst = (tile * DEC_PT + at % DEC_PT) * P.D;
        if (P.pages == 1) {
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(is_k ? P.k_pages : P.v_pages) + dst;
            for (int i = lane; i < half; i += 32) {
                pair(i, da, db, ya, yb);
                out[da] = __float2bfloat16_rn(ya);
                out[db] = __float2bfloat16_rn(yb);
            }
            continue;
        }
        uint32_t top = 0;
        for (int i = lane; i < half; i += 32) {
            pair(i, da, db, ya, yb);
            top = max(top, max(abs_bits(ya), abs_bits(yb)));
        }
        const int byte = row8_byte(__uint_as_float(__reduce_max_sync(0xffffffffu, top)));
        int8_t* out = static_cast<int8_t*>(is_k ? P.k_pages : P.v_pages) + dst;
        for (int i = lane; i < half; i += 32) {
            pair(i, da, db, ya, yb);
            out[da] = byte == kRowNaN ? 0 : (int8_t)row8_code(ya, row8_inverse(byte));
            out[db] = byte == kRowNaN ? 0 : (int8_t)row8_code(yb, row8_inverse(byte));
        }
        if (lane == 0) P.scales[(tile * 2 + (is_k ? 0 : 1)) * DEC_PT + at % DEC_PT] = (uint8_t)byte;
    }
}

// Dense export of pages: out [B][Hkv][len][D] (strided), rows past a sequence's length are zero.  The first `front[b]` rows of a
// sequence's first page have been evicted and are not exported.
struct GatherPageParams {
    void* k_out;
    void* v_out;
    int k_dtype, v_dtype;
    long long ks[3], vs[3];
    const void* k_pages;  // bf16, or codes
    const void* v_pages;
    const uint8_t* scales;
    const int* page_table;
    const int* end;    // [B]
    const int* front;  // [B]
    int max_pages, Hkv, len, B;
};

// Four codes times a step: the byte with its sign bit flipped under the exponent of 2^23, which is then taken off.  Exact.  BIG: for any
// step; else for steps up to 2^100, where taking off and multiplying are one operation.
template <bool BIG>
__device__ __forceinline__ void row8_values(uint32_t codes, float step, float* f) {
    const uint32_t w = codes ^ 0x80808080u;
    const float off = -8388736.0f * step;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float x = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + j));
        f[j] = BIG ? (x - 8388736.0f) * step : fmaf(x, step, off);
    }
}

// A warp takes a page of K, then of V, all its loads at once, eight elements (16-bit pages) or sixteen (8-bit) per lane.  T: type of the
// results, whose rows start on multiples of 16 bytes, or 3: any types, any rows.  blockIdx.y: (sequence, kv head).  Half bound by HBM, half
// by the instructions that make values of codes (3 per element): B4 H8 S4096 D128 8-bit pages to bf16 (33 MB read, 67 written) 20.1 us =
// 5 TB/s; K and V together with 80 registers and two blocks an SM 21.1, a thread per 16 codes 22.9.
template <int PAGES, int D, int T>
__global__ void __launch_bounds__(256, 4) kvcache_gather_page_kernel(const __grid_constant__ GatherPageParams P) {
    constexpr int E = PAGES == 2 ? 16 : 8, CH = D / E, ROWS = 32 / CH, N = DEC_PT / ROWS;  // elements of a lane, lanes of a row, rows at once, rounds
    after_previous_launch();
    const int lane = threadIdx.x & 31, c = lane % CH * E, row = lane / CH;
    for (int pair = blockIdx.y; pair < P.B * P.Hkv; pair += gridDim.y) {
        const int b = pair / P.Hkv, hk = pair % P.Hkv, front = P.front[b], end = P.end[b];
        const int pages = (front + P.len + DEC_PT - 1) / DEC_PT;
        for (int p = (int)((blockIdx.x * blockDim.x + threadIdx.x) >> 5); p < pages; p += (int)((gridDim.x * blockDim.x) >> 5)) {
            const bool any = p * DEC_PT < end;
            const long long tile = any ? (long long)P.page_table[(long long)b * P.max_pages + p] * P.Hkv + hk : 0;
            const float step = any && PAGES == 2 ? row8_step(P.scales[tile * 2 * DEC_PT + lane]) : 0.0f;
            const auto rows = [&](int which, auto big) {
                uint4 raw[N] = {};
                if (any) {
                    const uint4* from = reinterpret_cast<const uint4*>(which ? P.v_pages : P.k_pages) + tile * (DEC_PT * D / E) + lane;
#pragma unroll
                    for (int j = 0; j < N; ++j) raw[j] = ld_stream(from + j * 32);
                }
                const long long* st = which ? P.vs : P.ks;
                const int dtype = T < 3 ? T : which ? P.v_dtype : P.k_dtype;
                void* out = which ? P.v_out : P.k_out;
                const long long first = b * st[0] + hk * st[1] + (p * DEC_PT - front) * st[2] + c;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int at = row + j * ROWS, t = p * DEC_PT + at - front;
                    const float mine = PAGES == 2 ? __shfl_sync(0xffffffffu, step, which * DEC_PT + at) : 0.0f;
                    if (t < 0 || t >= P.len) continue;
                    const bool there = p * DEC_PT + at < end;
                    const uint4 x = there ? raw[j] : make_uint4(0, 0, 0, 0);  // (codes of 0)
                    const long long dst = first + at * st[2];
                    float f[E];
                    if (PAGES == 2) {
                        const float by = there ? mine : 0.0f;
                        row8_values<decltype(big)::value>(x.x, by, f);
                        row8_values<decltype(big)::value>(x.y, by, f + 4);
                        row8_values<decltype(big)::value>(x.z, by, f + E - 8);
                        row8_values<decltype(big)::value>(x.w, by, f + E - 4);
                    } else {
                        rope_unpack16<false>(x, *reinterpret_cast<float(*)[8]>(f));
                    }
                    if (T < 3) {
#pragma unroll
                        for (int k = 0; k < E; k += 8) rope_store8(out, T, dst + k, *reinterpret_cast<float(*)[8]>(f + k));
                    } else {
#pragma unroll
                        for (int e = 0; e < E; ++e) st_from_float(out, dtype, dst + e, f[e]);
                    }
                }
            };
            const bool big = PAGES == 2 && __any_sync(0xffffffffu, !(step <= 0x1p100f));
#pragma unroll 1
            for (int which = 0; which < 2; ++which) {
                if (big) rows(which, std::true_type{});
                else rows(which, std::false_type{});
            }
        }
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
