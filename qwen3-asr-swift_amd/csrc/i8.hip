// 8-bit integer products for gfx950: y[m][n] = (sum_k q[m][k] w[n][k]) * s_x[m] * s_w[n] + b[n].
//
// The sums are whole numbers in 32 bits (v_mfma_i32_16x16x64_i8), so they do not depend on the order of their terms: every
// tile shape and every split of K gives the same bits.  The only roundings are those of x / s_x to 8 bits (the operator's
// definition), of the sum to fp32, of the two products with the scales, and of the result to its type.
#include "i8.h"
#include "prof.h"
#include <algorithm>

typedef __attribute__((ext_vector_type(4))) int i32x4;

#define LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

namespace {

// ---- rounding of rows to 8 bits ----

// How a row's values become whole numbers.  scale = max |x| / 127 rounded to fp32.  x / scale is rounded to the nearest whole
// number without a rounding of the quotient in between: r = rint(x * inv) is at most one off, and the remainder x - r * scale is
// exact in one fused multiply-add (r * scale and x are multiples of half an ulp of scale wherever r != 0, and the difference
// is below scale), so comparing twice the remainder with scale decides.  Scales so small that 1 / scale overflows or that products
// with it leave the normal range are lifted by 2^64 together with x, which is exact.
// Rounding is bound by vector instructions, so eight values take a short way first: adding 1.5 * 2^23 in the multiply-add leaves
// the rounded quotient in the low bits, from where bytes are picked.  It is right unless some remainder reaches half of scale
// (about one value in 10^5 for arbitrary data), and then the long way is taken.
// Rows of bf16 need no remainder.  With x = a 2^i and max |x| = b 2^j for whole a, b < 256, the ratio 127 x / max |x| is either half way
// between two whole numbers or at least 1 / (254 * 255) > 2^-16 of itself away from there; the true quotient differs from it by 2^-24, the
// computed one by 2^-22.  So only the ratios that are half way have to be decided, by the side that scale was rounded to: side is the
// reciprocal, moved by one step where it lies on the other side of 127 / max |x| than 1 / scale does.  (Where 127 * scale is max |x|
// itself, scale is a power of two and so is its reciprocal.)
struct RowScale {
    float scale, s, inv, lift, side;
    bool simple;
    __device__ RowScale() {}
    __device__ explicit RowScale(float amax) {
        scale = amax / 127.0f;
        const bool bad = !(amax < INFINITY);       // infinity or NaN somewhere in the row
        lift = scale < 7.8886090522101181e-31f ? 18446744073709551616.0f : 1.0f;   // 2^-100, 2^64
        s = bad ? 0.f : scale * lift;
        inv = s > 0.f ? 1.0f / s : 0.f;
        simple = !bad && (s == 0.f || lift == 1.0f);
        const float up = fmaf(scale, 127.0f, -amax), over = fmaf(inv, amax, -127.0f);
        side = up > 0.f && over >= 0.f ? __uint_as_float(__float_as_uint(inv) - 1) : up < 0.f && over <= 0.f ? __uint_as_float(__float_as_uint(inv) + 1) : inv;
        if (s == 0.f) side = 0.f;
        if (bad) scale = __builtin_nanf("");
    }
    __device__ int whole(float x) const {
        const float v = x * lift;
        float r = rintf(v * inv);
        const float e2 = 2.0f * fabsf(fmaf(-r, s, v)), dir = copysignf(1.0f, fmaf(-r, s, v));
        if (e2 > s || (e2 == s && ((int)r & 1))) r += dir;
        return inv > 0.f ? (int)fminf(fmaxf(r, -127.0f), 127.0f) : 0;
    }
    static __device__ uint2 low_bytes(const uint32_t* bits) {
        uint2 b;
        b.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(bits[3], bits[2], 0x0c0c0400), __builtin_amdgcn_perm(bits[1], bits[0], 0x0c0c0400), 0x05040100);
        b.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(bits[7], bits[6], 0x0c0c0400), __builtin_amdgcn_perm(bits[5], bits[4], 0x0c0c0400), 0x05040100);
        return b;
    }
    template <bool F32>
    __device__ uint2 pack8(const float* v) const {
        uint32_t bits[8];
        if constexpr (!F32) {
            if (simple) {
#pragma unroll
                for (int e = 0; e < 8; ++e) bits[e] = __float_as_uint(fmaf(v[e], side, 12582912.0f));
                return low_bytes(bits);
            }
        }
        float far = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float t = fmaf(v[e], inv, 12582912.0f);
            bits[e] = __float_as_uint(t);
            far = fmaxf(far, fabsf(fmaf(12582912.0f - t, s, v[e])));
        }
        if (2.0f * far < s && lift == 1.0f) {   // false for rows of zeros and rows that are not finite as well
            return low_bytes(bits);
        }
        uint32_t b[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e >> 2] |= (uint32_t)(whole(v[e]) & 255) << (8 * (e & 3));
        return make_uint2(b[0], b[1]);
    }
};

template <bool F32>
__device__ __forceinline__ float i8_load(const void* row, int k) {
    if constexpr (F32) return ((const float*)row)[k];
    else return bf16_to_f32(((const bf16_t*)row)[k]);
}

// 16 bytes from a place aligned to a value only: one load, which the memory unit splits where it crosses a line.
__device__ __forceinline__ uint4 i8_load16(const void* at) {
    struct __attribute__((packed, aligned(2))) Loose { uint32_t x, y, z, w; };
    const Loose a = *(const Loose*)at;
    return make_uint4(a.x, a.y, a.z, a.w);
}
// 8 consecutive values of a row; values from `cols` on read as zero.
template <bool F32>
__device__ __forceinline__ void i8_load8(const void* row, int k, int cols, float* v) {
    if (k + 8 <= cols) {
        const uint4 a = i8_load16((const char*)row + (int64_t)k * (F32 ? 4 : 2));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
        if constexpr (F32) {
            const uint4 b = i8_load16((const float*)row + k + 4);
            const uint32_t u[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = __uint_as_float(w[e]);
                v[4 + e] = __uint_as_float(u[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[2 * e] = __uint_as_float(w[e] << 16);
                v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < cols ? i8_load<F32>(row, k + e) : 0.f;
}
// 8 values of a row of at least 8, requested unconditionally: a load behind a branch is waited for at once.  What reaches behind the
// row's end is read from its last 8 values; then those that precede it move out.
template <bool F32>
struct I8Piece {
    static constexpr int WORDS = F32 ? 8 : 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void request(const void* row, int k, int cols) {
        const char* at = (const char*)row + (int64_t)min(k, cols - 8) * (F32 ? 4 : 2);
#pragma unroll
        for (int j = 0; j < WORDS; j += 4) {
            const uint4 u = i8_load16(at + 4 * j);
            w[j] = u.x;
            w[j + 1] = u.y;
            w[j + 2] = u.z;
            w[j + 3] = u.w;
        }
    }
    // Behind the request: values from cols on become zero.
    __device__ __forceinline__ void settle(int k, int cols) {
        if (cols & 7) {   // wave-uniform
            const int by = k < cols ? max(k + 8 - cols, 0) : 0, words = F32 ? by : by >> 1;
#pragma unroll
            for (int step = WORDS / 2; step; step >>= 1)
#pragma unroll
                for (int e = 0; e < WORDS; ++e) w[e] = words & step ? (e + step < WORDS ? w[e + step] : 0u) : w[e];
            if (!F32 && (by & 1)) {
#pragma unroll
                for (int e = 0; e < WORDS; ++e) w[e] = __builtin_amdgcn_alignbit(e + 1 < WORDS ? w[e + 1] : 0u, w[e], 16);
            }
        }
#pragma unroll
        for (int e = 0; e < WORDS; ++e) w[e] = k < cols ? w[e] : 0u;
    }
    __device__ __forceinline__ void values(float* v) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(F32 ? w[e % WORDS] : (e & 1) ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    }
};
// Magnitudes are compared as the bits of non-negative floats, an order in which a NaN lies above infinity.
__device__ __forceinline__ uint32_t i8_max8(uint32_t m, const float* v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
    return m;
}
// Largest magnitude of four bf16 values, as the bits of a float.
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    const u16x2 m = __builtin_elementwise_max(__builtin_bit_cast(u16x2, a & 0x7fff7fffu), __builtin_bit_cast(u16x2, b & 0x7fff7fffu));
    return (uint32_t)max(m.x, m.y) << 16;
}
template <bool F32>
__device__ __forceinline__ uint32_t i8_top(const I8Piece<F32>& x) {
    if constexpr (F32) {
        float v[8];
        x.values(v);
        return i8_max8(0, v);
    } else {
        return max(max_bf16x2(x.w[0], x.w[1]), max_bf16x2(x.w[2], x.w[3]));
    }
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max_bits(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false));
}
// Maximum over the 64 lanes (all active), the same in every lane.
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
    v = dpp_max_bits<0xB1>(v);    // quad_perm [1,0,3,2]
    v = dpp_max_bits<0x4E>(v);    // quad_perm [2,3,0,1]
    v = dpp_max_bits<0x124>(v);   // row_ror:4
    v = dpp_max_bits<0x128>(v);   // row_ror:8
    const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16), c = __builtin_amdgcn_readlane(v, 32),
                   d = __builtin_amdgcn_readlane(v, 48);
    return max(max(a, b), max(c, d));
}

// A workgroup's four waves per row (WHOLE), or one wave where rows are many and short; 8 values per lane and step.  Rows of up to
// 2048 * HELD values (512 * HELD) stay in registers between the maximum and the rounding, longer ones (HELD 0) are read twice.
// HBM-bound: 8100 x 2048 bf16 13.3 us behind others of its kind (3.7 TB/s read and written; 15.9 alone), 8100 x 6144 28 (5.3),
// 387 x 1003 fp32 2.8.
// With a wave per row, before bf16 rows lost their remainders: 14.3 against 13.5, 36 against 29; 8100 x 1003: 9.4 against 10.7.
template <bool F32, int HELD, bool WHOLE>
__global__ __launch_bounds__(256) void i8_quantize_kernel(const void* x, int64_t ldx, int rows, int cols, int8_t* q, int64_t ldq, float* scales) {
    constexpr int STEP = WHOLE ? 256 : 64;
    const int lane = WHOLE ? threadIdx.x : threadIdx.x & 63;
    const int row = WHOLE ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;   // WHOLE: never
    __shared__ uint32_t top[4];
    auto row_max = [&](uint32_t m) {
        m = wave_max_bits(m);
        if constexpr (WHOLE) {
            if ((lane & 63) == 0) top[lane >> 6] = m;
            __syncthreads();
            m = max(max(top[0], top[1]), max(top[2], top[3]));
        }
        return __uint_as_float(m);
    };
    const void* src = (const char*)x + (int64_t)row * ldx * (F32 ? 4 : 2);
    int8_t* dst = q + (int64_t)row * ldq;
    const int k16 = (cols + 15) & ~15;
    uint32_t m = 0;
    auto place = [&](int i) { return (i * STEP + lane) * 8; };
    if constexpr (HELD > 0) {
        I8Piece<F32> x8[HELD];
#pragma unroll
        for (int i = 0; i < HELD; ++i) x8[i].request(src, place(i), cols);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            x8[i].settle(place(i), cols);
            m = max(m, i8_top(x8[i]));
        }
        const RowScale rs(row_max(m));
        if (lane == 0) scales[row] = rs.scale;
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            float v[8];
            x8[i].values(v);
            if (place(i) < k16) *(uint2*)(dst + place(i)) = rs.template pack8<F32>(v);
        }
    } else if (cols < 8) {
        float v[8];
        i8_load8<F32>(src, place(0), cols, v);
        const RowScale rs(row_max(i8_max8(0, v)));
        if (lane == 0) scales[row] = rs.scale;
        if (place(0) < k16) *(uint2*)(dst + place(0)) = rs.template pack8<F32>(v);
    } else {
        constexpr int AT_ONCE = 4;
        I8Piece<F32> x8[AT_ONCE];
        auto read = [&](int i0) {
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) x8[i].request(src, place(i0 + i), cols);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) x8[i].settle(place(i0 + i), cols);
        };
        const int pieces = (k16 + 8 * STEP - 1) / (8 * STEP);
        for (int i0 = 0; i0 < pieces; i0 += AT_ONCE) {
            read(i0);
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) m = max(m, i8_top(x8[i]));
        }
        const RowScale rs(row_max(m));
        if (lane == 0) scales[row] = rs.scale;
        for (int i0 = 0; i0 < pieces; i0 += AT_ONCE) {
            read(i0);
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                float v[8];
                x8[i].values(v);
                if (place(i0 + i) < k16) *(uint2*)(dst + place(i0 + i)) = rs.template pack8<F32>(v);
            }
        }
    }
}

// ---- products ----

__device__ __forceinline__ float i8_scaled(int acc, float sa, float sw) { return ((float)acc * sw) * sa; }

// Stores a wave's block of 16 rows x 4 * NV columns from column c on; lane (li, lg) holds columns c + NV * lg .. of row m, which is
// its own by li.  Pieces of 16 bytes are dealt anew among the four lanes of a row (a transposition by row swaps), so that a store
// instruction covers 64 bytes of every row: with fp32 results 8100 x 2048 -> 12288 takes 224 us, 263 with each lane's pieces where they
// are (bf16: 200, 199), 2087 x 1576 -> 11183 68, 79.  Rows may have any alignment: the memory unit splits a store where it crosses a line.
template <int NV>
__device__ __forceinline__ void i8_store(const I8Params& p, int m, int c, const float* y) {
    const int lg = (threadIdx.x & 63) >> 4;
    auto pieces = [&](auto type, uint32_t (*w)[4]) {   // w: the lane's pieces
        typedef decltype(type) T;
        constexpr int N = NV * (int)sizeof(T) / 16;
        auto swap16 = [](uint32_t* a, uint32_t* b) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const auto r = __builtin_amdgcn_permlane16_swap(a[e], b[e], false, false);
                a[e] = r[0];
                b[e] = r[1];
            }
        };
        auto swap32 = [](uint32_t* a, uint32_t* b) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const auto r = __builtin_amdgcn_permlane32_swap(a[e], b[e], false, false);
                a[e] = r[0];
                b[e] = r[1];
            }
        };
        if constexpr (N == 2) {
            swap16(w[0], w[1]);
            swap32(w[0], w[1]);
        }
        if constexpr (N == 4) {
            swap16(w[0], w[1]);
            swap16(w[2], w[3]);
            swap32(w[0], w[2]);
            swap32(w[1], w[3]);
        }
        if (m >= p.M) return;
        struct __attribute__((packed, aligned(sizeof(T)))) Loose { uint32_t x, y, z, w; };
        char* row = (char*)((T*)p.out + (int64_t)m * p.ldo + c) + 16 * lg;
#pragma unroll
        for (int k = 0; k < N; ++k) *(Loose*)(row + 64 * k) = Loose{w[k][0], w[k][1], w[k][2], w[k][3]};
    };
    if (c + 4 * NV <= p.N) {   // wave-uniform
        if (p.out_f32) {
            uint32_t w[NV / 4][4];
#pragma unroll
            for (int e = 0; e < NV; ++e) w[e >> 2][e & 3] = __float_as_uint(y[e]);
            pieces(0.f, w);
            return;
        }
        if constexpr (NV >= 8) {
            uint32_t w[NV / 8][4];
#pragma unroll
            for (int e = 0; e < NV; e += 2) w[e >> 3][(e & 7) >> 1] = pack_bf16x2(y[e], y[e + 1]);
            pieces((bf16_t)0, w);
        } else if (m < p.M) {
            struct __attribute__((packed, aligned(2))) Loose { uint32_t x, y; };
            *(Loose*)((bf16_t*)p.out + (int64_t)m * p.ldo + c + NV * lg) = Loose{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
        }
        return;
    }
    if (m >= p.M) return;
    c += NV * lg;
#pragma unroll
    for (int e = 0; e < NV; ++e)
        if (c + e < p.N) {
            if (p.out_f32) ((float*)p.out)[(int64_t)m * p.ldo + c + e] = y[e];
            else ((bf16_t*)p.out)[(int64_t)m * p.ldo + c + e] = f32_to_bf16(y[e]);
        }
}

// Tile BM x BN x 128 per 256-thread workgroup (4 waves as 2 x 2).  Operands are staged global -> LDS by 16-byte loads into a
// ring of STAGES tiles (lane-linear image, XOR swizzle on the source chunk and on the fragment read); the weight fragment
// is the MFMA "A" operand, with weight rows dealt to MFMA rows so that a lane owns 4 * NT consecutive output columns.
template <int MT, int NT, int STAGES, int SUB>
__global__ __launch_bounds__(256, 2) void i8_gemm_kernel(I8Params p) {
    constexpr int BM = 32 * MT, BN = 32 * NT;
    constexpr int A_BYTES = BM * 128, W_BYTES = BN * 128, PART = A_BYTES + W_BYTES, STAGE = SUB * PART;
    constexpr int AP = BM * 8 / 256, WP = BN * 8 / 256;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int uwave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = uwave >> 1, wc = uwave & 1, li = lane & 15, lg = lane >> 4;

    // workgroup -> tile: contiguous tiles per XCD, groups of 8 M tiles share each N tile
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
    int L;
    {
        const int nwg = gridDim.x, b = blockIdx.x, q = nwg >> 3, r = nwg & 7, x = b & 7;
        L = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (b >> 3);
    }
    constexpr int GROUP = 8;
    const int per_group = GROUP * tiles_n, first_m = L / per_group * GROUP, gsz = min(GROUP, tiles_m - first_m);
    const int m0 = (first_m + (L % per_group) % gsz) * BM, n0 = (L % per_group) / gsz * BN;

    const int k16 = (p.K + 15) & ~15;
    const int nt = (k16 + 128 * SUB - 1) / (128 * SUB);

    constexpr int BUF_RANGE = 0x40000000, BUF_OOB = 0x7f000000;   // offsets at or beyond the range read as zero (K tail)
    const auto a_rsrc = uniform_buffer(p.A + (int64_t)m0 * p.lda, BUF_RANGE);
    const auto w_rsrc = uniform_buffer(p.W + (int64_t)n0 * p.ldw, BUF_RANGE);
    int a_voff[AP], a_koff[AP], w_voff[WP], w_koff[WP];
#pragma unroll
    for (int q = 0; q < AP; ++q) {
        const int c = q * 256 + tid, row = c >> 3, sc = (c & 7) ^ ((row >> 1) & 7);
        a_koff[q] = sc * 16;
        a_voff[q] = (min(m0 + row, p.M - 1) - m0) * (int)p.lda + sc * 16;
    }
#pragma unroll
    for (int q = 0; q < WP; ++q) {
        const int c = q * 256 + tid, row = c >> 3;
        const int f = ((row >> 1) & 1) | (((row / (4 * NT)) & 3) << 1), sc = (c & 7) ^ f;
        w_koff[q] = sc * 16;
        w_voff[q] = (min(n0 + row, p.N - 1) - n0) * (int)p.ldw + sc * 16;
    }
    auto stage = [&](int buf, int t) {
#pragma unroll
        for (int h = 0; h < SUB; ++h) {
            char* sa = smem + buf * STAGE + h * PART;
            char* sw = sa + A_BYTES;
            const int kbase = (t * SUB + h) * 128;
            const bool tail = kbase + 128 > k16;
#pragma unroll
            for (int q = 0; q < AP; ++q) {
                const int v = tail && kbase + a_koff[q] >= k16 ? BUF_OOB : a_voff[q];
                __builtin_amdgcn_raw_ptr_buffer_load_lds(a_rsrc, LDS_PTR(sa + (q * 256 + uwave * 64) * 16), 16, v, kbase, 0, 0);
            }
#pragma unroll
            for (int q = 0; q < WP; ++q) {
                const int v = tail && kbase + w_koff[q] >= k16 ? BUF_OOB : w_voff[q];
                __builtin_amdgcn_raw_ptr_buffer_load_lds(w_rsrc, LDS_PTR(sw + (q * 256 + uwave * 64) * 16), 16, v, kbase, 0, 0);
            }
        }
    };

    // the epilogue's operands, ahead of everything else
    const int c0 = n0 + wc * 16 * NT + lg * 4 * NT;
    float scale_w[4 * NT], bias[4 * NT], scale_a[MT];
#pragma unroll
    for (int e = 0; e < 4 * NT; ++e) {
        const int c = min(c0 + e, p.N - 1);
        scale_w[e] = p.sw[c];
        bias[e] = p.bias ? p.bias[c] : 0.f;
    }
#pragma unroll
    for (int a = 0; a < MT; ++a) scale_a[a] = p.sa[min(m0 + wr * 16 * MT + a * 16 + li, p.M - 1)];
    __builtin_amdgcn_sched_barrier(0);

    i32x4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = (i32x4){0, 0, 0, 0};
    int a_rd[2], w_rd[2];
    {
        const int fa = (li >> 1) & 7, fw = ((li >> 1) & 1) | ((li >> 2) << 1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            a_rd[ks] = (wr * 16 * MT + li) * 128 + (((lg + 4 * ks) ^ fa) << 4);
            w_rd[ks] = A_BYTES + (wc * 16 * NT + (li >> 2) * (4 * NT) + (li & 3)) * 128 + (((lg + 4 * ks) ^ fw) << 4);
        }
    }
    // Iteration t: wait until this wave's loads of tile t have landed (the STAGES - 2 younger tiles stay in flight), barrier,
    // refill the buffer of tile t - 1, compute tile t.
    constexpr int INFLIGHT = (STAGES - 2) * SUB * (AP + WP);
    static_assert(INFLIGHT <= 63, "vmcnt field overflow");
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
        if (s < nt) stage(s, s);
    for (int t = 0; t < nt; ++t) {
        if (t + STAGES - 2 < nt) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(INFLIGHT) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (t + STAGES - 1 < nt) stage((t + STAGES - 1) % STAGES, t + STAGES - 1);
        const char* sb = smem + (t % STAGES) * STAGE;
        i32x4 wf[SUB][2][NT], af[SUB][2][MT];
#pragma unroll
        for (int h = 0; h < SUB; ++h)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
                for (int b = 0; b < NT; ++b) wf[h][ks][b] = *(const i32x4*)(sb + h * PART + w_rd[ks] + b * 4 * 128);
#pragma unroll
                for (int a = 0; a < MT; ++a) af[h][ks][a] = *(const i32x4*)(sb + h * PART + a_rd[ks] + a * 16 * 128);
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int h = 0; h < SUB; ++h)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int a = 0; a < MT; ++a)
#pragma unroll
                    for (int b = 0; b < NT; ++b)
                        acc[a][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[h][ks][b], af[h][ks][a], acc[a][b], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }

    // epilogue: lane (li, lg) owns row m, columns c0 .. c0 + 4 * NT - 1
#pragma unroll
    for (int a = 0; a < MT; ++a) {
        const int m = m0 + wr * 16 * MT + a * 16 + li;
        float y[4 * NT];
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[b * 4 + r] = i8_scaled(acc[a][b][r], scale_a[a], scale_w[b * 4 + r]) + bias[b * 4 + r];
        i8_store<4 * NT>(p, m, n0 + wc * 16 * NT, y);
    }
}

// ---- many rows: 256 x 256 x 128 tiles ----
//
// Matrix-core bound.  The bf16 kernel's scheme (one 512-thread workgroup per CU, 8 waves as 2 x 4, eight phases per two K tiles,
// each {LDS -> registers, one staging unit's loads, barrier, 16 MFMAs, barrier}, waves 4-7 one barrier behind waves 0-3) carries
// over byte for byte: a K tile is 128 bytes of a row, which are 64 bf16 or 128 int8 values, and a 16-byte fragment feeds one
// 16x16x32 bf16 or one 16x16x64 int8 MFMA of the same length.  Twice the work per byte moved, so the phases are the same and
// the rate doubles: 8100 x 2048 -> 12288 takes 184-212 us (1.9-2.2 POP/s), the library's 8-bit product of that size 223.
constexpr int UNIT = 128 * 128, BUF = 4 * UNIT;   // A0 | A1 | W0 | W1, two K tiles
constexpr int SCALES = 3 * 256 * 4;
constexpr int LDS256 = 2 * BUF + 2 * SCALES;   // scales of the tile's rows, columns, and the bias, for two tiles

__global__ __launch_bounds__(512, 2) void i8_gemm256_kernel(I8Params p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int uwave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = uwave >> 2, wc = uwave & 3, li = lane & 15, lg = lane >> 4;
    const int tiles_m = (p.M + 255) >> 8, tiles_n = (p.N + 255) >> 8, total = tiles_m * tiles_n;
    constexpr int GROUP = 8;
    const int per_group = GROUP * tiles_n;
    const int k16 = (p.K + 15) & ~15, nt = (k16 + 127) >> 7;

    // thread t fills 16-byte slots t and 512 + t of every unit: LDS row q * 64 + (t >> 3), slot t & 7, which holds chunk
    // (t & 7) ^ ((row >> 1) & 7) of the K tile
    const int srow = tid >> 3, koff = ((tid & 7) ^ ((srow >> 1) & 7)) * 16;
    constexpr int BUF_RANGE = 0x40000000, BUF_OOB = 0x7f000000;
    int m0 = 0, n0 = 0;
    int a_off[2][2], w_off[2][2];
    __amdgpu_buffer_rsrc_t a_rsrc, w_rsrc;
    int parity = 0;
    auto setup = [&](int b) {
        const int q8 = total >> 3, r8 = total & 7, x = b & 7;
        const int L = (x < r8 ? x * (q8 + 1) : r8 * (q8 + 1) + (x - r8) * q8) + (b >> 3);
        const int first_m = L / per_group * GROUP, gsz = min(GROUP, tiles_m - first_m);
        m0 = (first_m + (L % per_group) % gsz) << 8;
        n0 = ((L % per_group) / gsz) << 8;
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                a_off[q][u] = (min(m0 + q * 128 + u * 64 + srow, p.M - 1) - m0) * (int)p.lda + koff;
                const int rho = q * 64 + srow, i = rho & 15, j = (rho >> 4) & 1, c = rho >> 5;
                w_off[q][u] = (min(n0 + c * 64 + (i >> 2) * 16 + u * 8 + j * 4 + (i & 3), p.N - 1) - n0) * (int)p.ldw + koff;
            }
        a_rsrc = uniform_buffer(p.A + (int64_t)m0 * p.lda, BUF_RANGE);
        w_rsrc = uniform_buffer(p.W + (int64_t)n0 * p.ldw, BUF_RANGE);
    };
    const int lds_lane0 = uwave * 64 * 16;
    auto stage = [&](int buf, int unit, int kt) {
        char* dst = smem + buf * BUF + unit * UNIT + lds_lane0;
        const bool past = kt >= nt;
        const int kbase = past ? 0 : kt * 128;
        const bool masked = past || kbase + koff >= k16;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int v = masked ? BUF_OOB : (unit < 2 ? a_off[q][unit & 1] : w_off[q][unit & 1]);
            if (unit < 2) __builtin_amdgcn_raw_ptr_buffer_load_lds(a_rsrc, LDS_PTR(dst + q * 512 * 16), 16, v, kbase, 0, 0);
            else __builtin_amdgcn_raw_ptr_buffer_load_lds(w_rsrc, LDS_PTR(dst + q * 512 * 16), 16, v, kbase, 0, 0);
        }
    };
    const int sw = (li >> 1) & 7;
    const int a_rd = (wr * 64 + li) * 128 + ((lg ^ (sw & 3)) << 4) + ((sw >> 2) << 6);
    const int w_rd = (wc * 32 + li) * 128 + ((lg ^ (sw & 3)) << 4) + ((sw >> 2) << 6);

    i32x4 acc[2][4][2][2];
    // The scales come first: 4 bytes per thread, waves 0-3 the rows', waves 4-7 the columns', waves 0-3 the bias.  What lies behind
    // the last row or column reads as zero.
    auto prefetch = [&]() {
        char* sc = smem + 2 * BUF + parity * SCALES + uwave * 256;
        const bool rows = uwave < 4;
        const int at = (tid & 255) * 4;
        const auto rsrc = uniform_buffer(rows ? p.sa + m0 : p.sw + n0, min(256, rows ? p.M - m0 : p.N - n0) * 4);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, LDS_PTR(sc), 4, at, 0, 0, 0);
        if (rows && p.bias) {
            const auto brsrc = uniform_buffer(p.bias + n0, min(256, p.N - n0) * 4);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(brsrc, LDS_PTR(sc + 2048), 4, at, 0, 0, 0);
        }
        stage(0, 2, 0); stage(0, 0, 0); stage(0, 3, 0); stage(0, 1, 0);
        stage(1, 2, 1); stage(1, 0, 1); stage(1, 3, 1);
    };
    setup(blockIdx.x);
    prefetch();
    for (int vb = blockIdx.x; vb < total; vb += gridDim.x) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[a][f][u][j] = (i32x4){0, 0, 0, 0};
        // first tile: its first K tile has landed; later ones: all of their loads have, before the previous tile's stores
        if (vb == (int)blockIdx.x) asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (wr == 1) __builtin_amdgcn_s_barrier();
        i32x4 af[4][2], w0f[2][2], w1f[2][2];
        const int iters = (nt + 1) >> 1;
        for (int it = 0; it < iters; ++it) {
            const int te = 2 * it;
            bool tail = false;
#pragma unroll
            for (int ph = 0; ph < 8; ++ph) {
                const int buf = ph >> 2, sub = ph & 3;
                if (ph == 4 && te + 1 >= nt) { tail = true; break; }
                const char* sb = smem + buf * BUF;
                if (sub == 0) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks) w0f[j][ks] = *(const i32x4*)(sb + 2 * UNIT + ((w_rd + j * 2048) ^ (ks << 6)));
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int f = 0; f < 4; ++f)
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks) af[f][ks] = *(const i32x4*)(sb + ((a_rd + f * 2048) ^ (ks << 6)));
                } else if (sub == 1) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks) w1f[j][ks] = *(const i32x4*)(sb + 3 * UNIT + ((w_rd + j * 2048) ^ (ks << 6)));
                } else if (sub == 2) {
#pragma unroll
                    for (int f = 0; f < 4; ++f)
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks) af[f][ks] = *(const i32x4*)(sb + UNIT + ((a_rd + f * 2048) ^ (ks << 6)));
                }
                switch (ph) {
                    case 0: stage(1, 1, te + 1); break;
                    case 1: stage(0, 2, te + 2); break;
                    case 2: stage(0, 0, te + 2); break;
                    case 3: stage(0, 3, te + 2); break;
                    case 4: stage(0, 1, te + 2); break;
                    case 5: stage(1, 2, te + 3); break;
                    case 6: stage(1, 0, te + 3); break;
                    default: stage(1, 3, te + 3); break;
                }
                if (sub == 0) asm volatile("s_waitcnt lgkmcnt(8)" ::: "memory");
                if (sub == 3) asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_setprio(1);
                const int ua = sub >> 1, uw = (sub == 1 || sub == 2) ? 1 : 0;
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int f = 0; f < 4; ++f)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            acc[ua][f][uw][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(uw ? w1f[j][ks] : w0f[j][ks], af[f][ks], acc[ua][f][uw][j], 0, 0, 0);
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_s_barrier();
            }
            if (tail) break;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (wr == 0) __builtin_amdgcn_s_barrier();

        // The next tile's first loads travel while this tile's sums become results; they have landed before the first store is
        // issued, so that the stores drain under the next tile's first phases.
        const int e_m0 = m0, e_n0 = n0;
        const char* const sc = smem + 2 * BUF + parity * SCALES;
        parity ^= 1;
        if (vb + (int)gridDim.x < total) {
            setup(vb + gridDim.x);
            prefetch();
        }
        // lane (li, lg) owns rows e_m0 + wr * 128 + a * 64 + f * 16 + li, columns c0 .. c0 + 15
        const int c0 = wc * 64 + lg * 16;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float4 sw4 = *(const float4*)(sc + 1024 + (c0 + u * 8 + j * 4) * 4);
                float4 bias = make_float4(0.f, 0.f, 0.f, 0.f);
                if (p.bias) bias = *(const float4*)(sc + 2048 + (c0 + u * 8 + j * 4) * 4);
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                        const float sa = *(const float*)(sc + (wr * 128 + a * 64 + f * 16 + li) * 4);
                        i32x4& v = acc[a][f][u][j];
                        v[0] = __float_as_int(i8_scaled(v[0], sa, sw4.x) + bias.x);
                        v[1] = __float_as_int(i8_scaled(v[1], sa, sw4.y) + bias.y);
                        v[2] = __float_as_int(i8_scaled(v[2], sa, sw4.z) + bias.z);
                        v[3] = __float_as_int(i8_scaled(v[3], sa, sw4.w) + bias.w);
                    }
            }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const int m = e_m0 + wr * 128 + a * 64 + f * 16 + li;
                float y[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) y[e] = __int_as_float(acc[a][f][e >> 3][(e >> 2) & 1][e & 3]);
                i8_store<16>(p, m, e_n0 + wc * 64, y);
            }
    }
}

void launch_gemm256(const I8Params& p, hipStream_t s) {
    static PerDeviceOnce once;
    once.run([&] { HIP_CHECK(hipFuncSetAttribute((const void*)i8_gemm256_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS256)); });
    // persistent: one workgroup per CU, a multiple of 8 so that a workgroup's tiles all map to its XCD
    const int tiles = cdiv(p.M, 256) * cdiv(p.N, 256), cus = std::max(8, device_cus() & ~7);
    ProfScope ps("i8_gemm256_kernel", 2.0 * p.M * p.N * p.K, s);
    hipLaunchKernelGGL(i8_gemm256_kernel, dim3(std::min(tiles, cus)), dim3(512), LDS256, s, p);
    HIP_CHECK(hipGetLastError());
}

// ---- a few rows: weights stream once, straight into registers ----
//
// HBM-bound (N * K bytes of weights): one workgroup takes 16 weight rows, its 8 waves take 64-wide steps of K in turn, and a
// wave's share of up to NS steps is requested at once.  The activation rows are rounded to 8 bits by every workgroup for itself,
// underneath those loads: they are a few KB from the L2, and a second kernel in front would cost more than the whole product.
// Weight rows are the MFMA "A" operand (lane: row li, bytes 16 lg ..), the activation rows in LDS the "B".
// 1 x 2048 -> 4096: 4.7 us behind others of its kind; 5 x 6144 -> 2048: 10.1, of which 2.5 are the rounding of 5 rows.
// F32: fp32 rows, else bf16.  HELD > 0: K is at least 8 and a thread's share of the rows, at most HELD pieces of 8 values, is
// requested before the weights and held in registers, so that nothing waits behind the weights; 0: any K, read twice.
constexpr int FEW_THREADS = 512, FEW_WAVES = 8, FEW_ROWS = 16, FEW_LDS = 100 * 1024;
constexpr int FEW_RED = FEW_WAVES * 256 * 4;
__host__ __device__ inline int few_stride(int K) { return ((K + 63) & ~63) + 16; }   // rows 16 bytes apart modulo the banks

template <bool F32, int NS, int HELD>
__global__ __launch_bounds__(FEW_THREADS, 2) void i8_few_rows_kernel(I8Params p, I8Source src) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ uint32_t amax[FEW_ROWS];
    __shared__ RowScale scales[FEW_ROWS];
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int k16 = (p.K + 15) & ~15, steps = (p.K + 63) >> 6, stride = few_stride(p.K);
    const int per_row = steps * 8, pieces = p.M * per_row;   // pieces of 8 values, those behind K zero
    int* const red = (int*)smem;                 // [wave][row][column]
    char* const xq = smem + FEW_RED;             // [M][stride]

    i32x4 w[NS];
    // pairs of steps, so that a wave reads whole 128-byte lines
    auto step_of = [&](int i0, int i) { return i0 + 2 * wave + (i & 1) + 2 * FEW_WAVES * (i >> 1); };
    // a wave's steps of 16 weight rows.  Loads are unconditional (one behind a branch would make the waits
    // count as if it had not been issued): what lies behind a row's end is read from its last 16 bytes and meets zeros.
    auto request = [&](int n0, int i0) {
        const int8_t* row = p.W + (int64_t)min(n0 + li, p.N - 1) * p.ldw;
#pragma unroll
        for (int i = 0; i < NS; ++i)
            w[i] = __builtin_nontemporal_load((const i32x4*)(row + min(step_of(i0, i) * 64 + lg * 16, k16 - 16)));
    };
    int n0 = blockIdx.x * 16;
    if (tid < FEW_ROWS) amax[tid] = 0;
    if constexpr (HELD > 0) {
        I8Piece<F32> held[HELD];
        int row_of[HELD], k_of[HELD];
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int c = min(tid + FEW_THREADS * i, pieces - 1);
            row_of[i] = c / per_row;
            k_of[i] = (c - row_of[i] * per_row) * 8;
            held[i].request((const char*)src.x + (int64_t)row_of[i] * src.ldx * (F32 ? 4 : 2), k_of[i], p.K);
        }
        __builtin_amdgcn_sched_barrier(0);
        request(n0, 0);
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            held[i].settle(k_of[i], p.K);
            const uint32_t top = i8_top(held[i]);
            const int first = __builtin_amdgcn_readfirstlane(row_of[i]);
            if (first == __builtin_amdgcn_readlane(row_of[i], 63)) {   // the wave's pieces lie in one row
                const uint32_t all = wave_max_bits(top);
                if (lane == 0) atomicMax(&amax[first], all);
            } else {
                atomicMax(&amax[row_of[i]], top);
            }
        }
        __syncthreads();
        if (tid < p.M) scales[tid] = RowScale(__uint_as_float(amax[tid]));
        __syncthreads();
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const RowScale rs = scales[row_of[i]];
            float v[8];
            held[i].values(v);
            if (tid + FEW_THREADS * i < pieces) *(uint2*)(xq + row_of[i] * stride + k_of[i]) = rs.template pack8<F32>(v);
        }
    } else {
        __syncthreads();
        for (int c0 = 0; c0 < pieces; c0 += FEW_THREADS) {
            const int c = min(c0 + tid, pieces - 1), m = c / per_row, k = (c - m * per_row) * 8;
            const char* row = (const char*)src.x + (int64_t)m * src.ldx * (F32 ? 4 : 2);
            float v[8];
            i8_load8<F32>(row, k, p.K, v);
            const uint32_t top = i8_max8(0, v);
            const int first = __builtin_amdgcn_readfirstlane(m);
            if (first == __builtin_amdgcn_readlane(m, 63)) {
                const uint32_t all = wave_max_bits(top);
                if (lane == 0) atomicMax(&amax[first], all);
            } else {
                atomicMax(&amax[m], top);
            }
        }
        __syncthreads();
        if (tid < p.M) scales[tid] = RowScale(__uint_as_float(amax[tid]));
        __syncthreads();
        for (int c = tid; c < pieces; c += FEW_THREADS) {
            const int m = c / per_row, k = (c - m * per_row) * 8;
            const RowScale rs = scales[m];
            const char* row = (const char*)src.x + (int64_t)m * src.ldx * (F32 ? 4 : 2);
            float v[8];
            i8_load8<F32>(row, k, p.K, v);
            *(uint2*)(xq + m * stride + k) = rs.template pack8<F32>(v);
        }
        request(n0, 0);
    }
    __syncthreads();

    const char* const xr = xq + min(li, p.M - 1) * stride + lg * 16;
    for (;;) {
        i32x4 acc = (i32x4){0, 0, 0, 0};
        for (int i0 = 0; i0 < steps; i0 += FEW_WAVES * NS) {
            if (i0 > 0) request(n0, i0);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const int step = step_of(i0, i);
                if (step < steps) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], *(const i32x4*)(xr + step * 64), acc, 0, 0, 0);
            }
        }
        const int done = n0;
        n0 += gridDim.x * 16;
        if (n0 < p.N) request(n0, 0);            // the next rows' weights travel while these are summed
        // lane (li, lg) holds activation row li against weight rows 4 lg .. 4 lg + 3
        *(i32x4*)(red + wave * 256 + li * 16 + 4 * lg) = acc;
        __syncthreads();
        if (tid < 256) {
            const int m = tid >> 4, n = done + (tid & 15);
            if (m < p.M && n < p.N) {
                int sum = 0;
#pragma unroll
                for (int v = 0; v < FEW_WAVES; ++v) sum += red[v * 256 + tid];
                const float y = i8_scaled(sum, scales[m].scale, p.sw[n]) + (p.bias ? p.bias[n] : 0.f);
                if (p.out_f32) ((float*)p.out)[(int64_t)m * p.ldo + n] = y;
                else ((bf16_t*)p.out)[(int64_t)m * p.ldo + n] = f32_to_bf16(y);
            }
        }
        if (n0 >= p.N) return;                   // the same for the whole workgroup
        __syncthreads();
    }
}

template <bool F32, int NS, int HELD>
void launch_few(const I8Params& p, const I8Source& src, hipStream_t s) {
    const int lds = FEW_RED + p.M * few_stride(p.K);
    static PerDeviceOnce once;
    once.run([&] {
        HIP_CHECK(hipFuncSetAttribute((const void*)i8_few_rows_kernel<F32, NS, HELD>, hipFuncAttributeMaxDynamicSharedMemorySize, FEW_RED + FEW_LDS));
    });
    ProfScope ps("i8_few_rows_kernel", (double)p.N * p.K, s);
    hipLaunchKernelGGL((i8_few_rows_kernel<F32, NS, HELD>), dim3(std::min(cdiv(p.N, 16), 512)), dim3(FEW_THREADS), lds, s, p, src);
    HIP_CHECK(hipGetLastError());
}
template <bool F32, int HELD>
void launch_few_steps(const I8Params& p, const I8Source& src, hipStream_t s) {
    const int per_wave = cdiv(cdiv(p.K, 64), FEW_WAVES);
    if (per_wave <= 4) launch_few<F32, 4, HELD>(p, src, s);
    else launch_few<F32, 12, HELD>(p, src, s);
}
// Whether rounding the rows in every workgroup is cheaper than a launch of its own (us, calls of one graph, one kernel against two):
// 1 x 2048 -> 4096: 4.7, 7.1; 5: 5.5, 7.2; 8 (4 pieces per thread): 5.7, 7.3; 12 (6): 8.2, 7.5; 1 x 6144 -> 2048: 7.2, 10.9; 5 (8 pieces):
// 10.1, 11.2; 6 (9, in a form that holds 12): 11.5, 11.2; 8: 12.0, 11.2; 16 x 1024 -> 4096: 5.6, 5.7; 8 x 2048 -> 12288: 7.9, 9.8;
// 12: 11.2, 9.8.  A K that leaves many of a wave's steps empty is the exception: 6 x 2816 -> 1024 (5 pieces) 9.0, 7.5.
template <bool F32>
bool launch_few_rows(const I8Params& p, const I8Source& src, hipStream_t s) {
    const int64_t held = cdiv((int64_t)p.M * cdiv(p.K, 64) * 8, FEW_THREADS);
    if (p.M > FEW_ROWS || held > (p.M <= 6 ? 8 : 4) || (p.M > 8 && p.N > 8192)) return false;
    if (p.K < 8) launch_few_steps<F32, 0>(p, src, s);
    else if (held <= 2) launch_few_steps<F32, 2>(p, src, s);
    else if (held <= 4) launch_few_steps<F32, 4>(p, src, s);
    else launch_few_steps<F32, 8>(p, src, s);
    return true;
}

template <int MT, int NT, int STAGES, int SUB>
void launch_tile(const I8Params& p, hipStream_t s) {
    constexpr int BM = 32 * MT, BN = 32 * NT, LDS = STAGES * SUB * (BM + BN) * 128;
    static PerDeviceOnce once;
    once.run([&] {
        HIP_CHECK(hipFuncSetAttribute((const void*)i8_gemm_kernel<MT, NT, STAGES, SUB>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
    });
    ProfScope ps("i8_gemm_kernel", 2.0 * p.M * p.N * p.K, s);
    hipLaunchKernelGGL((i8_gemm_kernel<MT, NT, STAGES, SUB>), dim3(cdiv(p.M, BM) * cdiv(p.N, BN)), dim3(256), LDS, s, p);
    HIP_CHECK(hipGetLastError());
}

}  // namespace

void launch_i8_quantize(const I8Source& src, int rows, int cols, int8_t* q, int64_t ldq, float* scales, hipStream_t s) {
    ProfScope ps("i8_quantize_kernel", (double)rows * cols * (src.f32 ? 5 : 3), s);
    const bool whole = cols >= 8 && (rows <= 1024 || cols > 1024);
    const dim3 grid(whole ? rows : cdiv(rows, 4)), block(256);
#define I8_QUANTIZE(F32, HELD, WHOLE) \
    hipLaunchKernelGGL((i8_quantize_kernel<F32, HELD, WHOLE>), grid, block, 0, s, src.x, src.ldx, rows, cols, q, ldq, scales)
#define I8_QUANTIZE_TYPE(HELD, WHOLE) \
    if (src.f32) I8_QUANTIZE(true, HELD, WHOLE); \
    else I8_QUANTIZE(false, HELD, WHOLE)
    if (cols < 8) { I8_QUANTIZE_TYPE(0, false); }
    else if (whole) {
        if (cols <= 2048) { I8_QUANTIZE_TYPE(1, true); }
        else if (cols <= 8192) { I8_QUANTIZE_TYPE(4, true); }
        else if (cols <= 24576) { I8_QUANTIZE_TYPE(12, true); }
        else { I8_QUANTIZE_TYPE(0, true); }
    } else {
        I8_QUANTIZE_TYPE(2, false);
    }
#undef I8_QUANTIZE_TYPE
#undef I8_QUANTIZE
    HIP_CHECK(hipGetLastError());
}

bool launch_i8_linear_few_rows(const I8Params& p, const I8Source& src, hipStream_t s) {
    return src.f32 ? launch_few_rows<true>(p, src, s) : launch_few_rows<false>(p, src, s);
}

void launch_i8_matmul(const I8Params& p, hipStream_t s) {
    // Few rows that are rounded already go through the smallest tiles too.  The kernel above, fed with them, took (us, calls of one graph,
    // against the tiles) 1 x 2048 -> 4096: 4.3, 4.7; 4: 4.5, 4.7; 8: 5.0, 4.7; 1 x 6144 -> 2048: 7.2, 8.1; 6: 9.0, 8.3; 8: 9.7, 8.4; but
    // 1 x 2816 -> 1024: 6.8, 4.9; 1 x 1024 -> 4096: 4.0, 3.3; 1 x 896 -> 4864: 5.3, 3.4; 1 x 2048 -> 12288: 7.4, 6.9; 6: 8.0, 7.1.
    // The smallest tiles that still fit the device at once win while the sums are short of workgroups, because the walk along K
    // is then all latency (us at K = 2048, and 6144 with *; 32 x 32 by 512 bytes of K, 32 x 64 by 512, by 256, 64 x 64, 128 x 128,
    // 256 x 256):  64 x 4096: 5.0, 5.7, 5.9, 8.2, 13.8, 24;  128 x 2048*: 8.7, 11.1, 12.6, 18, 37, 58;  256 x 4096: 14, 9.8, 7.7, 8.3,
    // 14, 26;  512 x 4096: 26, 18, 13, 9.3, 14.6, 26;  2000 x 4096: 98, 65, 47, 32, 22.4, 30;  1000 x 12288: 147, 98, 70, 47, 34, 32.
    const auto tiles = [&](int bm, int bn) { return (int64_t)cdiv(p.M, bm) * cdiv(p.N, bn); };
    if (tiles(32, 32) <= 256) launch_tile<1, 1, 3, 4>(p, s);
    else if (tiles(32, 64) <= 256) launch_tile<1, 2, 3, 4>(p, s);
    else if (tiles(32, 64) <= 512) launch_tile<1, 2, 3, 2>(p, s);
    else if (tiles(64, 64) <= 512 || p.M <= 64) launch_tile<2, 2, 2, 2>(p, s);
    else if (tiles(256, 256) >= 192 && p.M > 128) launch_gemm256(p, s);
    else launch_tile<4, 4, 2, 1>(p, s);
}
