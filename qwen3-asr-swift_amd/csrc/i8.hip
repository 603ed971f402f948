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
struct RowScale {
    float scale, s, inv, lift;
    __device__ explicit RowScale(float amax) {
        scale = amax / 127.0f;
        const bool bad = !(amax < INFINITY);       // infinity or NaN somewhere in the row
        lift = scale < 7.8886090522101181e-31f ? 18446744073709551616.0f : 1.0f;   // 2^-100, 2^64
        s = scale * lift;
        inv = s > 0.f && !bad ? 1.0f / s : 0.f;
        if (bad) scale = __builtin_nanf("");
    }
    __device__ int whole(float x) const {
        const float v = x * lift;
        float r = rintf(v * inv);
        const float e2 = 2.0f * fabsf(fmaf(-r, s, v)), dir = copysignf(1.0f, fmaf(-r, s, v));
        if (e2 > s || (e2 == s && ((int)r & 1))) r += dir;
        return inv > 0.f ? (int)fminf(fmaxf(r, -127.0f), 127.0f) : 0;
    }
};

template <bool F32>
__device__ __forceinline__ float i8_load(const void* row, int k) {
    if constexpr (F32) return ((const float*)row)[k];
    else return bf16_to_f32(((const bf16_t*)row)[k]);
}

// Maximum magnitude that turns into NaN where a NaN is among the values (fmaxf would drop it).
__device__ __forceinline__ float amax_of(float m, float x) {
    const float a = fabsf(x);
    return a > m || !(a == a) ? a : m;
}
__device__ __forceinline__ float wave_amax(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float t = __shfl_xor(v, o, 64);
        v = t > v || !(t == t) ? t : v;
    }
    return v;
}

// One wave per row.
template <bool F32>
__global__ __launch_bounds__(256) void i8_quantize_kernel(const void* x, int64_t ldx, int rows, int cols, int8_t* q, int64_t ldq, float* scales) {
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const void* src = (const char*)x + (int64_t)row * ldx * (F32 ? 4 : 2);
    float m = 0.f;
    for (int k = lane; k < cols; k += 64) m = amax_of(m, i8_load<F32>(src, k));
    const RowScale rs(wave_amax(m));
    if (lane == 0) scales[row] = rs.scale;
    int8_t* dst = q + (int64_t)row * ldq;
    for (int k4 = lane; k4 * 4 < ((cols + 15) & ~15); k4 += 64) {
        uint32_t b = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = k4 * 4 + e;
            if (k < cols) b |= (uint32_t)(rs.whole(i8_load<F32>(src, k)) & 255) << (8 * e);
        }
        *(uint32_t*)(dst + k4 * 4) = b;
    }
}

// ---- products ----

__device__ __forceinline__ float i8_scaled(int acc, float sa, float sw) { return ((float)acc * sw) * sa; }

// Stores NV consecutive values of one row, from column c on.
template <int NV>
__device__ __forceinline__ void i8_store(const I8Params& p, int m, int c, const float* y) {
    if (p.vec_out && c + NV <= p.N) {
        if (p.out_f32) {
            float* o = (float*)p.out + (int64_t)m * p.ldo + c;
#pragma unroll
            for (int e = 0; e < NV; e += 4) *(float4*)(o + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
        } else {
            bf16_t* o = (bf16_t*)p.out + (int64_t)m * p.ldo + c;
#pragma unroll
            for (int e = 0; e < NV; e += 8)
                *(uint4*)(o + e) = make_uint4(pack_bf16x2(y[e], y[e + 1]), pack_bf16x2(y[e + 2], y[e + 3]),
                                              pack_bf16x2(y[e + 4], y[e + 5]), pack_bf16x2(y[e + 6], y[e + 7]));
        }
        return;
    }
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
template <int MT, int NT, int STAGES>
__global__ __launch_bounds__(256, 2) void i8_gemm_kernel(I8Params p) {
    constexpr int BM = 32 * MT, BN = 32 * NT;
    constexpr int A_BYTES = BM * 128, W_BYTES = BN * 128, STAGE = A_BYTES + W_BYTES;
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
    const int nk_total = (k16 + 127) >> 7;
    const int per = (nk_total + p.ksplit - 1) / p.ksplit;
    const int kt0 = blockIdx.z * per, kt1 = min(nk_total, kt0 + per);

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
    auto stage = [&](int buf, int kt) {
        char* sa = smem + buf * STAGE;
        char* sw = sa + A_BYTES;
        const int kbase = kt * 128;
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
    };

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
    constexpr int INFLIGHT = (STAGES - 2) * (AP + WP);
    static_assert(INFLIGHT <= 63, "vmcnt field overflow");
    const int nt = kt1 - kt0;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
        if (s < nt) stage(s, kt0 + s);
    for (int t = 0; t < nt; ++t) {
        if (t + STAGES - 2 < nt) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(INFLIGHT) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (t + STAGES - 1 < nt) stage((t + STAGES - 1) % STAGES, kt0 + t + STAGES - 1);
        const char* sb = smem + (t % STAGES) * STAGE;
        i32x4 wf[2][NT], af[2][MT];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
            for (int b = 0; b < NT; ++b) wf[ks][b] = *(const i32x4*)(sb + w_rd[ks] + b * 4 * 128);
#pragma unroll
            for (int a = 0; a < MT; ++a) af[ks][a] = *(const i32x4*)(sb + a_rd[ks] + a * 16 * 128);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int b = 0; b < NT; ++b) acc[a][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[ks][b], af[ks][a], acc[a][b], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }

    // epilogue: lane (li, lg) owns row m, columns c0 .. c0 + 4 * NT - 1
    const int c0 = n0 + wc * 16 * NT + lg * 4 * NT;
    if (p.ksplit > 1) {
#pragma unroll
        for (int a = 0; a < MT; ++a) {
            const int m = m0 + wr * 16 * MT + a * 16 + li;
            if (m >= p.M) continue;
            int* o = p.slab + ((int64_t)blockIdx.z * p.M + m) * p.N;
#pragma unroll
            for (int b = 0; b < NT; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (c0 + b * 4 + r < p.N) o[c0 + b * 4 + r] = acc[a][b][r];
        }
        return;
    }
    float sw[4 * NT], bias[4 * NT];
#pragma unroll
    for (int e = 0; e < 4 * NT; ++e) {
        const int c = min(c0 + e, p.N - 1);
        sw[e] = p.sw[c];
        bias[e] = p.bias ? p.bias[c] : 0.f;
    }
#pragma unroll
    for (int a = 0; a < MT; ++a) {
        const int m = m0 + wr * 16 * MT + a * 16 + li;
        if (m >= p.M) continue;
        const float sa = p.sa[m];
        float y[4 * NT];
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[b * 4 + r] = i8_scaled(acc[a][b][r], sa, sw[b * 4 + r]) + bias[b * 4 + r];
        i8_store<4 * NT>(p, m, c0, y);
    }
}

// Sums of the parts of a split K.
__global__ __launch_bounds__(256) void i8_reduce_kernel(I8Params p) {
    const int64_t total = (int64_t)p.M * p.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int m = (int)(i / p.N), n = (int)(i - (int64_t)m * p.N);
        int acc = 0;
        for (int z = 0; z < p.ksplit; ++z) acc += p.slab[z * total + i];
        const float y = i8_scaled(acc, p.sa[m], p.sw[n]) + (p.bias ? p.bias[n] : 0.f);
        if (p.out_f32) ((float*)p.out)[(int64_t)m * p.ldo + n] = y;
        else ((bf16_t*)p.out)[(int64_t)m * p.ldo + n] = f32_to_bf16(y);
    }
}

template <int MT, int NT, int STAGES>
void launch_tile(const I8Params& p, hipStream_t s) {
    constexpr int BM = 32 * MT, BN = 32 * NT, LDS = STAGES * (BM + BN) * 128;
    static PerDeviceOnce once;
    once.run([&] {
        HIP_CHECK(hipFuncSetAttribute((const void*)i8_gemm_kernel<MT, NT, STAGES>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
    });
    ProfScope ps("i8_gemm_kernel", 2.0 * p.M * p.N * p.K, s);
    hipLaunchKernelGGL((i8_gemm_kernel<MT, NT, STAGES>), dim3(cdiv(p.M, BM) * cdiv(p.N, BN), 1, p.ksplit), dim3(256), LDS, s, p);
    HIP_CHECK(hipGetLastError());
}

struct I8Plan {
    int tile;     // 0: 128 x 128, 1: 64 x 64
    int ksplit;
};
I8Plan i8_plan(int M, int N, int K) {
    if ((int64_t)cdiv(M, 128) * cdiv(N, 128) >= 384) return {0, 1};
    return {1, 1};
}

}  // namespace

void launch_i8_quantize(const I8Source& src, int rows, int cols, int8_t* q, int64_t ldq, float* scales, hipStream_t s) {
    ProfScope ps("i8_quantize_kernel", (double)rows * cols * (src.f32 ? 5 : 3), s);
    const dim3 grid(cdiv(rows, 4)), block(256);
    if (src.f32) hipLaunchKernelGGL((i8_quantize_kernel<true>), grid, block, 0, s, src.x, src.ldx, rows, cols, q, ldq, scales);
    else hipLaunchKernelGGL((i8_quantize_kernel<false>), grid, block, 0, s, src.x, src.ldx, rows, cols, q, ldq, scales);
    HIP_CHECK(hipGetLastError());
}

int64_t i8_matmul_scratch(int M, int N, int K) {
    const I8Plan plan = i8_plan(M, N, K);
    return plan.ksplit > 1 ? (int64_t)plan.ksplit * M * N * 4 : 0;
}

void launch_i8_matmul(I8Params p, void* scratch, int64_t scratch_bytes, hipStream_t s) {
    const I8Plan plan = i8_plan(p.M, p.N, p.K);
    Q3_REQUIRE(i8_matmul_scratch(p.M, p.N, p.K) <= scratch_bytes, "i8_matmul: workspace too small");
    p.vec_out = ((uintptr_t)p.out % 16 == 0) && p.ldo % (p.out_f32 ? 4 : 8) == 0;
    p.ksplit = plan.ksplit;
    p.slab = (int*)scratch;
    if (plan.tile == 0) launch_tile<4, 4, 2>(p, s);
    else launch_tile<2, 2, 4>(p, s);
    if (p.ksplit > 1) {
        hipLaunchKernelGGL(i8_reduce_kernel, dim3((int)std::min<int64_t>(cdiv((int64_t)p.M * p.N, 256), 4096)), dim3(256), 0, s, p);
        HIP_CHECK(hipGetLastError());
    }
}
