// Attention over the paged KV cache for sequences that share prefixes (gfx950).
//
// o = sum_j p_j v_j, p = softmax_j(scale q . k_j).  The keys of a sequence are cut into its group's shared pages and its own
// pages, and both into chunks; a workgroup takes one chunk for one KV head and all query rows that read it -- of every
// sequence of the group for a shared chunk, so that a shared key crosses HBM once per group -- and leaves (max, sum, weighted
// sum of values) per row.  A second kernel joins the parts of a row.  Both softmax statistics and the sums stay in fp32; the
// probabilities are rounded to bf16 for the matrix cores (2^-9 relative each, which averages out over the keys of a row).
//
// HBM-bound: with G query heads per KV head and H hypotheses a shared chunk is 16 * QT columns of a matrix product against
// 2 * head_dim * 2 bytes per key.  Four waves take tiles of 32 keys in turn, each with its own statistics: S^T = K Q^T with the K
// rows loaded from memory as MFMA A fragments, then O^T = V^T P^T, where the exponentiated scores are as they stand the B
// fragment and the V rows reach the A fragments through transposing reads of a wave's own LDS tile.
#include "paged.h"
#include "prof.h"
#include <algorithm>
#include <type_traits>

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;

namespace {

constexpr int WAVES = 4;
constexpr int CHUNK = 512;        // keys of a workgroup; at most 1024, a page number per lane and 16 keys

union Frag {
    bf16x8 v;
    uint4 u;
    uint2 h[2];
};

// Reductions over the four 16-lane rows of a wave, result in every lane.
__device__ __forceinline__ float rows_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float rows_sum(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

struct AttnParams {
    const bf16_t* q; int64_t q_ld;
    bf16_t* out; int64_t o_ld;
    float* lse;
    const bf16_t *K, *V;                       // of the layer
    int64_t page_stride, head_stride;          // values
    const int *table, *lens, *seqs, *cu_rows, *cu_groups, *shared;
    int* status;
    int max_seqs, max_seq_pages, pages, pt_shift;
    int n, rows, n_groups, heads, kv_heads, group;
    int max_rows, max_group_rows, max_len, max_own, max_shared;
    float scale_log2;
    // shared chunks first, then own ones
    int chunk_p, chunks_p, tiles_p, chunk_s, chunks_s, tiles_s, blocks_p, slots;
    float* part_o;                             // [rows][heads][slots][D]
    float2* part_ml;                           // [rows][heads][slots]: maximum (base 2), sum
};

// The query rows of a workgroup: row r of M is row r0 + r / group of the step, head kvh * group + r % group.
struct Queries {
    int r0, M, first;      // first: this workgroup's lowest r
    int limit0, limit_t;   // row r sees keys below limit0 + limit_t * (r / group)
};

struct Entry {             // a sequence of the step
    int seq, r0, T, len;
    bool ok;
};
__device__ __forceinline__ Entry entry_of(const AttnParams& p, int i) {
    Entry e;
    e.seq = p.seqs[i];
    const int a = p.cu_rows[i], b = p.cu_rows[i + 1];
    const bool ok = (unsigned)e.seq < (unsigned)p.max_seqs && a >= 0 && b >= a && b <= p.rows && b - a <= p.max_rows;
    e.r0 = ok ? a : 0;
    e.T = ok ? b - a : 0;
    e.len = ok ? p.lens[e.seq] : 0;
    e.ok = ok && e.len >= 0 && e.len <= p.max_len;
    if (!e.ok) {
        if (threadIdx.x == 0) pages_error(p.status, (unsigned)e.seq < (unsigned)p.max_seqs ? Q3ASR_PAGES_BAD_BATCH : Q3ASR_PAGES_BAD_INDEX, i);
        e.seq = ok ? e.seq : 0;
        e.len = min(max(e.len, 0), p.max_len);
    }
    return e;
}
// Tokens that a group reads from the pages of its first sequence.
__device__ __forceinline__ int shared_of(const AttnParams& p, int g, const Entry& first) {
    return max(0, min(p.shared[g], first.len - first.T)) >> p.pt_shift << p.pt_shift;
}

template <int D>
struct Lds {
    static constexpr int VROW = 2 * D + 32, OROW = D + 4;
    static constexpr int V_BYTES = WAVES * 32 * VROW, O_BYTES = WAVES * 16 * OROW * 4;
    static constexpr int BYTES = V_BYTES > O_BYTES ? V_BYTES : O_BYTES;
};

// One workgroup's part: keys [k0, k1) of the sequence whose page numbers are in `pages`, for 16 * QT of the queries.
template <int D, int QT>
__device__ __forceinline__ void attend(const AttnParams& p, const int* pages, int kvh, int k0, int k1, const Queries& qs, int slot,
                                       char* lds, float (*sm_m)[64], float (*sm_l)[64]) {
    constexpr int NKS = D / 32, NDT = D / 16, LPR = D / 8, RPI = 64 / LPR, IV = 16 / RPI, VROW = Lds<D>::VROW, OROW = Lds<D>::OROW;
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nsub = (k1 - k0 + 15) >> 4, ntiles = (nsub + 1) >> 1;

    // page numbers of the chunk, 16 keys per lane
    int ids = 0;
    if (lane < nsub) {
        ids = pages[(k0 + 16 * lane) >> p.pt_shift];
        if ((unsigned)ids >= (unsigned)p.pages) {
            pages_error(p.status, Q3ASR_PAGES_BAD_INDEX, 0);
            ids = 0;
        }
    }
    const int64_t head = (int64_t)kvh * p.head_stride;
    const int in_page = (1 << p.pt_shift) - 1;

    Frag kf[2][NKS], vf[2][IV];
    auto base_of = [&](int t, int h) -> int64_t {   // first value of 16 keys; those behind the last are read from the last's
        const int sub = min(2 * t + h, nsub - 1);
        const int64_t page = __builtin_amdgcn_readlane(ids, sub);
        return page * p.page_stride + head + (int64_t)((k0 + 16 * sub) & in_page) * D;
    };
    auto load_k = [&](int t) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bf16_t* src = p.K + base_of(t, h) + li * D + 8 * lg;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) kf[h][ks].v = __builtin_nontemporal_load((const bf16x8*)(src + 32 * ks));
        }
    };
    auto load_v = [&](int t) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bf16_t* src = p.V + base_of(t, h) + (lane / LPR) * D + 8 * (lane % LPR);
#pragma unroll
            for (int i = 0; i < IV; ++i) vf[h][i].v = __builtin_nontemporal_load((const bf16x8*)(src + i * RPI * D));
        }
    };
    int t = wave;
    if (t < ntiles) {
        load_k(t);
        load_v(t);
    }

    // queries as B fragments: lane (li, lg) holds values 32 ks + 8 lg .. of query li
    Frag qf[QT][NKS];
    int limit[QT], lowest = k1;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int r = qs.first + 16 * qt + li;
        const bool ok = r < qs.M;
        const int rr = ok ? r : 0, tok = rr / p.group;
        limit[qt] = ok ? min(k1, qs.limit0 + qs.limit_t * tok) : 0;
        const bf16_t* src = p.q + (int64_t)(qs.r0 + tok) * p.q_ld + (kvh * p.group + rr - tok * p.group) * D + 8 * lg;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) qf[qt][ks].u = ok ? *(const uint4*)(src + 32 * ks) : make_uint4(0, 0, 0, 0);
    }
    lowest = min(k1, qs.limit0);   // keys below it are seen by all rows

    float m[QT], l[QT];
    f32x4 o[QT][NDT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        m[qt] = -INFINITY;
        l[qt] = 0.f;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[qt][dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    char* const vt = lds + wave * 32 * VROW;
    char* const vw = vt + (lane / LPR) * VROW + 16 * (lane % LPR);
    // transposing reads: per 16 lanes a block of 4 keys x 16 dims, lane 4 a + b addresses key a, dims 4 b .. 4 b + 3
    const char* const vr = vt + (4 * lg + (li >> 2)) * VROW + (li & 3) * 8;

    auto tile = [&](auto last) {
        constexpr bool LAST = decltype(last)::value;
        const int kv0 = k0 + 32 * t;
        f32x4 s[QT][2];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s[qt][h] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < NKS; ++ks) s[qt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[h][ks].v, qf[qt][ks].v, s[qt][h], 0, 0, 0);
            }
        if constexpr (!LAST) load_k(t + WAVES);
        Frag pf[QT];
        float alpha[QT];
        bool moved = false;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            float sv[8], top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) sv[j] = s[qt][j >> 2][j & 3] * p.scale_log2;
            if (kv0 + 32 > lowest) {   // the same for the whole workgroup's tile
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (kv0 + 16 * (j >> 2) + 4 * lg + (j & 3) >= limit[qt]) sv[j] = -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, sv[j]);
            const float m_new = fmaxf(m[qt], rows_max(top));
            const float m_use = m_new == -INFINITY ? 0.f : m_new;   // no key seen yet
            alpha[qt] = __builtin_amdgcn_exp2f(m[qt] - m_use);
            float pe[8], ps = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                pe[j] = __builtin_amdgcn_exp2f(sv[j] - m_use);
                ps += pe[j];
            }
            l[qt] = l[qt] * alpha[qt] + ps;   // this lane's keys only: the four rows of lanes are added at the end
            moved |= m_new != m[qt];
            m[qt] = m_new;
            pf[qt].u = make_uint4(pack_bf16x2(pe[0], pe[1]), pack_bf16x2(pe[2], pe[3]), pack_bf16x2(pe[4], pe[5]), pack_bf16x2(pe[6], pe[7]));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < IV; ++i) {
                // what lies behind the last key may be anything: a NaN there would survive its zero weight
                const bool keep = !LAST || kv0 + 16 * h + i * RPI + lane / LPR < k1;
                *(uint4*)(vw + (16 * h + i * RPI) * VROW) = keep ? vf[h][i].u : make_uint4(0, 0, 0, 0);
            }
        if constexpr (!LAST) load_v(t + WAVES);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (__builtin_amdgcn_ballot_w64(moved) != 0) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) o[qt][dt] *= alpha[qt];
        }
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            union { s16x4 v; uint2 u; } lo, hi;   // keys 4 lg .. 4 lg + 3 and 16 + 4 lg .. of dim 16 dt + li
            lo.v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vr + 32 * dt));
            hi.v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vr + 16 * VROW + 32 * dt));
            Frag va;
            va.h[0] = lo.u;
            va.h[1] = hi.u;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) o[qt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va.v, pf[qt].v, o[qt][dt], 0, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();   // the next tile's rows are written after these reads
    };
    // a tile with a successor is full, and its loads of that successor are unconditional
    if (t < ntiles) {
        for (; t + WAVES < ntiles; t += WAVES) tile(std::false_type{});
        tile(std::true_type{});
    }

    // join the four waves, 16 queries at a time
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const float lt = rows_sum(l[qt]);
        if (lg == 0) {
            sm_m[wave][16 * qt + li] = m[qt];
            sm_l[wave][16 * qt + li] = lt;
        }
    }
    float* const so = (float*)lds;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        __syncthreads();
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) *(f32x4*)(so + (wave * 16 + li) * OROW + 16 * dt + 4 * lg) = o[qt][dt];
        __syncthreads();
        constexpr int PER = D / 16;   // values per thread
        const int qi = tid >> 4, d0 = (tid & 15) * PER, r = qs.first + 16 * qt + qi;
        if (r < qs.M) {
            float M = -INFINITY, L = 0.f, acc[PER];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) M = fmaxf(M, sm_m[w][16 * qt + qi]);
            const float use = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float f = __builtin_amdgcn_exp2f(sm_m[w][16 * qt + qi] - use);
                L += sm_l[w][16 * qt + qi] * f;
#pragma unroll
                for (int e = 0; e < PER; ++e) acc[e] += so[(w * 16 + qi) * OROW + d0 + e] * f;
            }
            const int tok = r / p.group, row = qs.r0 + tok, hq = kvh * p.group + r - tok * p.group;
            if (p.slots == 1) {
                const float inv = L > 0.f || L != L ? 1.0f / L : 0.f;
                uint32_t w[PER / 2];
#pragma unroll
                for (int e = 0; e < PER; e += 2) w[e / 2] = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
                bf16_t* dst = p.out + (int64_t)row * p.o_ld + hq * D + d0;
                if constexpr (PER == 8) *(uint4*)dst = make_uint4(w[0], w[1], w[2], w[3]);
                else *(uint2*)dst = make_uint2(w[0], w[1]);
                if (p.lse && d0 == 0) p.lse[(int64_t)row * p.heads + hq] = (use + __builtin_amdgcn_logf(L)) * 0.69314718055994530942f;
            } else {
                const int64_t at = ((int64_t)row * p.heads + hq) * p.slots + slot;
#pragma unroll
                for (int e = 0; e < PER; e += 4) *(float4*)(p.part_o + at * D + d0 + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
                if (d0 == 0) p.part_ml[at] = make_float2(M, L);
            }
        }
    }
}

template <int D, int QP, int QS>
__global__ __launch_bounds__(256, QP == 4 || QS == 4 ? 1 : 2) void paged_attn_kernel(AttnParams p) {
    __shared__ __attribute__((aligned(16))) char lds[Lds<D>::BYTES];
    __shared__ float sm_m[WAVES][64], sm_l[WAVES][64];
    int b = blockIdx.x;
    Queries qs;
    if (b < p.blocks_p) {
        const int kvh = b % p.kv_heads;
        b /= p.kv_heads;
        const int g = b % p.n_groups;
        b /= p.n_groups;
        const int tile = b % p.tiles_p, ch = b / p.tiles_p;
        const int i0 = p.cu_groups[g], i1 = p.cu_groups[g + 1];
        if (i0 < 0 || i1 <= i0 || i1 > p.n) {
            if (threadIdx.x == 0 && (i0 < 0 || i1 < i0 || i1 > p.n)) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, g);
            return;
        }
        const Entry first = entry_of(p, i0);
        const int end = p.cu_rows[i1], keys = shared_of(p, g, first);
        if (end < first.r0 || end > p.rows || end - first.r0 > p.max_group_rows) {
            if (threadIdx.x == 0) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, i0);
            return;
        }
        qs.r0 = first.r0;
        qs.M = (end - first.r0) * p.group;
        qs.first = tile * 16 * QP;
        qs.limit0 = 0x7fffffff;
        qs.limit_t = 0;
        if (qs.first >= qs.M) return;
        const int k0 = ch * p.chunk_p, k1 = min(keys, k0 + p.chunk_p);
        if (keys > p.max_shared && threadIdx.x == 0) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, i0);
        if (k1 <= k0) {
            for (int r = qs.first + threadIdx.x; r < min(qs.M, qs.first + 16 * QP); r += 256) {
                const int tok = r / p.group, hq = kvh * p.group + r - tok * p.group;
                p.part_ml[((int64_t)(qs.r0 + tok) * p.heads + hq) * p.slots + ch] = make_float2(-INFINITY, 0.f);
            }
            return;
        }
        attend<D, QP>(p, p.table + (int64_t)first.seq * p.max_seq_pages, kvh, k0, k1, qs, ch, lds, sm_m, sm_l);
        return;
    }
    b -= p.blocks_p;
    const int kvh = b % p.kv_heads;
    b /= p.kv_heads;
    const int i = b % p.n;
    b /= p.n;
    const int tile = b % p.tiles_s, ch = b / p.tiles_s;
    const Entry e = entry_of(p, i);
    int from = 0;   // keys before it are read by the group
    bool ok = e.ok;
    if (p.n_groups > 0) {
        int g = -1;   // the last group that begins at or before entry i
        for (int g0 = 0; g0 < p.n_groups; g0 += 64) {
            const int at = g0 + (threadIdx.x & 63);
            const unsigned long long below = __ballot(at < p.n_groups && p.cu_groups[at] <= i);
            g += __popcll(below);
            if (below != ~0ull) break;
        }
        if (g >= 0) {
            const int i0 = p.cu_groups[g], i1 = p.cu_groups[g + 1];
            if (i0 >= 0 && i >= i0 && i < i1 && i1 <= p.n) {
                const Entry first = i0 == i ? e : entry_of(p, i0);
                from = shared_of(p, g, first);
                ok = ok && first.ok;
            } else {
                g = -1;
            }
        }
        if (g < 0 && threadIdx.x == 0) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, i);
    }
    qs.r0 = e.r0;
    qs.M = e.T * p.group;
    qs.first = tile * 16 * QS;
    qs.limit0 = e.len - e.T + 1;
    qs.limit_t = 1;
    if (qs.first >= qs.M) return;
    const int k0 = from + ch * p.chunk_s, k1 = min(e.len, k0 + p.chunk_s);
    if (threadIdx.x == 0 && ok && (from > max(0, e.len - e.T) || e.len - from > p.max_own)) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, i);
    const int slot = p.chunks_p + ch;
    if (k1 <= k0 && p.slots > 1) {
        for (int r = qs.first + threadIdx.x; r < min(qs.M, qs.first + 16 * QS); r += 256) {
            const int tok = r / p.group, hq = kvh * p.group + r - tok * p.group;
            p.part_ml[((int64_t)(qs.r0 + tok) * p.heads + hq) * p.slots + slot] = make_float2(-INFINITY, 0.f);
        }
        return;
    }
    attend<D, QS>(p, p.table + (int64_t)e.seq * p.max_seq_pages, kvh, k0, max(k0, k1), qs, slot, lds, sm_m, sm_l);
}

// Joins the parts of a row: one wave per (row, head).
template <int D>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnParams p) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (item >= (int64_t)p.rows * p.heads) return;
    const int row = (int)(item / p.heads), hq = (int)(item - (int64_t)row * p.heads);
    if (row >= p.cu_rows[p.n]) return;
    float M = -INFINITY;
    for (int s = lane; s < p.slots; s += 64) M = fmaxf(M, p.part_ml[item * p.slots + s].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float use = M == -INFINITY ? 0.f : M;
    constexpr int PER = D / 64;
    float L = 0.f, acc[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = 0.f;
    for (int s = 0; s < p.slots; ++s) {
        const float2 ml = p.part_ml[item * p.slots + s];
        if (ml.x == -INFINITY) continue;   // nothing seen: its sums were not written
        const float f = __builtin_amdgcn_exp2f(ml.x - use);
        L += ml.y * f;
        const float* src = p.part_o + (item * p.slots + s) * D + lane * PER;
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] += src[e] * f;
    }
    const float inv = L > 0.f || L != L ? 1.0f / L : 0.f;
    bf16_t* dst = p.out + (int64_t)row * p.o_ld + hq * D + lane * PER;
    if constexpr (PER == 2) *(uint32_t*)dst = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    else *dst = f32_to_bf16(acc[0] * inv);
    if (p.lse && lane == 0) p.lse[item] = (use + __builtin_amdgcn_logf(L)) * 0.69314718055994530942f;
}

struct Plan {
    int qp, qs;   // 16-query tiles per workgroup
    int chunk_p, chunks_p, tiles_p, chunk_s, chunks_s, tiles_s, slots;
};
int tiles_for(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }
Plan plan_for(const q3asr_kv_pages& c, const q3asr_attn_batch& b, int heads) {
    Plan r{};
    const int group = heads / c.kv_heads;
    const bool shares = b.n_groups > 0 && b.max_shared >= c.page_tokens;
    r.qs = tiles_for(b.max_rows * group);
    r.qp = shares ? std::max(r.qs, tiles_for(std::min(b.max_group_rows, 64) * group)) : r.qs;
    r.tiles_s = cdiv((int64_t)b.max_rows * group, 16 * r.qs);
    r.chunk_s = CHUNK;
    const int own = shares ? b.max_own : b.max_len;
    r.chunks_s = std::max(1, cdiv(own, r.chunk_s));
    if (shares) {
        r.tiles_p = cdiv((int64_t)b.max_group_rows * group, 16 * r.qp);
        r.chunk_p = CHUNK;
        r.chunks_p = cdiv(b.max_shared, r.chunk_p);
    } else {
        r.tiles_p = 1;
        r.chunk_p = CHUNK;
    }
    r.slots = r.chunks_p + r.chunks_s;
    return r;
}
int64_t part_bytes(const q3asr_kv_pages& c, const q3asr_attn_batch& b, int heads, const Plan& r) {
    return r.slots > 1 ? (((int64_t)b.rows * heads * r.slots * 8 + 255) & ~255ll) + (int64_t)b.rows * heads * r.slots * c.head_dim * 4 : 0;
}

template <int D>
void launch_d(const AttnParams& p, const Plan& r, int blocks, hipStream_t s) {
    const dim3 grid(blocks), block(256);
    switch (r.qp * 10 + r.qs) {
        case 11: hipLaunchKernelGGL((paged_attn_kernel<D, 1, 1>), grid, block, 0, s, p); break;
        case 21: hipLaunchKernelGGL((paged_attn_kernel<D, 2, 1>), grid, block, 0, s, p); break;
        case 41: hipLaunchKernelGGL((paged_attn_kernel<D, 4, 1>), grid, block, 0, s, p); break;
        case 22: hipLaunchKernelGGL((paged_attn_kernel<D, 2, 2>), grid, block, 0, s, p); break;
        case 42: hipLaunchKernelGGL((paged_attn_kernel<D, 4, 2>), grid, block, 0, s, p); break;
        default: hipLaunchKernelGGL((paged_attn_kernel<D, 4, 4>), grid, block, 0, s, p); break;
    }
    HIP_CHECK(hipGetLastError());
    if (p.slots > 1) {
        hipLaunchKernelGGL((paged_attn_join_kernel<D>), dim3(cdiv((int64_t)p.rows * p.heads, 4)), block, 0, s, p);
        HIP_CHECK(hipGetLastError());
    }
}

}  // namespace

int64_t paged_attention_workspace(const q3asr_kv_pages& c, const q3asr_attn_batch& b, int heads) {
    return part_bytes(c, b, heads, plan_for(c, b, heads));
}

void launch_paged_attention(const q3asr_kv_pages& c, int layer, const bf16_t* q, int64_t q_ld, int heads, float scale,
                            const q3asr_attn_batch& b, bf16_t* out, int64_t o_ld, float* lse, void* workspace, hipStream_t s) {
    const Plan r = plan_for(c, b, heads);
    AttnParams p{};
    p.q = q; p.q_ld = q_ld; p.out = out; p.o_ld = o_ld; p.lse = lse;
    p.head_stride = (int64_t)c.page_tokens * c.head_dim;
    p.page_stride = p.head_stride * c.kv_heads;
    p.K = c.k + (int64_t)layer * c.pages * p.page_stride;
    p.V = c.v + (int64_t)layer * c.pages * p.page_stride;
    p.table = c.table; p.lens = c.lens; p.status = c.status;
    p.seqs = b.seqs; p.cu_rows = b.cu_rows; p.cu_groups = b.cu_groups; p.shared = b.shared;
    p.max_seqs = c.max_seqs; p.max_seq_pages = c.max_seq_pages; p.pages = c.pages;
    while ((1 << p.pt_shift) < c.page_tokens) ++p.pt_shift;
    p.n = b.n; p.rows = b.rows; p.n_groups = r.chunks_p > 0 ? b.n_groups : 0;
    p.heads = heads; p.kv_heads = c.kv_heads; p.group = heads / c.kv_heads;
    p.max_rows = b.max_rows; p.max_group_rows = b.max_group_rows; p.max_len = b.max_len;
    p.max_own = r.chunks_p > 0 ? b.max_own : b.max_len;
    p.max_shared = b.max_shared;
    p.scale_log2 = scale * 1.44269504088896340736f;
    p.chunk_p = r.chunk_p; p.chunks_p = r.chunks_p; p.tiles_p = r.tiles_p;
    p.chunk_s = r.chunk_s; p.chunks_s = r.chunks_s; p.tiles_s = r.tiles_s; p.slots = r.slots;
    const int64_t ml = ((int64_t)b.rows * heads * r.slots * 8 + 255) & ~255ll;
    p.part_ml = (float2*)workspace;
    p.part_o = (float*)((char*)workspace + ml);
    const int64_t bp = (int64_t)p.n_groups * c.kv_heads * r.tiles_p * r.chunks_p, bs = (int64_t)b.n * c.kv_heads * r.tiles_s * r.chunks_s;
    Q3_REQUIRE(bp + bs < (1ll << 31), "paged_attention: too many workgroups (smaller bounds in the batch make fewer)");
    p.blocks_p = (int)bp;
    ProfScope ps("paged_attn_kernel", 4.0 * b.rows * heads * (double)b.max_len * c.head_dim, s);
    if (c.head_dim == 64) launch_d<64>(p, r, (int)(bp + bs), s);
    else launch_d<128>(p, r, (int)(bp + bs), s);
}
