// Attention over the paged KV cache for sequences that share prefixes (gfx950).
//
// o = sum_j p_j v_j, p = softmax_j(scale q . k_j).  The keys of a sequence are cut into its group's shared pages and its own
// pages, and both into chunks; a work item is one chunk for one KV head and up to 16 * QT of the query rows that read it -- of
// every sequence of the group for a shared chunk, so that a shared key crosses HBM once per group -- and leaves (max, sum,
// weighted sum of values) per row.  Three launches: one workgroup plans the items from the lengths and tables on the device,
// sorted by size; a grid that fills the device once works them off; a last one joins the parts of the rows that have several.
// Both softmax statistics and the sums stay in fp32; the probabilities are rounded to bf16 for the matrix cores (2^-9 relative
// each on average, which averages out over the keys of a row).
//
// HBM-bound: with G query heads per KV head and H hypotheses a shared chunk is 16 * QT columns of a matrix product against
// 2 * head_dim * 2 bytes per key.  Four waves take tiles of 32 keys in turn, each with its own statistics: S^T = K Q^T with the K
// rows loaded from memory as MFMA A fragments, then O^T = V^T P^T, where the exponentiated scores are as they stand the B
// fragment and the V rows reach the A fragments through transposing reads of a wave's own LDS tile.  A workgroup requests the
// next item's first tile before it joins its waves' results, and that item's page numbers an item ahead.
#include "paged.h"
#include "prof.h"
#include <algorithm>
#include <type_traits>

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;

namespace {

constexpr int WAVES = 4, PLAN = 1024;
constexpr int CHUNK_MAX = 1024;                   // keys: one page number per lane and 16 keys
constexpr int BUCKETS = CHUNK_MAX / 32 + 1;       // items by their number of 32-key tiles; at most 64
constexpr int BATCH = 64;                         // items whose descriptions a workgroup holds at a time
constexpr int CUS = 256, PLAIN_ITEMS = 512;

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

// LDS written by some lanes of a wave is read by others behind this.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A chunk of keys for up to 16 * QT query rows: row r of M is row r0 + r / group of the step, head kvh * group + r % group, and
// sees keys below `limit` + r / group of an own chunk, all keys of a shared one.
struct __attribute__((aligned(16))) Item {
    int r0, M, first;   // first: the lowest r
    int seq, k0, k1;    // keys [k0, k1) of the pages of sequence seq
    int limit;          // SHARED: a shared chunk
    int slot;           // where the part goes; DIRECT: it is the rows' only one and goes to the output
};
constexpr int SHARED = 0x7fffffff, DIRECT = -1;

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
    int chunk, chunks_p, chunks_s, slots, rows_p, rows_s;   // shared chunks' slots first, then own ones'; query rows of an item
    int plain;                                 // no plan: own items of whole sequences, tiles_s each
    int tiles_s;
    void* plan_ws;                             // what of a plan does not fit LDS
    int* count;                                // [1] items
    int* parts;                                // [rows] parts of a row: shared | own << 16
    Item* items;
    float2* part_ml;                           // [rows][heads][slots]: maximum (base 2), sum
    float* part_o;                             // [rows][heads][slots][D]
};

// ---- plan ----
struct Entry {             // a sequence of the step
    int seq, r0, T, len;
    bool ok;
};
__device__ __forceinline__ Entry entry_of(const AttnParams& p, int i, bool report) {
    Entry e;
    e.seq = p.seqs[i];
    const int a = p.cu_rows[i], b = p.cu_rows[i + 1];
    const bool in = (unsigned)e.seq < (unsigned)p.max_seqs, ok = in && a >= 0 && b >= a && b <= p.rows && b - a <= p.max_rows;
    e.r0 = ok ? a : 0;
    e.T = ok ? b - a : 0;
    e.len = ok ? p.lens[e.seq] : 0;
    e.ok = ok && e.len >= 0 && e.len <= p.max_len;
    if (!e.ok) {
        if (report) pages_error(p.status, in ? Q3ASR_PAGES_BAD_BATCH : Q3ASR_PAGES_BAD_INDEX, i);
        e.seq = in ? e.seq : 0;
        e.len = min(max(e.len, 0), p.max_len);
    }
    return e;
}

// Two dependent loads per sequence (its number, its length), everything else from LDS: with one workgroup nothing covers latency.
// Lists beyond HELD entries or groups stay in the workspace.
constexpr int HELD = 1024;
__global__ __launch_bounds__(PLAN) void paged_attn_plan_kernel(AttnParams p) {
    __shared__ int bucket[64];
    __shared__ Entry held[HELD];
    __shared__ int held_cu[HELD + 1], held_from[HELD];
    const int tid = threadIdx.x;
    Entry* const entry = p.n <= HELD ? held : (Entry*)p.plan_ws;
    int* const from = p.n_groups <= HELD ? held_from : (int*)((Entry*)p.plan_ws + p.n);   // tokens that a group shares
    const int* const cu = p.n_groups <= HELD ? held_cu : p.cu_groups;
    if (tid < 64) bucket[tid] = 0;
    for (int r = tid; r < p.rows; r += PLAN) p.parts[r] = 0;
    for (int i = tid; i < p.n; i += PLAN) entry[i] = entry_of(p, i, true);
    if (p.n_groups > 0 && p.n_groups <= HELD)
        for (int g = tid; g <= p.n_groups; g += PLAN) held_cu[g] = p.cu_groups[g];
    __syncthreads();
    for (int g = tid; g < p.n_groups; g += PLAN) {
        const int i0 = cu[g], i1 = cu[g + 1], shared = p.shared[g];
        from[g] = 0;
        if (i0 < 0 || i1 < i0 || i1 > p.n) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, g);
        else if (i1 > i0) {
            const Entry first = entry[i0];
            const int end = p.cu_rows[i1];
            if (shared > p.max_shared || (first.ok && (end < first.r0 || end > p.rows || end - first.r0 > p.max_group_rows)))
                pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, i0);
            from[g] = max(0, min(min(shared, p.max_shared), first.len - first.T)) >> p.pt_shift << p.pt_shift;
        }
    }
    __syncthreads();
    // the items of group g (which = g) or sequence i (which = n_groups + i), in any order: f(item)
    auto items_of = [&](int which, bool report, auto f) {
        Item it;
        if (which < p.n_groups) {
            const int i0 = cu[which], i1 = cu[which + 1], keys = from[which];
            if (i0 < 0 || i1 <= i0 || i1 > p.n) return;
            const Entry first = entry[i0];
            const int end = min(p.cu_rows[i1], first.r0 + p.max_group_rows);
            if (!first.ok || end > p.rows) return;
            it.r0 = first.r0;
            it.M = max(0, end - first.r0) * p.group;
            it.seq = first.seq;
            it.limit = SHARED;
            for (int ch = 0; ch * p.chunk < keys; ++ch)
                for (it.first = 0; it.first < it.M; it.first += p.rows_p) {
                    it.k0 = ch * p.chunk;
                    it.k1 = min(keys, it.k0 + p.chunk);
                    it.slot = ch;
                    f(it);
                }
            return;
        }
        const int i = which - p.n_groups;
        const Entry e = entry[i];
        int behind = 0;    // keys before it are read by the group
        bool ok = e.ok;
        if (p.n_groups > 0) {
            int lo = 0, hi = p.n_groups;   // the last group that begins at or before entry i
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= i) lo = mid;
                else hi = mid;
            }
            const int i0 = cu[lo], i1 = cu[lo + 1];
            if (i0 >= 0 && i >= i0 && i < i1 && i1 <= p.n) {
                behind = from[lo];
                ok = ok && entry[i0].ok;
            } else if (report) {
                pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, i);
            }
        }
        if (report && ok && (behind > max(0, e.len - e.T) || e.len - behind > p.max_own)) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, i);
        const int own = min(max(0, e.len - behind), p.chunks_s * p.chunk), parts_p = (behind + p.chunk - 1) / p.chunk;
        const int parts_s = max((own + p.chunk - 1) / p.chunk, parts_p ? 0 : 1);   // a row without keys has one empty part
        it.r0 = e.r0;
        it.M = e.T * p.group;
        it.seq = e.seq;
        it.limit = e.len - e.T + 1;
        if (report)
            for (int t = 0; t < e.T; ++t) p.parts[e.r0 + t] = parts_p | parts_s << 16;
        for (int ch = 0; ch < parts_s; ++ch)
            for (it.first = 0; it.first < it.M; it.first += p.rows_s) {
                it.k0 = behind + ch * p.chunk;
                it.k1 = min(behind + own, it.k0 + p.chunk);
                it.slot = parts_p + parts_s == 1 ? DIRECT : p.chunks_p + ch;
                f(it);
            }
    };
    // the largest first, so that the last items to be taken up are small
    auto bucket_of = [](const Item& it) { return BUCKETS - 1 - ((it.k1 - it.k0 + 31) >> 5); };
    const int all = p.n_groups + p.n;
    for (int w = tid; w < all; w += PLAN) items_of(w, true, [&](const Item& it) { atomicAdd(&bucket[bucket_of(it)], 1); });
    __syncthreads();
    if (tid < 64) {
        const int n = bucket[tid];
        int x = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(x, o, 64);
            if (tid >= o) x += t;
        }
        bucket[tid] = x - n;
        if (tid == 63) *p.count = x;
    }
    __syncthreads();
    for (int w = tid; w < all; w += PLAN) items_of(w, false, [&](const Item& it) { p.items[atomicAdd(&bucket[bucket_of(it)], 1)] = it; });
}

// Without a plan the groups are not used; a workgroup of its own checks them all the same.
__device__ void check_groups(const AttnParams& p) {
    if (threadIdx.x == 0 && (p.cu_groups[0] != 0 || p.cu_groups[p.n_groups] != p.n)) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, 0);
    for (int g = threadIdx.x; g < p.n_groups; g += 256) {
        const int i0 = p.cu_groups[g], i1 = p.cu_groups[g + 1], shared = p.shared[g];
        if (i0 < 0 || i1 < i0 || i1 > p.n) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, g);
        else if (i1 > i0) {
            const Entry first = entry_of(p, i0, false);
            const int end = p.cu_rows[i1], behind = max(0, min(shared, first.len - first.T)) >> p.pt_shift << p.pt_shift;
            if (!first.ok) continue;
            if (shared > p.max_shared || end < first.r0 || end > p.rows || end - first.r0 > p.max_group_rows)
                pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, i0);
            for (int i = i0; i < i1; ++i) {
                const Entry e = entry_of(p, i, false);
                if (e.ok && (behind > max(0, e.len - e.T) || e.len - behind > p.max_own)) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, i);
            }
        }
    }
}

template <int D>
struct Lds {
    static constexpr int KROW = 2 * D + 16, VROW = 2 * D + 32, OROW = D + 4;   // padded: fragment and transposing reads meet all banks
    static constexpr int V_BYTES = WAVES * 32 * VROW, O_BYTES = WAVES * 16 * OROW * 4;
    static constexpr int BYTES = V_BYTES > O_BYTES ? V_BYTES : O_BYTES;
};

// A wave's registers that carry over from one item to the next.
template <int D, int QMAX>
struct Stream {
    static constexpr int NKS = D / 32, LPR = D / 8, RPI = 64 / LPR, IV = 16 / RPI, NQ = (16 * QMAX * LPR + 255) / 256;
    Frag kf[2][IV], vf[2][IV];    // a tile of 32 keys, as rows
    uint4 qv[NQ];                 // the thread's pieces of the item's query rows, on their way to LDS
    int ids;                      // page numbers of the item's chunk, 16 keys per lane

    const AttnParams& p;
    const int lane, li, lg;
    int k0, nsub;
    int64_t head;
    __device__ Stream(const AttnParams& p_, int lane_) : p(p_), lane(lane_), li(lane_ & 15), lg(lane_ >> 4) {}

    __device__ int page_numbers(int seq, int k0_, int k1_) const {
        const int n = (k1_ - k0_ + 15) >> 4;
        if (n <= 0) return 0;
        return p.table[(int64_t)seq * p.max_seq_pages + ((k0_ + 16 * min(lane, n - 1)) >> p.pt_shift)];
    }
    __device__ void begin(int ids_, int kvh, int k0_, int k1_) {
        k0 = k0_;
        nsub = (k1_ - k0_ + 15) >> 4;
        head = (int64_t)kvh * p.head_stride;
        ids = ids_;
        if ((unsigned)ids >= (unsigned)p.pages) {
            if (nsub > 0) pages_error(p.status, Q3ASR_PAGES_BAD_INDEX, 0);
            ids = 0;
        }
    }
    __device__ void load_q(const Item& it, int kvh, int most) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int idx = threadIdx.x + 256 * i, in = idx / LPR, r = it.first + in;
            qv[i] = make_uint4(0, 0, 0, 0);
            if (in < most && r < it.M) {
                const int tok = r / p.group;
                qv[i] = *(const uint4*)(p.q + (int64_t)(it.r0 + tok) * p.q_ld + (kvh * p.group + r - tok * p.group) * D + 8 * (idx % LPR));
            }
        }
    }
    __device__ void store_q(char* sq) const {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int idx = threadIdx.x + 256 * i, in = idx / LPR;
            if (in < 16 * QMAX) *(uint4*)(sq + in * (2 * D + 16) + 16 * (idx % LPR)) = qv[i];
        }
    }
    __device__ int64_t base_of(int t, int h) const {   // first value of 16 keys; those behind the last are read from the last's
        const int sub = min(2 * t + h, nsub - 1);
        const int64_t page = __builtin_amdgcn_readlane(ids, sub);
        return page * p.page_stride + head + (int64_t)((k0 + 16 * sub) & ((1 << p.pt_shift) - 1)) * D;
    }
    // 32 keys of K or V as whole rows, RPI of them per instruction
    __device__ void load(const bf16_t* pool, Frag (&x)[2][IV], int t) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bf16_t* src = pool + base_of(t, h) + (lane / LPR) * D + 8 * (lane % LPR);
#pragma unroll
            for (int i = 0; i < IV; ++i) x[h][i].v = __builtin_nontemporal_load((const bf16x8*)(src + i * RPI * D));
        }
    }
    __device__ void load_k(int t) { load(p.K, kf, t); }
    __device__ void load_v(int t) { load(p.V, vf, t); }
};

// One item for one KV head; its first tile has been requested.  request_next: the same for the next one, which a single group of
// queries leaves registers for before the join.
template <int D, int QT, int QMAX, class F>
__device__ __forceinline__ void attend(const AttnParams& p, const Item& it, int kvh, Stream<D, QMAX>& st, char* lds, char* sq, float (*sm_m)[64],
                                       float (*sm_l)[64], F request_next) {
    constexpr int NKS = D / 32, NDT = D / 16, LPR = D / 8, RPI = 64 / LPR, IV = 16 / RPI;
    constexpr int KROW = Lds<D>::KROW, VROW = Lds<D>::VROW, OROW = Lds<D>::OROW;
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int k0 = it.k0, k1 = it.k1, ntiles = (k1 - k0 + 31) >> 5;
    int t = wave;

    int limit[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int r = it.first + 16 * qt + li;
        limit[qt] = r >= it.M ? 0 : it.limit == SHARED ? k1 : min(k1, it.limit + r / p.group);
    }
    // queries as B fragments: lane (li, lg) reads values 32 ks + 8 lg .. of query li
    const char* const qr = sq + li * (2 * D + 16) + 16 * lg;
    const int lowest = min(k1, it.limit);   // keys below it are seen by all rows

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
    char* const kw = vt + (lane / LPR) * KROW + 16 * (lane % LPR);
    char* const vw = vt + (lane / LPR) * VROW + 16 * (lane % LPR);
    const char* const kr = vt + li * KROW + 16 * lg;
    // transposing reads: per 16 lanes a block of 4 keys x 16 dims, lane 4 a + b addresses key a, dims 4 b .. 4 b + 3
    const char* const vr = vt + (4 * lg + (li >> 2)) * VROW + (li & 3) * 8;

    auto tile = [&](auto last) {
        constexpr bool LAST = decltype(last)::value;
        const int kv0 = k0 + 32 * t;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < IV; ++i) *(uint4*)(kw + (16 * h + i * RPI) * KROW) = st.kf[h][i].u;
        if constexpr (!LAST) st.load_k(t + WAVES);
        wave_lds_fence();
        Frag ka[2][NKS];   // K rows as A fragments: lane (li, lg) reads values 32 ks + 8 lg .. of key li
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) ka[h][ks].u = *(const uint4*)(kr + 16 * h * KROW + 64 * ks);
        Frag pf[QT];
        float alpha[QT];
        bool moved = false;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            Frag qf[NKS];
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) qf[ks].u = *(const uint4*)(qr + qt * 16 * (2 * D + 16) + 64 * ks);
            f32x4 s[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s[h] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < NKS; ++ks) s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[h][ks].v, qf[ks].v, s[h], 0, 0, 0);
            }
            float sv[8], top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) sv[j] = s[j >> 2][j & 3] * p.scale_log2;
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
            if constexpr (QT > 1) __builtin_amdgcn_sched_barrier(0);   // one group of queries' fragments in registers at a time
        }
        __builtin_amdgcn_wave_barrier();   // the V rows go where the K rows were
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < IV; ++i) {
                // what lies behind the last key may be anything: a NaN there would survive its zero weight
                const bool keep = !LAST || kv0 + 16 * h + i * RPI + lane / LPR < k1;
                *(uint4*)(vw + (16 * h + i * RPI) * VROW) = keep ? st.vf[h][i].u : make_uint4(0, 0, 0, 0);
            }
        if constexpr (!LAST) st.load_v(t + WAVES);
        wave_lds_fence();
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

    if constexpr (QT == 1) request_next();
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
        if (QT == 1) st.store_q(sq);   // the next item's: all waves are done with this one's
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) *(f32x4*)(so + (wave * 16 + li) * OROW + 16 * dt + 4 * lg) = o[qt][dt];
        __syncthreads();
        constexpr int PER = D / 16;   // values per thread
        const int qi = tid >> 4, d0 = (tid & 15) * PER, r = it.first + 16 * qt + qi;
        if (r < it.M) {
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
            const int tok = r / p.group, row = it.r0 + tok, hq = kvh * p.group + r - tok * p.group;
            if (it.slot == DIRECT) {
                const float inv = L > 0.f || L != L ? 1.0f / L : 0.f;
                uint32_t w[PER / 2];
#pragma unroll
                for (int e = 0; e < PER; e += 2) w[e / 2] = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
                bf16_t* dst = p.out + (int64_t)row * p.o_ld + hq * D + d0;
                if constexpr (PER == 8) *(uint4*)dst = make_uint4(w[0], w[1], w[2], w[3]);
                else *(uint2*)dst = make_uint2(w[0], w[1]);
                if (p.lse && d0 == 0) p.lse[(int64_t)row * p.heads + hq] = (use + __builtin_amdgcn_logf(L)) * 0.69314718055994530942f;
            } else {
                const int64_t at = ((int64_t)row * p.heads + hq) * p.slots + it.slot;
#pragma unroll
                for (int e = 0; e < PER; e += 4) *(float4*)(p.part_o + at * D + d0 + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
                if (d0 == 0) p.part_ml[at] = make_float2(M, L);
            }
        }
    }
    if constexpr (QT > 1) {
        request_next();
        st.store_q(sq);
    }
    __syncthreads();   // the next item's tiles go where these results were
}

template <int D, int QP, int QS>
__global__ __launch_bounds__(256, D == 64 || QP == 1 ? 3 : 2) void paged_attn_kernel(AttnParams p) {
    __shared__ __attribute__((aligned(16))) char lds[Lds<D>::BYTES];
    __shared__ __attribute__((aligned(16))) char sq[16 * QP * (2 * D + 16)];
    __shared__ float sm_m[WAVES][64], sm_l[WAVES][64];
    __shared__ Item items[BATCH];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int total = (p.plain ? p.n * p.tiles_s : *p.count) * p.kv_heads;
    const int grid = (int)gridDim.x - (p.plain && p.n_groups > 0);
    if ((int)blockIdx.x == grid) {
        check_groups(p);
        return;
    }
    Stream<D, QP> st(p, tid & 63);
    auto item_at = [&](int j) {
        Item it;
        const int* src = (const int*)&items[j];
        int* dst = (int*)&it;
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[e] = __builtin_amdgcn_readfirstlane(src[e]);
        return it;
    };
    for (int w0 = blockIdx.x; w0 < total; w0 += BATCH * grid) {
        const int n = min(BATCH, (total - w0 + grid - 1) / grid);
        __syncthreads();
        if (p.plain && tid < n) {
            const int x = (w0 + tid * grid) / p.kv_heads, i = x / p.tiles_s;
            const Entry e = entry_of(p, i, true);
            items[tid] = Item{e.r0, e.T * p.group, (x - i * p.tiles_s) * 16 * QS, e.seq, 0, min(e.len, CHUNK_MAX), e.len - e.T + 1, DIRECT};
        } else if (tid < n) {
            const uint4* src = (const uint4*)&p.items[(w0 + tid * grid) / p.kv_heads];
            uint4* dst = (uint4*)&items[tid];
            dst[0] = src[0];
            dst[1] = src[1];
        }
        __syncthreads();
        Item it = item_at(0);
        auto request = [&](const Item& x, int kvh, int ids) {
            st.begin(ids, kvh, x.k0, x.k1);
            st.load_q(x, kvh, x.limit == SHARED ? 16 * QP : 16 * QS);
            if (wave < (x.k1 - x.k0 + 31) >> 5) {
                st.load_k(wave);
                st.load_v(wave);
            }
        };
        request(it, w0 % p.kv_heads, st.page_numbers(it.seq, it.k0, it.k1));
        st.store_q(sq);
        __syncthreads();
        for (int j = 0; j < n; ++j) {
            const int w = w0 + j * grid, kvh = w % p.kv_heads, next_kvh = (w + grid) % p.kv_heads;
            const Item next = item_at(min(j + 1, n - 1));
            const int next_ids = st.page_numbers(next.seq, next.k0, next.k1);
            auto request_next = [&] { if (j + 1 < n) request(next, next_kvh, next_ids); };
            if (QP != QS && it.limit == SHARED) attend<D, QP, QP>(p, it, kvh, st, lds, sq, sm_m, sm_l, request_next);
            else attend<D, QS, QP>(p, it, kvh, st, lds, sq, sm_m, sm_l, request_next);
            it = next;
        }
    }
}

// Joins the parts of a row that has several: one wave per (row, head).
template <int D>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnParams p) {
    constexpr int PER = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= (int64_t)p.rows * p.heads) return;
    const int row = (int)(item / p.heads), hq = (int)(item - (int64_t)row * p.heads);
    const int parts = __builtin_amdgcn_readfirstlane(p.parts[row]), np = parts & 0xffff, n = np + (parts >> 16);
    if (n <= 1) return;   // written already, or not a row of this step
    auto slot_of = [&](int i) { return item * p.slots + (i < np ? i : p.chunks_p + i - np); };
    float M = -INFINITY, L = 0.f, acc[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = 0.f;
    // parts are requested several at a time, behind the last one the last again
    auto turn = [&](int i0, auto ahead, bool maximum_known) {
        constexpr int A = decltype(ahead)::value;
        float2 ml[A];
        float v[A][PER];
#pragma unroll
        for (int a = 0; a < A; ++a) {
            const int64_t at = slot_of(min(i0 + a, n - 1));
            ml[a] = p.part_ml[at];
#pragma unroll
            for (int e = 0; e < PER; ++e) v[a][e] = p.part_o[at * D + lane * PER + e];
        }
        if (!maximum_known) {
#pragma unroll
            for (int a = 0; a < A; ++a) M = fmaxf(M, ml[a].x);
        }
        const float use = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int a = 0; a < A; ++a) {
            const float f = i0 + a < n ? __builtin_amdgcn_exp2f(ml[a].x - use) : 0.f;
            L += ml[a].y * f;
#pragma unroll
            for (int e = 0; e < PER; ++e) acc[e] += v[a][e] * f;
        }
    };
    if (n <= 2) turn(0, std::integral_constant<int, 2>{}, false);
    else {
        for (int i = lane; i < n; i += 64) M = fmaxf(M, p.part_ml[slot_of(i)].x);
        M = wave_max(M);
        for (int i0 = 0; i0 < n; i0 += 8) turn(i0, std::integral_constant<int, 8>{}, true);
    }
    const float use = M == -INFINITY ? 0.f : M;
    const float inv = L > 0.f || L != L ? 1.0f / L : 0.f;
    bf16_t* dst = p.out + (int64_t)row * p.o_ld + hq * D + lane * PER;
    if constexpr (PER == 2) *(uint32_t*)dst = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    else *dst = f32_to_bf16(acc[0] * inv);
    if (p.lse && lane == 0) p.lse[item] = (use + __builtin_amdgcn_logf(L)) * 0.69314718055994530942f;
}

struct Plan {
    int qp, qs;           // 16-row tiles of a shared and of an own item
    int chunk, chunks_p, chunks_s, slots;
    int64_t items;        // at most
    int64_t at_parts, at_plan, at_items, at_ml, at_o, bytes;
    bool plain;
    int tiles_s;
};
int tiles_for(int64_t rows) { return rows <= 16 ? 1 : 2; }
Plan plan_for(const q3asr_kv_pages& c, const q3asr_attn_batch& b, int heads) {
    Plan r{};
    const int group = heads / c.kv_heads;
    r.qs = tiles_for((int64_t)b.max_rows * group);
    r.tiles_s = cdiv((int64_t)b.max_rows * group, 16 * r.qs);
    // A small step is all latency: whole sequences as items that fit the device at once, shared or not, in one launch.
    r.plain = b.max_len <= CHUNK_MAX && (int64_t)b.n * r.tiles_s * c.kv_heads <= PLAIN_ITEMS;
    const bool shares = !r.plain && b.n_groups > 0 && b.max_shared >= c.page_tokens;
    const int own = shares ? b.max_own : b.max_len;
    r.qp = shares ? std::max(r.qs, tiles_for((int64_t)b.max_group_rows * group)) : r.qs;
    // About three items per workgroup of a full device: fewer and larger items have less to join and less that begins and ends, more
    // and smaller ones spread a few long sequences over the device.
    const int64_t keys = (shares ? (int64_t)b.n_groups * b.max_shared : 0) + (int64_t)b.n * own;
    r.chunk = (int)std::min<int64_t>(CHUNK_MAX, std::max<int64_t>(128, (keys * c.kv_heads / (CUS * 9) + 127) / 128 * 128));
    r.chunks_p = shares ? cdiv(b.max_shared, r.chunk) : 0;
    r.chunks_s = std::max(1, cdiv(own, r.chunk));
    r.slots = r.chunks_p + r.chunks_s;
    r.items = (shares ? (int64_t)b.n_groups * r.chunks_p * cdiv((int64_t)b.max_group_rows * group, 16 * r.qp) : 0) +
              (int64_t)b.n * r.chunks_s * cdiv((int64_t)b.max_rows * group, 16 * r.qs);
    if (r.plain) {
        r.chunk = CHUNK_MAX;
        r.chunks_p = 0;
        r.chunks_s = r.slots = 1;
        r.qp = r.qs;
        r.items = (int64_t)b.n * r.tiles_s;
        return r;
    }
    auto round = [](int64_t x) { return (x + 255) & ~255ll; };
    r.at_parts = 256;
    r.at_plan = r.at_parts + round((int64_t)b.rows * 4);
    r.at_items = r.at_plan + (b.n > HELD || b.n_groups > HELD ? round((int64_t)b.n * (int64_t)sizeof(Entry) + (int64_t)b.n_groups * 4) : 0);
    r.at_ml = r.at_items + round(r.items * (int64_t)sizeof(Item));
    r.at_o = r.at_ml + (r.slots > 1 ? round((int64_t)b.rows * heads * r.slots * 8) : 0);
    r.bytes = r.at_o + (r.slots > 1 ? round((int64_t)b.rows * heads * r.slots * c.head_dim * 4) : 0);
    return r;
}

template <int D>
void launch_d(const AttnParams& p, const Plan& r, hipStream_t s) {
    const dim3 block(256);
    if (!r.plain) {
        hipLaunchKernelGGL(paged_attn_plan_kernel, dim3(1), dim3(PLAN), 0, s, p);
        HIP_CHECK(hipGetLastError());
    }
    const dim3 grid((int)std::min<int64_t>(r.items * p.kv_heads, CUS * (D == 64 || r.qp == 1 ? 3 : 2)) + (r.plain && p.n_groups > 0));
    switch (r.qp * 10 + r.qs) {
        case 11: hipLaunchKernelGGL((paged_attn_kernel<D, 1, 1>), grid, block, 0, s, p); break;
        case 21: hipLaunchKernelGGL((paged_attn_kernel<D, 2, 1>), grid, block, 0, s, p); break;
        default: hipLaunchKernelGGL((paged_attn_kernel<D, 2, 2>), grid, block, 0, s, p); break;
    }
    HIP_CHECK(hipGetLastError());
    if (p.slots > 1) {
        hipLaunchKernelGGL((paged_attn_join_kernel<D>), dim3(cdiv((int64_t)p.rows * p.heads, 4)), block, 0, s, p);
        HIP_CHECK(hipGetLastError());
    }
}

}  // namespace

int64_t paged_attention_workspace(const q3asr_kv_pages& c, const q3asr_attn_batch& b, int heads) { return plan_for(c, b, heads).bytes; }

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
    const bool shares = b.n_groups > 0 && b.max_shared >= c.page_tokens;
    p.n = b.n; p.rows = b.rows; p.n_groups = shares ? b.n_groups : 0;
    p.heads = heads; p.kv_heads = c.kv_heads; p.group = heads / c.kv_heads;
    p.max_rows = b.max_rows; p.max_group_rows = b.max_group_rows; p.max_len = b.max_len;
    p.max_own = shares ? b.max_own : b.max_len;
    p.max_shared = b.max_shared;
    p.scale_log2 = scale * 1.44269504088896340736f;
    p.chunk = r.chunk; p.chunks_p = r.chunks_p; p.chunks_s = r.chunks_s; p.slots = r.slots;
    p.rows_p = 16 * r.qp; p.rows_s = 16 * r.qs;
    char* ws = (char*)workspace;
    p.plain = r.plain;
    p.tiles_s = r.tiles_s;
    p.count = (int*)ws;
    p.plan_ws = ws + r.at_plan;
    p.parts = (int*)(ws + r.at_parts);
    p.items = (Item*)(ws + r.at_items);
    p.part_ml = (float2*)(ws + r.at_ml);
    p.part_o = (float*)(ws + r.at_o);
    Q3_REQUIRE(r.items * c.kv_heads < (1ll << 30) && r.slots < (1 << 15), "paged_attention: too much work for one call (smaller bounds in the batch make less)");
    ProfScope ps("paged_attn_kernel", 4.0 * b.rows * heads * (double)b.max_len * c.head_dim, s);
    if (c.head_dim == 64) launch_d<64>(p, r, s);
    else launch_d<128>(p, r, s);
}
