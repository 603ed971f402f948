// Attention over the paged KV cache for sequences that share prefixes (gfx950).
//
// o = sum_j p_j v_j, p = softmax_j(scale q . k_j).  The keys of a sequence are its group's shared pages and its own pages; all query
// rows that read a shared key -- of every sequence of the group, with all query heads of the KV head -- are columns of one matrix
// product, so that a shared key crosses HBM once per group.  Partial results (max, sum, weighted sum of values) are joined per
// row.  Both softmax statistics and the sums stay in fp32; a probability meets the matrix cores as the sum of two bf16 numbers, its
// rounding and the rounding of what that leaves (2^-16 of it is lost at most).  Rounded to bf16 once, they took the results' error against 64
// bits from 0.00166, which is their own rounding's, to 0.0021-0.0025; the second product costs 40.1 -> 42.0 us where query rows are
// many (12 x 7 scored) and nothing that shows where HBM bounds (96 x 5: 120.5, 120.7; 16 x 8: 149.0, 149.3).
//
// HBM-bound: 2 * head_dim * 2 bytes per key and KV head against 16 * QT columns.  A wave works on tiles of 32 keys: the K rows,
// loaded whole, become MFMA A fragments of S^T = K Q^T through an LDS tile of the wave's own; the exponentiated scores are as
// they stand the B fragment of O^T = V^T P^T, whose A fragments are transposing reads of the V rows in the same LDS tile.  The
// next tile's rows are requested as soon as this one's have left their registers.
//
//   plain   few rows: a workgroup per sequence and KV head, its eight waves taking tiles in turn; one launch, nothing shared
//   stream  the tiles of all sequences and groups in one row, cut into equal parts, one per wave of a full device: no wave waits for
//           another, and each has a tile in flight all the time.  Where a wave goes over to other rows counts like a tile.  Two
//           launches: the waves, which find out first where every sequence's tiles begin, and the join of what was cut.
// The stream takes 111 us for 96 groups of 5 after 405 tokens (8 KV heads of 128, 5.2 TB/s), 139 for 16 groups of 8 after 16 000 (5.9), 31
// for 12 groups of 7 x up to 24 rows after 1111 (14 heads of 64, compute and parts); the join 5-8; plain 7.7 for 4 sequences of 406 keys.
// Measured against 4-wave work items of up to 1024 keys, sorted by size: rounding to four tiles and joining cost 1.2 to 1.4 times
// the mean load there.
#include "paged.h"
#include "prof.h"
#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;

namespace {

constexpr int WAVES = 4, PLAN = 1024, CUS = 256;
constexpr int STREAM_WAVES = CUS * 2 * WAVES;     // two workgroups per CU
constexpr int PLAIN_ITEMS = 512, PLAIN_KEYS = 1024;

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

// Query rows that read the same keys: row r of M is row r0 + r / group of the step, head kvh * group + r % group.  They read keys
// [k0, k1) of the pages of sequence seq, row r those below limit + r / group (SHARED: all of them).
struct __attribute__((aligned(16))) Segment {
    int r0, M, seq, k0, k1, limit;
    int start;    // place in the row of all tiles: stream h * query tiles + q (KV head h, query tile q) takes ntiles + 1 places from
                  // start + stream * (ntiles + 1) on, one for its beginning and one per tile
    int tag;      // 2 * the entry of the batch that errors name, a group's first sequence for its own segment; + 1: its rows read nothing else
};
constexpr int SHARED = 0x7fffffff;
// Where a row's parts are: tiles of its group's and of its own segment (0: none), their starts, first rows and query tiles.
struct __attribute__((aligned(16))) RowParts {
    int start[2], tiles[2], r0[2], streams[2];
    int known, pad[3];
};
struct __attribute__((aligned(16))) Total {
    int places, per, segments, pad;   // per: places of a wave
};

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
    float scale_log2;                          // positive; a negative scale's sign is taken into the queries
    uint32_t flip;
    int shift_q;                               // query rows of a wave: 16 * QT = 1 << shift_q
    int tiles_q;                               // plain: query tiles of a sequence
    int per_min, slots_p, slots;               // parts of a row at most: of its group's segment first
    Total* total;
    void* plan_ws;                             // of a plan that does not fit LDS, and its segments
    Segment* segments;
    RowParts* parts;                           // [rows]
    float2* part_ml;                           // [rows][heads][slots]: maximum (base 2), sum
    float* part_o;                             // [rows][heads][slots][D]
};

struct Entry {             // a sequence of the step
    int seq, r0, T, len;
    bool ok;
};
__device__ __forceinline__ Entry entry_of(const AttnParams& p, int i, int seq, int a, int b, bool report) {
    Entry e;
    e.seq = seq;
    const bool in = (unsigned)e.seq < (unsigned)p.max_seqs, ok = in && a >= 0 && b >= a && b <= p.rows && b - a <= p.max_rows;
    const bool none = e.seq == -1 && a == b;   // stands for no sequence: shares nothing, has no rows
    e.r0 = ok ? a : 0;
    e.T = ok ? b - a : 0;
    e.len = ok ? p.lens[e.seq] : 0;
    e.ok = ok && e.len >= 0 && e.len <= p.max_len;
    if (!e.ok) {
        if (report && !none) pages_error(p.status, in ? Q3ASR_PAGES_BAD_BATCH : Q3ASR_PAGES_BAD_INDEX, i);
        e.seq = in ? e.seq : 0;
        e.len = min(max(e.len, 0), p.max_len);
    }
    return e;
}
__device__ __forceinline__ Entry entry_of(const AttnParams& p, int i, bool report) {
    return entry_of(p, i, p.seqs[i], p.cu_rows[i], p.cu_rows[i + 1], report);
}

// ---- plan ----
// Where every segment's tiles begin, from the lengths.  Up to HELD groups and sequences every workgroup finds out for itself, in LDS
// (two dependent loads per sequence, its number and its length, and no launch of its own); beyond that one workgroup does it
// for all, in the workspace.  tell: errors are reported and the rows' parts written down, by one workgroup of all.
constexpr int HELD = 1024;   // as a launch of its own the plan costs 6 us, in front of every wave 4
struct PlanMemory {
    Entry* entry;            // [n]
    int *from, *lead;        // [n_groups] tokens that a group shares, and its first entry that stands for a sequence
    int *cu, *rows;          // [n_groups + 1], [n + 1]: of the batch
    static constexpr int64_t bytes(int64_t n, int64_t groups) { return n * (int64_t)sizeof(Entry) + (3 * groups + n + 2) * 4; }
    __device__ PlanMemory(void* at, int n, int groups) {
        entry = (Entry*)at;
        from = (int*)(entry + n);
        lead = from + groups;
        cu = lead + groups;
        rows = cu + groups + 1;
    }
};
// The batch's entries, and what its groups share.  All threads of the workgroup; ends behind a barrier.  False: cu_rows or cu_groups goes down
// somewhere, so that rows or entries may count several times, and there may be more tiles than 32 bits count.
template <int THREADS>
__device__ __forceinline__ bool read_batch(const AttnParams& p, const PlanMemory& mem, bool tell) {
    const int tid = threadIdx.x, lane = tid & 63;
    Entry* const entry = mem.entry;
    int *const from = mem.from, *const cu = mem.cu, *const cu_rows = mem.rows;
    const int last_g = p.n_groups - 1, last = p.n - 1;
    bool down = false;
    for (int i = tid; i <= p.n; i += THREADS) {   // there are no more groups than entries
        // all that does not depend on another load at once
        const int seq = p.seqs[min(i, last)], a = p.cu_rows[min(i, last)], b = p.cu_rows[min(i, last) + 1];
        const int group = last_g < 0 ? 0 : p.cu_groups[min(i, last_g + 1)], shared = last_g < 0 ? 0 : p.shared[min(i, last_g)];
        __builtin_amdgcn_sched_barrier(0);
        if (i <= last) {
            entry[i] = entry_of(p, i, seq, a, b, tell);
            down |= b < a;
            cu_rows[i] = a;
            if (i == last) cu_rows[i + 1] = b;
        }
        if (i <= last_g) from[i] = shared;
        if (last_g >= 0 && i <= last_g + 1) cu[i] = group;
    }
    __syncthreads();
    for (int g0 = 0; g0 < p.n_groups; g0 += THREADS) {
        const int g = g0 + tid;
        int i0 = 0, i1 = 0;
        if (g < p.n_groups) {
            i0 = cu[g];
            i1 = cu[g + 1];
            down |= i1 < i0;
            if (i0 < 0 || i1 < i0 || i1 > p.n) {
                if (tell) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, min(max(i0, 0), last));   // where the group would begin
                i0 = i1 = 0;
            }
        }
        // Entries that stand for no sequence (-1: hypotheses that have ended) may come first: a thread looks past a few, its wave past more.
        int lead = i0;
        const int near = min(i1, i0 + 8);
        while (lead < near && !entry[lead].ok) ++lead;
        for (unsigned long long open = __ballot(lead == near && near < i1); open; open &= open - 1) {
            const int who = __ffsll(open) - 1, end = __shfl(i1, who, 64);
            int at = __shfl(lead, who, 64);
            unsigned long long found = 0;
            while (at < end) {
                found = __ballot(at + lane < end && entry[min(at + lane, last)].ok);
                if (found) break;
                at += 64;
            }
            if (lane == who) lead = found ? at + __ffsll(found) - 1 : end;
        }
        if (g >= p.n_groups) continue;
        const int shared = from[g];
        from[g] = 0;
        mem.lead[g] = lead;
        if (lead < i1) {   // a group without sequences shares nothing
            const Entry first = entry[lead];
            const int end = cu_rows[i1];
            const bool fits = end >= first.r0 && end <= p.rows && end - first.r0 <= p.max_group_rows;
            if (shared > p.max_shared || !fits) if (tell) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, lead);
            if (fits) from[g] = max(0, min(min(shared, p.max_shared), first.len - first.T)) >> p.pt_shift << p.pt_shift;
        }
    }
    return !__syncthreads_or(down);
}
// Behind read_batch: the group of entry i (-1: none), and how many of the entry's first keys are read by the group.
struct Member {
    int group, behind;
};
__device__ __forceinline__ Member member_of(const AttnParams& p, const PlanMemory& mem, int i, bool tell) {
    Member m{-1, 0};
    const Entry e = mem.entry[i];
    if (p.n_groups > 0) {
        int lo = 0, hi = p.n_groups;   // the last group that begins at or before entry i
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (mem.cu[mid] <= i) lo = mid;
            else hi = mid;
        }
        const int i0 = mem.cu[lo], i1 = mem.cu[lo + 1];
        if (i0 >= 0 && i >= i0 && i < i1 && i1 <= p.n) m = Member{lo, mem.from[lo]};
        else if (tell) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, i);
    }
    // keys behind max_own would be left out
    if (tell && e.ok && (m.behind > max(0, e.len - e.T) || e.len - m.behind > p.max_own)) pages_error(p.status, Q3ASR_PAGES_BAD_BATCH, i);
    return m;
}
// scan: a word per wave; segments: [n_groups + n].
template <int THREADS>
__device__ __forceinline__ Total plan_segments(const AttnParams& p, const PlanMemory& mem, int* scan, Segment* segments, bool tell) {
    const int tid = threadIdx.x;
    if (tell)
        for (int r = tid; r < p.rows; r += THREADS) p.parts[r].known = 0;
    const bool rising = read_batch<THREADS>(p, mem, tell);
    // segments: the groups', then the sequences'
    const int all = p.n_groups + p.n;
    int carry = 0;
    for (int w0 = 0; w0 < all; w0 += THREADS) {
        const int w = w0 + tid;
        Segment sg{};
        int g = -1, count = 0;
        Entry e{};
        if (w < p.n_groups) {
            if (mem.from[w] > 0) {
                const Entry first = mem.entry[mem.lead[w]];
                sg = Segment{first.r0, (mem.rows[mem.cu[w + 1]] - first.r0) * p.group, first.seq, 0, mem.from[w], SHARED, 0, 2 * mem.lead[w]};
            }
        } else if (w < all) {
            const int i = w - p.n_groups;
            e = mem.entry[i];
            const Member m = member_of(p, mem, i, tell);
            g = m.group;
            sg = Segment{e.r0, e.T * p.group, e.seq, m.behind, m.behind + min(max(0, e.len - m.behind), p.max_own), e.len - e.T + 1, 0, 2 * i + (m.behind == 0)};
        }
        const int tiles = (sg.k1 - sg.k0 + 31) >> 5;
        const int streams = (sg.M + (1 << p.shift_q) - 1) >> p.shift_q;
        count = tiles > 0 ? (tiles + 1) * streams * p.kv_heads : 0;
        // exclusive prefix sum
        const int lane = tid & 63, wave = tid >> 6;
        int x = count;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(x, o, 64);
            if (lane >= o) x += t;
        }
        if (lane == 63) scan[wave] = x;
        __syncthreads();
        int before = carry;
        for (int v = 0; v < THREADS / 64; ++v) {
            before += v < wave ? scan[v] : 0;
            carry += scan[v];
        }
        sg.start = before + x - count;
        if (w < all) segments[w] = sg;
        __syncthreads();   // scan is written again; the groups' segments are read below
        if (tell && rising && w >= p.n_groups && w < all) {
            RowParts rp{};
            if (g >= 0 && mem.from[g] > 0) {
                const Segment& sh = segments[g];
                rp.start[0] = sh.start;
                rp.tiles[0] = (sh.k1 - sh.k0 + 31) >> 5;
                rp.r0[0] = sh.r0;
                rp.streams[0] = (sh.M + (1 << p.shift_q) - 1) >> p.shift_q;
            }
            rp.start[1] = sg.start;
            rp.tiles[1] = tiles;
            rp.r0[1] = sg.r0;
            rp.streams[1] = streams;
            rp.known = 1;
            for (int t = 0; t < e.T; ++t) p.parts[e.r0 + t] = rp;
        }
    }
    if (!rising) carry = 0;   // reported; no row is computed
    const Total total{carry, max(p.per_min, (carry + STREAM_WAVES - 1) / STREAM_WAVES), all, 0};
    if (tell && tid == 0) *p.total = total;
    return total;
}
__global__ __launch_bounds__(PLAN) void paged_attn_plan_kernel(AttnParams p) {
    __shared__ int scan[PLAN / 64];
    plan_segments<PLAN>(p, PlanMemory(p.plan_ws, p.n, p.n_groups), scan, p.segments, true);
}

// ---- a wave's work ----
template <int D>
struct Rows {
    static constexpr int KROW = 2 * D + 16, VROW = 2 * D + 32;   // padded: fragment and transposing reads meet all banks
    static constexpr int TILE = 32 * VROW;
};

// ONCE: no key is read by several waves, so its rows need not stay in a cache.  A step whose loads say so takes 152 us where others take 171
// (256 sequences of 900 tokens, 8 KV heads of 128); where query tiles read the same keys it takes 66 against 60 (three of them: 12 x 7 x 24
// rows after 1111 tokens, 14 heads of 64) and 93 against 61 (17: 2 x 14 x 19 rows after 3584, 16 / 8 heads of 128).
template <int D, int QT, bool ONCE>
struct Wave {
    static constexpr int NKS = D / 32, NDT = D / 16, LPR = D / 8, RPI = 64 / LPR, IV = 16 / RPI, PAIR = QT < 2 ? 1 : 2;
    static constexpr int KROW = Rows<D>::KROW, VROW = Rows<D>::VROW;
    const AttnParams& p;
    const int lane, li, lg;
    char* const tile;             // the wave's LDS
    Frag kf[2][IV], vf[2][IV];    // 32 keys, as rows
    Frag qf[QT][NKS];             // queries as B fragments: lane (li, lg) holds values 32 ks + 8 lg .. of query 16 qt + li
    int limit[QT];                // the lane's queries see keys below
    int lowest;                   // keys below it are seen by all of them
    int active;                   // groups of 16 queries that there are
    // Weights are powers of two above m, a bound that no score so far exceeds by more than SLACK: it is only moved, and the sums
    // with it, when one does.  So weights are below 2^SLACK; fp32 sums and relative roundings are as good there.
    static constexpr float SLACK = 8.f;
    float m[QT], less[QT], l[QT];   // less: -m, 0 while there is no m; l: of this lane's keys only, until the end
    f32x4 o[QT][NDT];             // lane (li, lg) holds values 16 dt + 4 lg .. of query 16 qt + li
    int ids, id_base;             // page numbers of 64 times 16 keys from key id_base on, one per lane
    __device__ Wave(const AttnParams& p_, char* tile_) : p(p_), lane(threadIdx.x & 63), li(threadIdx.x & 15), lg((threadIdx.x & 63) >> 4), tile(tile_) {}

    __device__ void page_numbers(const Segment& sg, int base) {
        id_base = base;
        const int key = min(base + 16 * lane, sg.k1 - 1);
        ids = p.table[(int64_t)sg.seq * p.max_seq_pages + (key >> p.pt_shift)];
        if ((unsigned)ids >= (unsigned)p.pages) {
            pages_error(p.status, Q3ASR_PAGES_BAD_INDEX, sg.tag >> 1);
            ids = 0;
        }
    }
    __device__ int64_t base_of(int64_t head, int key) const {   // 16 keys of a page
        const int64_t page = __builtin_amdgcn_readlane(ids, (key - id_base) >> 4);
        return page * p.page_stride + head + (int64_t)(key & ((1 << p.pt_shift) - 1)) * D;
    }
    static __device__ __forceinline__ bf16x8 row(const bf16x8* at) {
        if constexpr (ONCE) return __builtin_nontemporal_load(at);
        else return *at;
    }
    // Keys behind the last one are read from its row, so that they cost no memory traffic.
    __device__ void load(const bf16_t* pool, Frag (&x)[2][IV], int64_t head, int kv0, int k1) const {
        if (kv0 + 32 <= k1) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bf16_t* src = pool + base_of(head, kv0 + 16 * h) + (lane / LPR) * D + 8 * (lane % LPR);
#pragma unroll
                for (int i = 0; i < IV; ++i) x[h][i].v = row((const bf16x8*)(src + i * RPI * D));
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = min(kv0 + 16 * h, (k1 - 1) & ~15);
                const bf16_t* src = pool + base_of(head, key) + 8 * (lane % LPR);
#pragma unroll
                for (int i = 0; i < IV; ++i)
                    x[h][i].v = row((const bf16x8*)(src + min(lane / LPR + i * RPI, k1 - 1 - key) * D));
            }
        }
    }
    __device__ void queries(const Segment& sg, int first, int kvh) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            const int r = first + 16 * qt + li;
            const bool ok = r < sg.M;
            const int tok = (ok ? r : 0) / p.group;
            limit[qt] = !ok ? 0 : sg.limit == SHARED ? sg.k1 : min(sg.k1, sg.limit + tok);
            const bf16_t* src = p.q + (int64_t)(sg.r0 + tok) * p.q_ld + (kvh * p.group + (ok ? r - tok * p.group : 0)) * D + 8 * lg;
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                const uint4 u = *(const uint4*)(src + 32 * ks);
                qf[qt][ks].u = make_uint4(u.x ^ p.flip, u.y ^ p.flip, u.z ^ p.flip, u.w ^ p.flip);
            }
            m[qt] = -INFINITY;
            less[qt] = l[qt] = 0.f;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[qt][dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
        lowest = min(sg.k1, sg.limit);
        active = (sg.M - first + 15) >> 4;
    }
    // The tile of keys kv0 .. whose rows are in kf and vf; next_k and next_v request the next tile's once these are free.
    template <class NK, class NV>
    __device__ void step(int kv0, int k1, NK next_k, NV next_v) {
        char* const kw = tile + (lane / LPR) * KROW + 16 * (lane % LPR);
        char* const vw = tile + (lane / LPR) * VROW + 16 * (lane % LPR);
        const char* const kr = tile + li * KROW + 16 * lg;
        // transposing reads: per 16 lanes a block of 4 keys x 16 dims, lane 4 a + b addresses key a, dims 4 b .. 4 b + 3
        const char* const vr = tile + (4 * lg + (li >> 2)) * VROW + (li & 3) * 8;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < IV; ++i) *(uint4*)(kw + (16 * h + i * RPI) * KROW) = kf[h][i].u;
        next_k();
        wave_lds_fence();
        Frag ka[2][NKS];   // K rows as A fragments: lane (li, lg) reads values 32 ks + 8 lg .. of key li
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) ka[h][ks].u = *(const uint4*)(kr + 16 * h * KROW + 64 * ks);
        Frag pf[QT], pr[QT];   // the weights rounded to bf16, and what that left over
#pragma unroll
        for (int g = 0; g < QT; g += PAIR) {
            if (g > 0 && g >= active) break;   // wave-uniform
            f32x4 s[PAIR][2];
            float top[PAIR];
#pragma unroll
            for (int i = 0; i < PAIR; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    s[i][h] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < NKS; ++ks) s[i][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[h][ks].v, qf[g + i][ks].v, s[i][h], 0, 0, 0);
                }
            if (kv0 + 32 > lowest) {   // wave-uniform
#pragma unroll
                for (int i = 0; i < PAIR; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (kv0 + 16 * (j >> 2) + 4 * lg + (j & 3) >= limit[g + i]) s[i][j >> 2][j & 3] = -INFINITY;
            }
            bool beyond = false;
#pragma unroll
            for (int i = 0; i < PAIR; ++i) {
                top[i] = s[i][0][0];
#pragma unroll
                for (int j = 1; j < 8; ++j) top[i] = __builtin_elementwise_maximum(top[i], s[i][j >> 2][j & 3]);   // a NaN stays: the row is NaN
                beyond |= top[i] * p.scale_log2 > m[g + i] + SLACK;
            }
            if (__builtin_amdgcn_ballot_w64(beyond) != 0) {
#pragma unroll
                for (int i = 0; i < PAIR; ++i) {
                    const int qt = g + i;
                    const float m_new = fmaxf(m[qt], rows_max(top[i]) * p.scale_log2);
                    const float use = m_new == -INFINITY ? 0.f : m_new;   // no key seen yet
                    const float alpha = __builtin_amdgcn_exp2f(m[qt] - use);
                    m[qt] = m_new;
                    less[qt] = -use;
                    l[qt] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < NDT; ++dt) o[qt][dt] *= alpha;
                }
            }
#pragma unroll
            for (int i = 0; i < PAIR; ++i) {
                const int qt = g + i;
                float pe[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    pe[j] = __builtin_amdgcn_exp2f(fmaf(s[i][j >> 2][j & 3], p.scale_log2, less[qt]));
                    l[qt] += pe[j];
                }
                uint32_t whole[4], rest[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    whole[j] = pack_bf16x2(pe[2 * j], pe[2 * j + 1]);
                    rest[j] = pack_bf16x2(pe[2 * j] - __uint_as_float(whole[j] << 16), pe[2 * j + 1] - __uint_as_float(whole[j] & 0xffff0000u));
                }
                pf[qt].u = make_uint4(whole[0], whole[1], whole[2], whole[3]);
                pr[qt].u = make_uint4(rest[0], rest[1], rest[2], rest[3]);
            }
        }
        __builtin_amdgcn_wave_barrier();   // the V rows go where the K rows were
        if (kv0 + 32 > k1) {
            // what lies behind the last key may be anything: a NaN there would survive its zero weight
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < IV; ++i)
                    if (kv0 + 16 * h + i * RPI + lane / LPR >= k1) vf[h][i].u = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < IV; ++i) *(uint4*)(vw + (16 * h + i * RPI) * VROW) = vf[h][i].u;
        next_v();
        wave_lds_fence();
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            union { s16x4 v; uint2 u; } lo, hi;   // keys 4 lg .. 4 lg + 3 and 16 + 4 lg .. of dim 16 dt + li
            lo.v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vr + 32 * dt));
            hi.v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vr + 16 * VROW + 32 * dt));
            Frag va;
            va.h[0] = lo.u;
            va.h[1] = hi.u;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                if (qt >= PAIR && qt / PAIR * PAIR >= active) break;
                o[qt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va.v, pr[qt].v, o[qt][dt], 0, 0, 0);
                o[qt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va.v, pf[qt].v, o[qt][dt], 0, 0, 0);
            }
        }
        __builtin_amdgcn_wave_barrier();   // the next tile's rows are written after these reads
    }
};

__device__ __forceinline__ float lse_of(float m, float l) { return (m + __builtin_amdgcn_logf(l)) * 0.69314718055994530942f; }
__device__ __forceinline__ float inverse_of(float l) { return l > 0.f || l != l ? 1.0f / l : 0.f; }   // no keys: zeros

// ---- stream ----
template <int D, int QT, bool ONCE, bool PLANNED>
__global__ __launch_bounds__(256, 2) void paged_attn_stream_kernel(AttnParams p) {
    constexpr int PLAN_BYTES = PLANNED ? 0 : (int)PlanMemory::bytes(HELD, HELD) + WAVES * 4, TILES = WAVES * Rows<D>::TILE;
    __shared__ __attribute__((aligned(16))) char lds[PLAN_BYTES > TILES ? PLAN_BYTES : TILES];
    __shared__ Segment held[PLANNED ? 1 : HELD];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const Segment* const segments = PLANNED ? p.segments : held;
    Total total;
    if constexpr (PLANNED) total = *p.total;
    else {
        const PlanMemory mem(lds, HELD, HELD);
        total = plan_segments<256>(p, mem, mem.rows + HELD + 1, held, blockIdx.x == 0);
        __syncthreads();   // the tiles go where the plan was made
    }
    int share = blockIdx.x;
    if constexpr (!ONCE) {   // neighbouring shares go to one XCD, in whose L2 all query tiles but the first find their keys
        const int64_t used = (((int64_t)total.places + total.per - 1) / total.per + WAVES - 1) / WAVES;
        const int chunk = (int)((used + 7) >> 3);
        if ((int)(blockIdx.x >> 3) >= chunk) return;
        share = (blockIdx.x & 7) * chunk + (blockIdx.x >> 3);
    }
    const int64_t begin = (int64_t)(share * WAVES + wave) * total.per;   // may lie behind what 32 bits hold, places do not
    if (begin >= total.places) return;
    int pos = (int)begin;
    const int end = (int)min((int64_t)total.places, begin + total.per);
    Wave<D, QT, ONCE> w(p, lds + wave * Rows<D>::TILE);

    // the last segment that begins at or before pos: 64 probes at a time
    int lo = 0, hi = total.segments;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) >> 6, at = lo + lane * step;
        const unsigned long long before = __ballot(at < hi && segments[at].start <= pos);
        lo += (__popcll(before) - 1) * step;
        hi = min(hi, lo + step);
    }
    int which = lo;
    Segment sg;
    int ntiles, rel, kvh, first;   // rel: tile within the stream
    auto fetch = [&] {             // wave-uniform
        const int* src = (const int*)&segments[which];
        int* dst = (int*)&sg;
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[e] = __builtin_amdgcn_readfirstlane(src[e]);
        ntiles = (sg.k1 - sg.k0 + 31) >> 5;
    };
    fetch();
    {
        // segments without tiles are never the last one before a place
        const int at = pos - sg.start, stream = at / (ntiles + 1), streams = (sg.M + 16 * QT - 1) / (16 * QT);
        rel = at - stream * (ntiles + 1) - 1;
        kvh = stream / streams;
        first = (stream - kvh * streams) * (16 * QT);
        if (rel < 0) {   // the place of a beginning; a wave has two places at least, so the tile behind it is its own
            rel = 0;
            ++pos;
        }
    }
    int64_t head = (int64_t)kvh * p.head_stride;
    auto window = [&] { w.page_numbers(sg, sg.k0 + 32 * rel); };
    window();
    w.load(p.K, w.kf, head, sg.k0 + 32 * rel, sg.k1);
    w.load(p.V, w.vf, head, sg.k0 + 32 * rel, sg.k1);
    w.queries(sg, first, kvh);

    // A tile, and the request of the next one.  That is unconditional where there is one (the wave's last tile has code of its own): a
    // load behind a branch would make the waits count as if it had not been issued.
    auto tile = [&](auto is_last) {
        constexpr bool LAST = decltype(is_last)::value;
        const Segment now = sg;
        const int now_kvh = kvh, now_first = first, now_tiles = ntiles, kv0 = sg.k0 + 32 * rel;
        const bool over = rel + 1 == ntiles;
        auto next_k = [&] {
            if constexpr (LAST) return;
            if (!over) {
                ++rel;
                if (sg.k0 + 32 * rel - w.id_base >= 1024) window();
            } else {
                rel = 0;
                first += 16 * QT;
                bool other = false;
                if (first >= sg.M) {
                    first = 0;
                    if (++kvh == p.kv_heads) {
                        kvh = 0;
                        other = true;
                        do {
                            ++which;
                            fetch();
                        } while (ntiles == 0 || sg.M == 0);   // there is a tile left, so there is such a segment
                    }
                }
                if (other || w.id_base != sg.k0) window();
                head = (int64_t)kvh * p.head_stride;
            }
            w.load(p.K, w.kf, head, sg.k0 + 32 * rel, sg.k1);
        };
        auto next_v = [&] {
            if constexpr (!LAST) w.load(p.V, w.vf, head, sg.k0 + 32 * rel, sg.k1);
        };
        w.step(kv0, now.k1, next_k, next_v);
        if (over || LAST) {
            // a part, or all there is for these rows
            const int streams = (now.M + 16 * QT - 1) / (16 * QT);
            const int tile0 = now.start + (now_kvh * streams + now_first / (16 * QT)) * (now_tiles + 1) + 1;   // the first tile's place
            const int before = tile0 / total.per, piece = pos / total.per - before;
            const bool direct = (now.tag & 1) && (tile0 + now_tiles - 1) / total.per == before;
            const int slot = (now.limit == SHARED ? 0 : p.slots_p) + piece;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                const int r = now_first + 16 * qt + w.li;
                const float L = rows_sum(w.l[qt]);
                if (r < now.M) {
                    const int tok = r / p.group, row = now.r0 + tok, hq = now_kvh * p.group + r - tok * p.group;
                    if (direct) {
                        const float inv = inverse_of(L);
                        bf16_t* dst = p.out + (int64_t)row * p.o_ld + hq * D + 4 * w.lg;
#pragma unroll
                        for (int dt = 0; dt < D / 16; ++dt)
                            *(uint2*)(dst + 16 * dt) = make_uint2(pack_bf16x2(w.o[qt][dt][0] * inv, w.o[qt][dt][1] * inv),
                                                                  pack_bf16x2(w.o[qt][dt][2] * inv, w.o[qt][dt][3] * inv));
                        if (p.lse && w.lg == 0) p.lse[(int64_t)row * p.heads + hq] = lse_of(w.m[qt] == -INFINITY ? 0.f : w.m[qt], L);
                    } else {
                        const int64_t at = ((int64_t)row * p.heads + hq) * p.slots + slot;
#pragma unroll
                        for (int dt = 0; dt < D / 16; ++dt) *(f32x4*)(p.part_o + at * D + 16 * dt + 4 * w.lg) = w.o[qt][dt];
                        if (w.lg == 0) p.part_ml[at] = make_float2(w.m[qt], L);
                    }
                }
            }
            if constexpr (!LAST) w.queries(sg, first, kvh);
        }
    };
    for (;;) {
        const int next = pos + (rel + 1 == ntiles ? 2 : 1);
        if (next >= end) break;
        tile(std::false_type{});
        pos = next;
    }
    tile(std::true_type{});
}

// Joins the parts of a row that has several, and writes rows without keys: D / 2 lanes per (row, head), or (SPREAD) a workgroup, whose
// teams of D / 2 lanes take its parts in turn.
template <int D, bool SPREAD>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnParams p) {
    constexpr int LANES = D / 2, TEAMS = 256 / LANES;
    const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES, row = blockIdx.x, hq = SPREAD ? blockIdx.y : blockIdx.y * TEAMS + team;
    const RowParts rp = p.parts[row];
    const int per = p.total->per;
    if (hq >= p.heads || !rp.known) return;
    const int64_t item = (int64_t)row * p.heads + hq;
    const int kvh = hq / p.group;
    // quotients of places by the places of a wave: a first guess in 64 bits is off by one at most
    const double inverse = 1.0 / per;
    auto wave_of = [&](int place) {
        int q = (int)(place * inverse);
        const int rest = place - q * per;
        return rest < 0 ? q - 1 : rest >= per ? q + 1 : q;
    };
    int count[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int r = (row - rp.r0[k]) * p.group + hq - kvh * p.group;
        const int begin = rp.start[k] + (kvh * rp.streams[k] + (r >> p.shift_q)) * (rp.tiles[k] + 1) + 1;
        count[k] = rp.tiles[k] > 0 ? wave_of(begin + rp.tiles[k] - 1) - wave_of(begin) + 1 : 0;
    }
    const int np = min(count[0], p.slots_p), n = np + min(count[1], p.slots - p.slots_p);
    if (np == 0 && n == 1) return;   // written already
    auto slot_of = [&](int i) { return item * p.slots + (i < np ? i : p.slots_p + i - np); };
    float M = -INFINITY, L = 0.f, a0 = 0.f, a1 = 0.f;
    // parts are requested several at a time, behind the last one the last again
    auto turn = [&](int i0, auto ahead, bool maximum_known) {
        constexpr int A = decltype(ahead)::value;
        float2 ml[A], v[A];
#pragma unroll
        for (int a = 0; a < A; ++a) {
            const int64_t at = slot_of(min(i0 + a, n - 1));
            ml[a] = p.part_ml[at];
            v[a] = *(const float2*)(p.part_o + at * D + lane * 2);
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
            a0 += v[a].x * f;
            a1 += v[a].y * f;
        }
    };
    if constexpr (SPREAD) {
        __shared__ float2 ml_of[TEAMS], sum_of[TEAMS][LANES];
        for (int i0 = team; i0 < n; i0 += 8 * TEAMS) {   // eight parts requested at a time, behind the last one the last again
            float2 ml[8], v[8];
#pragma unroll
            for (int a = 0; a < 8; ++a) {
                const int64_t at = slot_of(min(i0 + a * TEAMS, n - 1));
                ml[a] = p.part_ml[at];
                v[a] = *(const float2*)(p.part_o + at * D + lane * 2);
            }
            float top = M;
#pragma unroll
            for (int a = 0; a < 8; ++a) top = fmaxf(top, ml[a].x);
            const float use = top == -INFINITY ? 0.f : top, before = __builtin_amdgcn_exp2f(M - use);
            M = top;
            L *= before;
            a0 *= before;
            a1 *= before;
#pragma unroll
            for (int a = 0; a < 8; ++a) {
                const float f = i0 + a * TEAMS < n ? __builtin_amdgcn_exp2f(ml[a].x - use) : 0.f;
                L += ml[a].y * f;
                a0 += v[a].x * f;
                a1 += v[a].y * f;
            }
        }
        if (lane == 0) ml_of[team] = make_float2(M, L);
        sum_of[team][lane] = make_float2(a0, a1);
        __syncthreads();
        if (team > 0) return;
#pragma unroll
        for (int t = 0; t < TEAMS; ++t) M = fmaxf(M, ml_of[t].x);
        const float use = M == -INFINITY ? 0.f : M;
        L = a0 = a1 = 0.f;
#pragma unroll
        for (int t = 0; t < TEAMS; ++t) {
            const float f = __builtin_amdgcn_exp2f(ml_of[t].x - use);
            L += ml_of[t].y * f;
            a0 += sum_of[t][lane].x * f;
            a1 += sum_of[t][lane].y * f;
        }
    } else if (n > 8) {
        for (int i = lane; i < n; i += LANES) M = fmaxf(M, p.part_ml[slot_of(i)].x);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, LANES));
        for (int i0 = 0; i0 < n; i0 += 8) turn(i0, std::integral_constant<int, 8>{}, true);
    } else if (n > 4) {
        turn(0, std::integral_constant<int, 8>{}, false);
    } else if (n > 2) {
        turn(0, std::integral_constant<int, 4>{}, false);
    } else if (n > 0) {
        turn(0, std::integral_constant<int, 2>{}, false);
    }
    const float inv = inverse_of(L);
    *(uint32_t*)(p.out + (int64_t)row * p.o_ld + hq * D + lane * 2) = pack_bf16x2(a0 * inv, a1 * inv);
    if (p.lse && lane == 0) p.lse[item] = lse_of(M == -INFINITY ? 0.f : M, L);
}

// ---- plain ----
constexpr int PLAIN_WAVES = 8;
template <int D, int QT>
__global__ __launch_bounds__(64 * PLAIN_WAVES) void paged_attn_plain_kernel(AttnParams p) {
    constexpr int WAVES = PLAIN_WAVES, OROW = D + 4, PER = D / 32;
    __shared__ __attribute__((aligned(16))) char lds[WAVES * Rows<D>::TILE];
    __shared__ float sm_m[WAVES][16], sm_l[WAVES][16];
    static_assert(WAVES * Rows<D>::TILE >= WAVES * 16 * OROW * 4, "the waves' results fit where their tiles were");
    static_assert(WAVES * Rows<D>::TILE >= PlanMemory::bytes(HELD, HELD) && HELD >= 2 * PLAIN_ITEMS, "so does the batch");
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % p.kv_heads, x = blockIdx.x / p.kv_heads, i = x / p.tiles_q;
    if (i == p.n) {   // the groups are not used here; a workgroup of its own checks them all the same
        const PlanMemory mem(lds, HELD, HELD);
        read_batch<64 * PLAIN_WAVES>(p, mem, true);
        for (int k = tid; k < p.n; k += 64 * PLAIN_WAVES) member_of(p, mem, k, true);
        return;
    }
    const Entry e = entry_of(p, i, true);
    const Segment sg{e.r0, e.T * p.group, e.seq, 0, min(e.len, PLAIN_KEYS), e.len - e.T + 1, 0, 2 * i + 1};
    const int first = (x - i * p.tiles_q) * 16 * QT, ntiles = (sg.k1 + 31) >> 5;
    if (first >= sg.M) return;
    Wave<D, QT, true> w(p, lds + wave * Rows<D>::TILE);
    const int64_t head = (int64_t)kvh * p.head_stride;
    int t = wave;
    if (t < ntiles) {
        w.page_numbers(sg, 0);
        w.load(p.K, w.kf, head, 32 * t, sg.k1);
        w.load(p.V, w.vf, head, 32 * t, sg.k1);
    }
    w.queries(sg, first, kvh);
    // a tile with a successor requests it unconditionally: a load behind a branch would make the waits count as if it had not been issued
    if (t < ntiles) {
        for (; t + WAVES < ntiles; t += WAVES)
            w.step(32 * t, sg.k1, [&] { w.load(p.K, w.kf, head, 32 * (t + WAVES), sg.k1); }, [&] { w.load(p.V, w.vf, head, 32 * (t + WAVES), sg.k1); });
        w.step(32 * t, sg.k1, [] {}, [] {});
    }
    // join the waves, 16 queries at a time
    float* const so = (float*)lds;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const float lt = rows_sum(w.l[qt]);
        __syncthreads();
        if (w.lg == 0) {
            sm_m[wave][w.li] = w.m[qt];
            sm_l[wave][w.li] = lt;
        }
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) *(f32x4*)(so + (wave * 16 + w.li) * OROW + 16 * dt + 4 * w.lg) = w.o[qt][dt];
        __syncthreads();
        const int qi = tid >> 5, d0 = (tid & 31) * PER, r = first + 16 * qt + qi;
        if (r < sg.M) {
            float M = -INFINITY, L = 0.f, acc[PER];
#pragma unroll
            for (int v = 0; v < WAVES; ++v) M = fmaxf(M, sm_m[v][qi]);
            const float use = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int d = 0; d < PER; ++d) acc[d] = 0.f;
#pragma unroll
            for (int v = 0; v < WAVES; ++v) {
                const float f = __builtin_amdgcn_exp2f(sm_m[v][qi] - use);
                L += sm_l[v][qi] * f;
#pragma unroll
                for (int d = 0; d < PER; ++d) acc[d] += so[(v * 16 + qi) * OROW + d0 + d] * f;
            }
            const int tok = r / p.group, row = sg.r0 + tok, hq = kvh * p.group + r - tok * p.group;
            const float inv = inverse_of(L);
            uint32_t b[PER / 2];
#pragma unroll
            for (int d = 0; d < PER; d += 2) b[d / 2] = pack_bf16x2(acc[d] * inv, acc[d + 1] * inv);
            bf16_t* dst = p.out + (int64_t)row * p.o_ld + hq * D + d0;
            if constexpr (PER == 4) *(uint2*)dst = make_uint2(b[0], b[1]);
            else *(uint32_t*)dst = b[0];
            if (p.lse && d0 == 0) p.lse[(int64_t)row * p.heads + hq] = lse_of(use, L);
        }
    }
}

struct Plan {
    bool plain, once, spread;
    int qt, tiles_q, per_min, slots_p, slots;
    int64_t at_plan, at_segments, at_parts, at_ml, at_o, bytes;
};
bool groups_count(const q3asr_kv_pages& c, const q3asr_attn_batch& b) { return b.n_groups > 0 && b.max_shared >= c.page_tokens; }
Plan plan_for(const q3asr_kv_pages& c, const q3asr_attn_batch& b, int heads) {
    Plan r{};
    const int group = heads / c.kv_heads;
    // A small step is all latency: whole sequences that fit the device at once, shared or not, in one launch (head_dim 128: two
    // workgroups per CU, 64: three, or four that follow soon).  us against the stream, the write of the step included, no keys in the
    // caches: 128 sequences of 20 and of 900 tokens, 4 KV heads of 128: 11.6, 44 against 12.0, 48 (there PLAIN_ITEMS is reached); 8 KV heads:
    // 18.1, 85 against 13.0, 83; 256 of 20, 210, 450 and 900 tokens, 4 KV heads of 64: 11.5, 17.4, 24, 42 against 11.6, 20.5, 30, 48.
    r.qt = (int64_t)b.max_rows * group <= 16 ? 1 : 2;
    r.tiles_q = cdiv((int64_t)b.max_rows * group, 16 * r.qt);
    r.plain = b.max_len <= PLAIN_KEYS && (int64_t)b.n * r.tiles_q * c.kv_heads <= (c.head_dim == 128 ? PLAIN_ITEMS : 2 * PLAIN_ITEMS);
    if (r.plain) return r;
    const bool shares = groups_count(c, b);
    const int64_t rows = (int64_t)(shares ? b.max_group_rows : b.max_rows) * group;
    // as many rows at once as the registers of two waves per SIMD hold (64 x 128 sums do not fit).  64 x 64 sums against 32 x 64, us of a
    // step after 1111 tokens, 12 groups, 14 heads: 7 x 24 rows 61, 63; 7 x 48: 96, 97; 7 x up to 24, which fill 87 of 128 rows: 46, 45;
    // after 3584, 2 groups, 16 / 8 heads: 14 x 19 rows 45, 41.
    r.qt = rows <= 16 ? 1 : rows <= 32 || c.head_dim == 128 ? 2 : 4;
    r.once = rows <= 16 * r.qt;
    // Parts of a row: tiles of its longest segment by the least tiles of a wave, and one for where it begins.  More parts spread a few
    // long sequences over the device; the shared and the own segments' are kept to 64 MB each, or 16 where that is more, and one.
    const int64_t part = (int64_t)b.rows * heads * (c.head_dim * 4 + 8);
    const int most = (int)std::max<int64_t>(16, std::min<int64_t>(1024, (64ll << 20) / part));
    const int own = shares ? b.max_own : b.max_len, longest = std::max({own, shares ? b.max_shared : 0, 1});
    r.per_min = std::max(2, cdiv(cdiv(longest, 32), most));
    r.slots_p = shares ? cdiv(cdiv(b.max_shared, 32), r.per_min) + 1 : 0;
    r.slots = r.slots_p + cdiv(cdiv(own, 32), r.per_min) + 1;
    r.spread = r.slots > 32 && (int64_t)b.rows * heads <= 1024;
    auto round = [](int64_t x) { return (x + 255) & ~255ll; };
    const int64_t groups = shares ? b.n_groups : 0;
    r.at_plan = 256;
    r.at_segments = r.at_plan + (b.n + groups > HELD ? round(PlanMemory::bytes(b.n, groups)) : 0);
    r.at_parts = r.at_segments + (b.n + groups > HELD ? round((b.n + groups) * (int64_t)sizeof(Segment)) : 0);
    r.at_ml = r.at_parts + round((int64_t)b.rows * (int64_t)sizeof(RowParts));
    r.at_o = r.at_ml + round((int64_t)b.rows * heads * r.slots * 8);
    r.bytes = r.at_o + round((int64_t)b.rows * heads * r.slots * c.head_dim * 4);
    return r;
}

template <int D>
void launch_d(const AttnParams& p, const Plan& r, hipStream_t s) {
    const dim3 block(256);
    if (r.plain) {
        const dim3 grid(p.n * r.tiles_q * p.kv_heads + (p.n_groups > 0));
        const dim3 plain_block(64 * PLAIN_WAVES);
        if (r.qt == 1) hipLaunchKernelGGL((paged_attn_plain_kernel<D, 1>), grid, plain_block, 0, s, p);
        else hipLaunchKernelGGL((paged_attn_plain_kernel<D, 2>), grid, plain_block, 0, s, p);
        HIP_CHECK(hipGetLastError());
        return;
    }
    const dim3 grid(STREAM_WAVES / WAVES);
    const bool planned = p.n + p.n_groups > HELD;
    if (planned) {
        hipLaunchKernelGGL(paged_attn_plan_kernel, dim3(1), dim3(PLAN), 0, s, p);
        HIP_CHECK(hipGetLastError());
    }
    constexpr int MOST = D == 128 ? 2 : 4;
    auto stream = [&](auto qt, auto once) {
        if (planned) hipLaunchKernelGGL((paged_attn_stream_kernel<D, decltype(qt)::value, decltype(once)::value, true>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((paged_attn_stream_kernel<D, decltype(qt)::value, decltype(once)::value, false>), grid, block, 0, s, p);
    };
    if (r.qt == 1) stream(std::integral_constant<int, 1>{}, std::true_type{});
    else if (r.once && r.qt == 2) stream(std::integral_constant<int, 2>{}, std::true_type{});
    else if (r.qt == 2) stream(std::integral_constant<int, 2>{}, std::false_type{});
    else if (r.once) stream(std::integral_constant<int, MOST>{}, std::true_type{});
    else stream(std::integral_constant<int, MOST>{}, std::false_type{});
    HIP_CHECK(hipGetLastError());
    if (r.spread) hipLaunchKernelGGL((paged_attn_join_kernel<D, true>), dim3(p.rows, p.heads), block, 0, s, p);
    else hipLaunchKernelGGL((paged_attn_join_kernel<D, false>), dim3(p.rows, cdiv(p.heads, 256 / (D / 2))), block, 0, s, p);
    HIP_CHECK(hipGetLastError());
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
    const bool shares = groups_count(c, b);
    p.n = b.n; p.rows = b.rows; p.n_groups = shares ? b.n_groups : 0;
    p.heads = heads; p.kv_heads = c.kv_heads; p.group = heads / c.kv_heads;
    p.max_rows = b.max_rows; p.max_group_rows = b.max_group_rows; p.max_len = b.max_len;
    p.max_own = shares ? b.max_own : b.max_len;
    p.max_shared = b.max_shared;
    // not 0, so that a masked score stays minus infinity
    p.scale_log2 = std::max(std::fabs(scale) * 1.44269504088896340736f, std::numeric_limits<float>::min());
    p.flip = scale < 0.f ? 0x80008000u : 0u;
    p.shift_q = r.qt == 1 ? 4 : r.qt == 2 ? 5 : 6; p.tiles_q = r.tiles_q; p.per_min = r.per_min; p.slots_p = r.slots_p; p.slots = r.slots;
    char* ws = (char*)workspace;
    p.total = (Total*)ws;
    p.plan_ws = ws + r.at_plan;
    p.segments = (Segment*)(ws + r.at_segments);
    p.parts = (RowParts*)(ws + r.at_parts);
    p.part_ml = (float2*)(ws + r.at_ml);
    p.part_o = (float*)(ws + r.at_o);
    ProfScope ps("paged_attn_kernel", 4.0 * b.rows * heads * (double)b.max_len * c.head_dim, s);
    if (c.head_dim == 64) launch_d<64>(p, r, s);
    else launch_d<128>(p, r, s);
}
