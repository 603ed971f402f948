// Page tables of the KV cache: fork, reserve (copy on write), compact, write (gfx950).
//
// The tables, lengths and reference counts live on the device and change in stream order, so a decode loop never waits for the
// host.  fork, reserve and compact are a plan -- one workgroup checks every entry, ranks what it needs with prefix sums and
// changes the tables, all or nothing -- followed, where page contents move, by a grid of copies that reads its list from the
// workspace.  A plan is latency, phases of one workgroup: 2.5 us (fork of 5) to 11 (reserve for 200 sequences).  All results are
// fixed by the order of the list: atomics only add to whole numbers or take a minimum of them.
#include "paged.h"
#include "prof.h"
#include <algorithm>
#include <climits>

typedef __attribute__((ext_vector_type(4))) int i32x4;

namespace {

constexpr int PLAN = 1024;   // threads of a planning workgroup

struct Pages {
    bf16_t* kv[2];
    int *table, *lens, *refs, *status, *ws;
    int layers, pages, kv_heads, head_dim, page_tokens, max_seqs, max_seq_pages;
};

Pages device_pages(const q3asr_kv_pages& c) {
    return Pages{{c.k, c.v}, c.table, c.lens, c.refs, c.status, (int*)c.workspace, c.layers, c.pages, c.kv_heads, c.head_dim, c.page_tokens,
                 c.max_seqs, c.max_seq_pages};
}

// What an entry of reserve's list needs.
struct __attribute__((aligned(16))) Need {
    int seq, tokens, fill, page;        // fill, page: of the last page if tokens are added to a partly filled one, else fill 0
    int old_pages, new_pages, start, copy;   // start: rank of its first new page; copy: 0, or 1 + rank among the copies
};

// Workspace, in 4-byte words: [0] entries of the copy list, [1] 1 where a call goes on in its next kernel, [16...) the parts below.
struct Layout {
    int64_t rows, row_lens, need, copies, free, per_page, total;
};
__host__ __device__ inline Layout layout(int pages, int max_seqs, int max_seq_pages) {
    Layout l;
    l.rows = 16;                                              // fork: the new table rows
    l.row_lens = l.rows + (int64_t)max_seqs * max_seq_pages;  // fork: their lengths; behind them fork's and reserve's claims
    l.need = (l.row_lens + 2 * (int64_t)max_seqs + 3) & ~3ll;
    l.copies = l.need + 8 * (int64_t)max_seqs;                // (from, to, tokens) of every copy
    l.free = l.copies + 3 * (int64_t)(max_seqs > pages ? max_seqs : pages);
    l.per_page = l.free + pages;                              // reserve: holders in the list and the first; compact: new number
    l.total = l.per_page + 2 * (int64_t)pages;
    return l;
}

// Exclusive prefix sums over the workgroup's threads, and the totals.  Wanted pages need 64 bits: 1024 entries of 2^27.
struct Sums {
    long long wanted;
    int copies;
};
__device__ __forceinline__ Sums block_scan(Sums v, Sums* total, Sums* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sums x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long a = __shfl_up(x.wanted, o, 64);
        const int b = __shfl_up(x.copies, o, 64);
        if (lane >= o) {
            x.wanted += a;
            x.copies += b;
        }
    }
    __syncthreads();
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    Sums before{0, 0}, all{0, 0};
#pragma unroll
    for (int w = 0; w < PLAN / 64; ++w) {
        const Sums t = lds[w];
        if (w < wave) {
            before.wanted += t.wanted;
            before.copies += t.copies;
        }
        all.wanted += t.wanted;
        all.copies += t.copies;
    }
    *total = all;
    return Sums{before.wanted + x.wanted - v.wanted, before.copies + x.copies - v.copies};
}

// A word that atomics of this kernel have changed: read where they are performed, past the compute unit's own cache.
__device__ __forceinline__ int counted(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The lowest wrong entry of a list, as entry * 8 + code.
__device__ __forceinline__ void note(int* worst, int entry, int code) { atomicMin(worst, entry * 8 + code); }

__global__ __launch_bounds__(256) void pages_reset_kernel(Pages p) {
    const int64_t n = (int64_t)p.max_seqs * p.max_seq_pages, i0 = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
    for (int64_t i = i0; i < n; i += step) p.table[i] = -1;
    for (int64_t i = i0; i < p.max_seqs; i += step) p.lens[i] = 0;
    for (int64_t i = i0; i < p.pages; i += step) p.refs[i] = 0;
    if (i0 < 4) p.status[i0] = 0;
}

__global__ void pages_clear_status_kernel(int* status) { if (threadIdx.x < 4) status[threadIdx.x] = 0; }

// Which entry of a list names a sequence first: in LDS where the cache has few sequences, else in `far`, a word per sequence.
constexpr int HELD_SEQS = 4096;
struct Claims {
    int* near;
    int* far;     // NULL: near
    __device__ void open(int seq) const { if (far) far[seq] = INT_MAX; else near[seq] = INT_MAX; }
    __device__ void claim(int seq, int entry) const { if (far) atomicMin(&far[seq], entry); else atomicMin(&near[seq], entry); }
    __device__ int first(int seq) const { return far ? counted(&far[seq]) : near[seq]; }
};

// ---- fork ----
// Short lists (up to FORK_HELD table entries) are checked and carried out by one workgroup, with the rows to come in registers between
// reading all old rows and writing the new ones.  Longer ones take two kernels over the whole device, with the rows in the
// workspace: every workgroup of the first one checks the list for itself, the second one learns the outcome from the workspace.
constexpr int FORK_ROUNDS = 2, FORK_HELD = FORK_ROUNDS * PLAN;

// The lowest wrong entry as entry * 8 + code, INT_MAX if there is none.  All threads of the workgroup; ends behind a barrier.
__device__ __forceinline__ int fork_check(const Pages& p, const int* dst, const int* src, int n, const Claims& claims, int* worst) {
    const int tid = threadIdx.x, threads = blockDim.x;
    if (tid == 0) *worst = INT_MAX;
    const int own = tid < n ? dst[tid] : -1, own_src = tid < n && src ? src[tid] : -1;
    auto named = [&](int i) { return i == tid ? own : dst[i]; };
    for (int i = tid; i < n; i += threads) {
        const int d = named(i);
        if ((unsigned)d < (unsigned)p.max_seqs) claims.open(d);
    }
    __syncthreads();
    for (int i = tid; i < n; i += threads) {
        const int d = named(i), s = i == tid ? own_src : src ? src[i] : -1;
        if (d < -1 || d >= p.max_seqs || s < -1 || s >= p.max_seqs) note(worst, i, Q3ASR_PAGES_BAD_INDEX);
        else if (d >= 0) claims.claim(d, i);   // -1: no entry
    }
    __syncthreads();
    for (int i = tid; i < n; i += threads) {
        const int d = named(i);
        if ((unsigned)d < (unsigned)p.max_seqs && claims.first(d) < i) note(worst, i, Q3ASR_PAGES_DUPLICATE);
    }
    __syncthreads();
    return *worst;
}

__global__ __launch_bounds__(PLAN) void pages_fork_kernel(Pages p, const int* dst, const int* src, int n) {
    __shared__ int worst, claimed[HELD_SEQS];
    const int tid = threadIdx.x, width = p.max_seq_pages;
    const Claims claims{claimed, p.max_seqs <= HELD_SEQS ? nullptr : p.ws + layout(p.pages, p.max_seqs, width).row_lens + p.max_seqs};
    const int wrong = fork_check(p, dst, src, n, claims, &worst);
    if (wrong != INT_MAX) {   // the same for the whole workgroup
        if (tid == 0) pages_error(p.status, wrong & 7, wrong >> 3);
        return;
    }
    const int total = n * width;
    const unsigned magic = 0xffffffffu / (unsigned)width + 1;   // e / width = e * magic >> 32 for these few e
    int now[FORK_ROUNDS], old[FORK_ROUNDS], at[FORK_ROUNDS];
#pragma unroll
    for (int k = 0; k < FORK_ROUNDS; ++k) {
        const int e = tid + k * PLAN;
        now[k] = old[k] = at[k] = -1;
        if (e < total) {
            const int i = width > 1 ? (int)__umulhi((unsigned)e, magic) : e, j = e - i * width, d = dst[i], s = src ? src[i] : -1;
            if (d >= 0) {
                at[k] = d * width + j;   // below 2^31: the table has fewer entries
                if (s >= 0) now[k] = p.table[s * width + j];
                old[k] = p.table[at[k]];
            }
        }
    }
    int lens = 0;
    if (tid < n && src && src[tid] >= 0) lens = p.lens[src[tid]];
    __syncthreads();          // every old row and length has been read
#pragma unroll
    for (int k = 0; k < FORK_ROUNDS; ++k)
        if (at[k] >= 0) {
            p.table[at[k]] = now[k];
            if ((unsigned)now[k] < (unsigned)p.pages) atomicAdd(&p.refs[now[k]], 1);
            if ((unsigned)old[k] < (unsigned)p.pages) atomicSub(&p.refs[old[k]], 1);
        }
    if (tid < n && dst[tid] >= 0) p.lens[dst[tid]] = lens;
}

// A cache of more than HELD_SEQS sequences has its claims in the workspace, where there is one word per sequence: one workgroup checks the
// list in a launch of its own.
__global__ __launch_bounds__(PLAN) void pages_fork_check_kernel(Pages p, const int* dst, const int* src, int n) {
    __shared__ int worst;
    const Claims claims{nullptr, p.ws + layout(p.pages, p.max_seqs, p.max_seq_pages).row_lens + p.max_seqs};
    const int wrong = fork_check(p, dst, src, n, claims, &worst);
    if (threadIdx.x == 0) {
        if (wrong != INT_MAX) pages_error(p.status, wrong & 7, wrong >> 3);
        p.ws[1] = wrong == INT_MAX;
    }
}
template <bool CHECK>
__global__ __launch_bounds__(256) void pages_fork_read_kernel(Pages p, const int* dst, const int* src, int n) {
    if constexpr (CHECK) {
        __shared__ int worst, claimed[HELD_SEQS];
        const int wrong = fork_check(p, dst, src, n, Claims{claimed, nullptr}, &worst);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            if (wrong != INT_MAX) pages_error(p.status, wrong & 7, wrong >> 3);
            p.ws[1] = wrong == INT_MAX;   // for the next kernel
        }
        if (wrong != INT_MAX) return;
    } else {
        if (p.ws[1] == 0) return;
    }
    const int width = p.max_seq_pages;
    const Layout l = layout(p.pages, p.max_seqs, width);
    int *rows = p.ws + l.rows, *row_lens = p.ws + l.row_lens;
    const int lane = threadIdx.x & 63;
    for (int i = blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += gridDim.x * 4) {
        const int d = dst[i], s = src ? src[i] : -1;
        if (d < 0) continue;
        const int64_t to = (int64_t)d * width, from = (int64_t)s * width;
        for (int j = lane; j < width; j += 64) {
            const int now = s < 0 ? -1 : p.table[from + j], old = p.table[to + j];
            rows[(int64_t)i * width + j] = now;
            if ((unsigned)now < (unsigned)p.pages) atomicAdd(&p.refs[now], 1);
            if ((unsigned)old < (unsigned)p.pages) atomicSub(&p.refs[old], 1);
        }
        if (lane == 0) row_lens[i] = s < 0 ? 0 : p.lens[s];
    }
}
__global__ __launch_bounds__(256) void pages_fork_write_kernel(Pages p, const int* dst, int n) {
    if (p.ws[1] == 0) return;
    const int width = p.max_seq_pages;
    const Layout l = layout(p.pages, p.max_seqs, width);
    const int *rows = p.ws + l.rows, *row_lens = p.ws + l.row_lens;
    const int lane = threadIdx.x & 63;
    for (int i = blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += gridDim.x * 4) {
        const int d = dst[i];
        if (d < 0) continue;
        const int64_t to = (int64_t)d * width;
        for (int j = lane; j < width; j += 64) p.table[to + j] = rows[(int64_t)i * width + j];
        if (lane == 0) p.lens[d] = row_lens[i];
    }
}

// ---- reserve ----
constexpr int HELD_STARTS = 2048, HELD_FREE = 4096, HELD_NEED = 512;

__global__ __launch_bounds__(PLAN) void pages_reserve_kernel(Pages p, const int* seqs, const int* tokens, int n) {
    __shared__ int worst, wave_free[PLAN / 64];
    __shared__ Sums scan[PLAN / 64];
    __shared__ int held_start[HELD_STARTS], held_free[HELD_FREE];
    __shared__ Need held_need[HELD_NEED];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, width = p.max_seq_pages, pt = p.page_tokens;
    const Layout l = layout(p.pages, p.max_seqs, width);
    int* copies = p.ws + l.copies;
    __shared__ int claimed[HELD_SEQS];
    const Claims claims{claimed, p.max_seqs <= HELD_SEQS ? nullptr : p.ws + l.row_lens + p.max_seqs};
    int *here = p.ws + l.per_page, *first = here + p.pages;
    Need* const need = (Need*)(p.ws + l.need);
    // free pages, counted by every wave over a contiguous span of the pool
    const int span = ((p.pages + PLAN / 64 - 1) / (PLAN / 64) + 63) & ~63;
    const int s0 = wave * span, s1 = min(p.pages, s0 + span);
    int mine = 0;
    for (int q = s0 + lane; q < s1; q += 64) mine += p.refs[q] == 0;
    if (tid == 0) {
        worst = INT_MAX;
        p.ws[0] = 0;
    }
    __syncthreads();
    // what every entry needs; a thread keeps its first one in registers
    Need own{};
    int own_refs = 0;
    for (int i = tid; i < n; i += PLAN) {
        Need r{};
        r.seq = seqs[i];
        r.tokens = tokens[i];
        int code = Q3ASR_PAGES_OK;
        if (r.seq < -1 || r.seq >= p.max_seqs || r.tokens < 0) code = Q3ASR_PAGES_BAD_INDEX;
        else if (r.seq == -1) r.tokens = 0;   // no entry
        else {
            claims.open(r.seq);
            const int len = p.lens[r.seq];
            if (len < 0 || (int64_t)len + r.tokens > (int64_t)width * pt) code = Q3ASR_PAGES_TOO_LONG;
            else {
                r.old_pages = (len + pt - 1) / pt;
                r.new_pages = (len + r.tokens + pt - 1) / pt;   // both below 2^31 - pt: a table's tokens are
                r.fill = r.tokens > 0 ? len & (pt - 1) : 0;
                if (r.fill) {
                    r.page = p.table[(int64_t)r.seq * width + r.old_pages - 1];
                    if ((unsigned)r.page >= (unsigned)p.pages) code = Q3ASR_PAGES_BAD_INDEX;
                    else {
                        if (i == tid) own_refs = p.refs[r.page];
                        here[r.page] = 0;
                        first[r.page] = INT_MAX;
                    }
                }
            }
        }
        if (code != Q3ASR_PAGES_OK) note(&worst, i, code);
        if (i == tid) own = r;
        else need[i] = r;
    }
    __syncthreads();
    auto entry = [&](int i) { return i == tid ? own : need[i]; };
    for (int i = tid; i < n; i += PLAN) {
        const int s = entry(i).seq;
        if ((unsigned)s < (unsigned)p.max_seqs) claims.claim(s, i);
    }
    __syncthreads();
    for (int i = tid; i < n; i += PLAN) {
        const int s = entry(i).seq;
        if ((unsigned)s < (unsigned)p.max_seqs && claims.first(s) < i) note(&worst, i, Q3ASR_PAGES_DUPLICATE);
    }
    __syncthreads();
    if (worst != INT_MAX) {
        if (tid == 0) pages_error(p.status, worst & 7, worst >> 3);
        return;
    }
    for (int i = tid; i < n; i += PLAN) {
        const Need r = entry(i);
        if (!r.fill) continue;
        atomicAdd(&here[r.page], 1);
        atomicMin(&first[r.page], i);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o, 64);
    if (lane == 0) wave_free[wave] = mine;
    __syncthreads();
    // pages wanted: one for a copy, one for every page begun; ranks in the order of the list
    long long carry = 0;
    int copied = 0;
    for (int i0 = 0; i0 < n; i0 += PLAN) {
        const int i = i0 + tid;
        int copy = 0;
        Need r{};
        if (i < n) {
            r = entry(i);
            if (r.fill) {
                const int refs = i == tid ? own_refs : p.refs[r.page];
                copy = refs > 1 && !(counted(&here[r.page]) == refs && counted(&first[r.page]) == i);
            }
        }
        Sums total;
        const Sums before = block_scan(Sums{copy + r.new_pages - r.old_pages, copy}, &total, scan);
        if (i < n) {
            r.start = (int)min(carry + before.wanted, (long long)INT_MAX);   // a call that wants so many pages is refused below
            r.copy = copy ? 1 + copied + before.copies : 0;
            if (i == tid) own = r;
            if (n <= HELD_NEED) held_need[i] = r;
            else need[i] = r;
            if (i < HELD_STARTS) held_start[i] = r.start;
        }
        carry += total.wanted;
        copied += total.copies;
    }
    // the lowest `carry` free pages
    int at = 0, all = 0;
    for (int w = 0; w < PLAN / 64; ++w) {
        at += w < wave ? wave_free[w] : 0;
        all += wave_free[w];
    }
    if (carry > all) {
        if (tid == 0) pages_error(p.status, Q3ASR_PAGES_NO_PAGES, n, (int)min(carry - all, (long long)INT_MAX));
        return;
    }
    const int pages = (int)carry;
    int* const free = pages <= HELD_FREE ? held_free : p.ws + l.free;
    for (int q0 = s0; q0 < s1 && at < pages; q0 += 64) {
        const bool is = q0 + lane < s1 && p.refs[q0 + lane] == 0;
        const unsigned long long m = __ballot(is);
        const int k = at + __popcll(m & ((1ull << lane) - 1));
        if (is && k < pages) free[k] = q0 + lane;
        at += __popcll(m);
    }
    __syncthreads();
    // every page goes to the last entry that starts at or before its rank (those that want none start where the next one does)
    const bool in_lds = n <= HELD_STARTS;
    for (int k = tid; k < pages; k += PLAN) {
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((in_lds ? held_start[mid] : need[mid].start) <= k) lo = mid;
            else hi = mid;
        }
        const Need r = n <= HELD_NEED ? held_need[lo] : need[lo];
        const int to = free[k], j = k - r.start;
        p.refs[to] = 1;
        if (r.copy && j == 0) {
            int* c = copies + 3 * (r.copy - 1);
            c[0] = r.page;
            c[1] = to;
            c[2] = r.fill;
            atomicSub(&p.refs[r.page], 1);
            p.table[(int64_t)r.seq * width + r.old_pages - 1] = to;
        } else {
            p.table[(int64_t)r.seq * width + r.old_pages + j - (r.copy ? 1 : 0)] = to;
        }
    }
    for (int i = tid; i < n; i += PLAN) {
        const Need r = entry(i);
        if (r.tokens) p.lens[r.seq] += r.tokens;
    }
    if (tid == 0) p.ws[0] = copied;
}

// ---- compact ----
__global__ __launch_bounds__(PLAN) void pages_compact_kernel(Pages p) {
    __shared__ int used[PLAN / 64], gaps[PLAN / 64], far[PLAN / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Layout l = layout(p.pages, p.max_seqs, p.max_seq_pages);
    int *copies = p.ws + l.copies, *to = p.ws + l.per_page;
    const int span = ((p.pages + PLAN / 64 - 1) / (PLAN / 64) + 63) & ~63;
    const int s0 = wave * span, s1 = min(p.pages, s0 + span);
    int mine = 0;
    for (int q = s0 + lane; q < s1; q += 64) mine += p.refs[q] > 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o, 64);
    if (lane == 0) used[wave] = mine;
    __syncthreads();
    int n = 0;
    for (int w = 0; w < PLAN / 64; ++w) n += used[w];
    // gaps are free pages in front of page n, far pages are used ones from n on; there are as many of either
    int g = 0, f = 0;
    for (int q0 = s0; q0 < s1; q0 += 64) {
        const int q = q0 + lane;
        const bool in = q < s1, is = in && p.refs[q] > 0;
        g += __popcll(__ballot(in && !is && q < n));
        f += __popcll(__ballot(is && q >= n));
    }
    if (lane == 0) {
        gaps[wave] = g;
        far[wave] = f;
    }
    __syncthreads();
    int at_g = 0, at_f = 0, moves = 0;
    for (int w = 0; w < PLAN / 64; ++w) {
        at_g += w < wave ? gaps[w] : 0;
        at_f += w < wave ? far[w] : 0;
        moves += far[w];
    }
    for (int q0 = s0; q0 < s1; q0 += 64) {
        const int q = q0 + lane;
        const bool in = q < s1, is = in && p.refs[q] > 0, gap = in && !is && q < n, move = is && q >= n;
        const unsigned long long mg = __ballot(gap), mf = __ballot(move), below = (1ull << lane) - 1;
        if (gap) copies[3 * (at_g + __popcll(mg & below)) + 1] = q;
        if (move) copies[3 * (at_f + __popcll(mf & below))] = q;
        if (in) to[q] = q;
        at_g += __popcll(mg);
        at_f += __popcll(mf);
    }
    __syncthreads();
    for (int k = tid; k < moves; k += PLAN) {
        const int from = copies[3 * k], gap = copies[3 * k + 1];
        copies[3 * k + 2] = p.page_tokens;
        to[from] = gap;
        p.refs[gap] = p.refs[from];
        p.refs[from] = 0;
    }
    if (tid == 0) {
        p.ws[0] = moves;
        p.status[3] = n;
    }
}

// ---- copies of page contents: one wave per (K or V, page, layer, head), a run of filled tokens that is contiguous on both sides ----
// Bound by HBM, as a large copy is: 657 MB moved in 264 us (5.0 TB/s read and written), 40 prompts' last pages to 5 heirs each 54 us.
// RENUMBER: page numbers of the table change on the way (compact).
constexpr int COPY_THREADS = 512;
template <bool RENUMBER>
__global__ __launch_bounds__(COPY_THREADS) void pages_copy_kernel(Pages p) {
    const int copies = p.ws[0];
    if (copies == 0) return;
    const Layout l = layout(p.pages, p.max_seqs, p.max_seq_pages);
    const int* list = p.ws + l.copies;
    if constexpr (RENUMBER) {
        const int* to = p.ws + l.per_page;
        const int64_t n = (int64_t)p.max_seqs * p.max_seq_pages;
        for (int64_t i = (int64_t)blockIdx.x * COPY_THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * COPY_THREADS) {
            const int q = p.table[i];
            if ((unsigned)q < (unsigned)p.pages && to[q] != q) p.table[i] = to[q];
        }
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int runs = p.layers * p.kv_heads;
    const int64_t items = (int64_t)copies * runs * 2, head = (int64_t)p.page_tokens * p.head_dim;
    constexpr int PER = COPY_THREADS / 64;
    for (int64_t it = (int64_t)blockIdx.x * PER + wave; it < items; it += (int64_t)gridDim.x * PER) {
        const int which = (int)(it & 1);
        const int k = (int)((it >> 1) / runs), run = (int)((it >> 1) - (int64_t)k * runs);
        const int layer = run / p.kv_heads, h = run - layer * p.kv_heads;
        const int from = list[3 * k], to = list[3 * k + 1], chunks = list[3 * k + 2] * (p.head_dim / 8);
        const int64_t base = (int64_t)layer * p.pages;
        bf16_t* pool = which ? p.kv[1] : p.kv[0];
        const i32x4* a = (const i32x4*)(pool + ((base + from) * p.kv_heads + h) * head);
        i32x4* b = (i32x4*)(pool + ((base + to) * p.kv_heads + h) * head);
        for (int c = lane; c < chunks; c += 256) {   // 4 KB under way at a time
            const int last = chunks - 1;
            // compact reads and writes every page once (past the caches: 16 / 12 sequences' turnover 554 against 571 us); a
            // prompt's last page is read for each of its heirs
            auto get = [&](int at) { return RENUMBER ? __builtin_nontemporal_load(a + at) : a[at]; };
            auto put = [&](int at, i32x4 v) {
                if (RENUMBER) __builtin_nontemporal_store(v, b + at);
                else b[at] = v;
            };
            const i32x4 v0 = get(c), v1 = get(min(c + 64, last)), v2 = get(min(c + 128, last)), v3 = get(min(c + 192, last));
            put(c, v0);
            if (c + 64 < chunks) put(c + 64, v1);
            if (c + 128 < chunks) put(c + 128, v2);
            if (c + 192 < chunks) put(c + 192, v3);
        }
    }
}

// ---- write: one workgroup per row of the step ----
// All latency: four dependent loads (entry, length, page, its count) lead to the place; the row itself and the search for an earlier
// entry of the same sequence travel beside them.
__global__ __launch_bounds__(256) void pages_write_kernel(Pages p, int layer, const bf16_t* k, int64_t k_ld, const bf16_t* v, int64_t v_ld,
                                                          const int* seqs, const int* cu_rows, int n, int rows) {
    const int row = blockIdx.x, tid = threadIdx.x;
    const int per_head = p.head_dim / 8, chunks = p.kv_heads * per_head;
    auto source = [&](int c) {
        const int which = c >= chunks;
        return (const uint4*)((which ? v + (int64_t)row * v_ld : k + (int64_t)row * k_ld) + (c - which * chunks) * 8);
    };
    uint4 first = make_uint4(0, 0, 0, 0);
    if (tid < 2 * chunks) first = *source(tid);
    // the entry of the list that the row belongs to: the row's own number where every sequence has one row, else the last that begins
    // at or before it
    int lo = min(row, n - 1), r0 = cu_rows[lo], r1 = cu_rows[lo + 1], seq = seqs[lo];
    if (row < r0 || row >= r1) {   // the same for the whole workgroup
        int before = 0;
        for (int i0 = 0; i0 < n; i0 += 256) before += __syncthreads_count(i0 + tid < n && cu_rows[i0 + tid] <= row);
        lo = max(before - 1, 0);
        r0 = cu_rows[lo];
        r1 = cu_rows[lo + 1];
        seq = seqs[lo];
    }
    bool twice = false;
    for (int i = tid; i < lo; i += 256) twice |= seqs[i] == seq;
    twice = __syncthreads_or(twice);
    int code = Q3ASR_PAGES_OK, page = 0, pos = 0;
    if (row >= cu_rows[n]) return;   // behind the last sequence; the same for the whole workgroup
    if (row < r0 || row >= r1 || r1 > rows) code = Q3ASR_PAGES_BAD_BATCH;
    else if ((unsigned)seq >= (unsigned)p.max_seqs) code = Q3ASR_PAGES_BAD_INDEX;
    else if (twice) code = Q3ASR_PAGES_DUPLICATE;
    else {
        pos = p.lens[seq] - (r1 - row);
        const int64_t slot = (int64_t)pos / p.page_tokens;
        if (pos < 0 || slot >= p.max_seq_pages) code = Q3ASR_PAGES_BAD_BATCH;
        else {
            page = p.table[(int64_t)seq * p.max_seq_pages + slot];
            if ((unsigned)page >= (unsigned)p.pages) code = Q3ASR_PAGES_BAD_INDEX;
            else if (p.refs[page] != 1) code = Q3ASR_PAGES_BAD_BATCH;
        }
    }
    if (code != Q3ASR_PAGES_OK) {   // the same for the whole workgroup
        if (tid == 0) pages_error(p.status, code, lo);
        return;
    }
    const int token = pos & (p.page_tokens - 1);
    const int64_t base = ((int64_t)layer * p.pages + page) * p.kv_heads;
    for (int c = tid; c < 2 * chunks; c += 256) {
        const int which = c >= chunks, cc = c - which * chunks, h = cc / per_head, d = (cc - h * per_head) * 8;
        bf16_t* pool = which ? p.kv[1] : p.kv[0];
        *(uint4*)(pool + ((base + h) * p.page_tokens + token) * p.head_dim + d) = c == tid ? first : *source(c);
    }
}

// Copies take what the list holds; a grid that fills the device when it is long and ends at once when it is empty.
template <bool RENUMBER>
void launch_copies(const Pages& p, int64_t most, hipStream_t s) {
    const int64_t items = std::max<int64_t>(most * p.layers * p.kv_heads * 2, RENUMBER ? 1 : 0);
    if (items <= 0) return;
    ProfScope ps("pages_copy_kernel", 0, s);
    constexpr int PER = COPY_THREADS / 64;
    const int grid = (int)std::min<int64_t>((items + PER - 1) / PER, 4 * device_cus());   // items may pass 2^32
    hipLaunchKernelGGL((pages_copy_kernel<RENUMBER>), dim3(grid), dim3(COPY_THREADS), 0, s, p);
    HIP_CHECK(hipGetLastError());
}

}  // namespace

int64_t pages_workspace(const q3asr_kv_pages& c) { return layout(c.pages, c.max_seqs, c.max_seq_pages).total * 4; }

void launch_pages_reset(const q3asr_kv_pages& c, hipStream_t s) {
    const Pages p = device_pages(c);
    const int64_t n = std::max<int64_t>({(int64_t)c.max_seqs * c.max_seq_pages, c.pages, 4});
    ProfScope ps("pages_reset_kernel", 4.0 * n, s);
    hipLaunchKernelGGL(pages_reset_kernel, dim3((int)std::min<int64_t>((n + 255) / 256, 4096)), dim3(256), 0, s, p);
    HIP_CHECK(hipGetLastError());
}

void launch_pages_clear_status(const q3asr_kv_pages& c, hipStream_t s) {
    hipLaunchKernelGGL(pages_clear_status_kernel, dim3(1), dim3(64), 0, s, c.status);
    HIP_CHECK(hipGetLastError());
}

void launch_pages_fork(const q3asr_kv_pages& c, const int* dst, const int* src, int n, hipStream_t s) {
    const Pages p = device_pages(c);
    ProfScope ps("pages_fork_kernel", 12.0 * n * c.max_seq_pages, s);
    // the register form also needs an entry per thread and table offsets of 31 bits
    const bool held = (int64_t)n * c.max_seq_pages <= FORK_HELD && n <= PLAN && (int64_t)c.max_seqs * c.max_seq_pages < (1ll << 31);
    if (held) {
        hipLaunchKernelGGL(pages_fork_kernel, dim3(1), dim3(PLAN), 0, s, p, dst, src, n);
        HIP_CHECK(hipGetLastError());
        return;
    }
    const dim3 grid(std::min(cdiv(n, 4), 4 * device_cus()));
    if (c.max_seqs <= HELD_SEQS) {
        hipLaunchKernelGGL(pages_fork_read_kernel<true>, grid, dim3(256), 0, s, p, dst, src, n);
        HIP_CHECK(hipGetLastError());
    } else {
        hipLaunchKernelGGL(pages_fork_check_kernel, dim3(1), dim3(PLAN), 0, s, p, dst, src, n);
        HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL(pages_fork_read_kernel<false>, grid, dim3(256), 0, s, p, dst, src, n);
        HIP_CHECK(hipGetLastError());
    }
    hipLaunchKernelGGL(pages_fork_write_kernel, grid, dim3(256), 0, s, p, dst, n);
    HIP_CHECK(hipGetLastError());
}

void launch_pages_reserve(const q3asr_kv_pages& c, const int* seqs, const int* tokens, int n, hipStream_t s) {
    const Pages p = device_pages(c);
    {
        ProfScope ps("pages_reserve_kernel", 4.0 * c.pages, s);
        hipLaunchKernelGGL(pages_reserve_kernel, dim3(1), dim3(PLAN), 0, s, p, seqs, tokens, n);
        HIP_CHECK(hipGetLastError());
    }
    launch_copies<false>(p, n, s);
}

void launch_pages_compact(const q3asr_kv_pages& c, hipStream_t s) {
    const Pages p = device_pages(c);
    {
        ProfScope ps("pages_compact_kernel", 4.0 * c.pages, s);
        hipLaunchKernelGGL(pages_compact_kernel, dim3(1), dim3(PLAN), 0, s, p);
        HIP_CHECK(hipGetLastError());
    }
    launch_copies<true>(p, c.pages / 2, s);
}

void launch_pages_write(const q3asr_kv_pages& c, int layer, const bf16_t* k, int64_t k_ld, const bf16_t* v, int64_t v_ld,
                        const q3asr_attn_batch& b, hipStream_t s) {
    const Pages p = device_pages(c);
    ProfScope ps("pages_write_kernel", 8.0 * b.rows * c.kv_heads * c.head_dim, s);
    hipLaunchKernelGGL(pages_write_kernel, dim3(b.rows), dim3(256), 0, s, p, layer, k, k_ld, v, v_ld, b.seqs, b.cu_rows, b.n, b.rows);
    HIP_CHECK(hipGetLastError());
}
