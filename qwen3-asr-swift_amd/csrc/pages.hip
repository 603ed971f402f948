// Page tables of the KV cache: fork, reserve (copy on write), compact, write (gfx950).
//
// The tables, lengths and reference counts live on the device and change in stream order, so a decode loop never waits for the
// host.  fork, reserve and compact are a plan -- one workgroup checks every entry, ranks what it needs with prefix sums and
// changes the tables, all or nothing -- followed, where page contents move, by a grid of copies that reads its list from the
// workspace.  All results are fixed by the order of the list: atomics only add to whole numbers or take a minimum of them.
#include "paged.h"
#include "prof.h"
#include <algorithm>
#include <climits>

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

// Workspace, in 4-byte words: [0] entries of the copy list, [1] 1 where a call goes on to its second kernel, [16...) the parts below.
struct Layout {
    int64_t rows, row_lens, need, copies, free, per_page, total;
};
__host__ __device__ inline Layout layout(int pages, int max_seqs, int max_seq_pages) {
    Layout l;
    l.rows = 16;                                              // fork: the new table rows; reserve: marks of the named sequences
    l.row_lens = l.rows + (int64_t)max_seqs * max_seq_pages;  // fork: their lengths and marks
    l.need = l.row_lens + 2 * (int64_t)max_seqs;              // reserve: first free page of an entry, and whether it copies
    l.copies = l.need + max_seqs;                             // (from, to, tokens) of every copy
    l.free = l.copies + 3 * (int64_t)(max_seqs > pages ? max_seqs : pages);
    l.per_page = l.free + pages;                              // reserve: holders in the list and the first; compact: new number
    l.total = l.per_page + 2 * (int64_t)pages;
    return l;
}

// Exclusive prefix sum over the workgroup's threads, and the total.
__device__ __forceinline__ int block_scan(int v, int* total, int* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(x, o, 64);
        if (lane >= o) x += t;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < PLAN / 64; ++w) {
        const int t = lds[w];
        before += w < wave ? t : 0;
        all += t;
    }
    *total = all;
    return before + x - v;
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

// ---- fork ----
__global__ __launch_bounds__(PLAN) void pages_fork_kernel(Pages p, const int* dst, const int* src, int n) {
    __shared__ int worst;
    const int tid = threadIdx.x, width = p.max_seq_pages;
    const Layout l = layout(p.pages, p.max_seqs, width);
    int *rows = p.ws + l.rows, *row_lens = p.ws + l.row_lens, *mark = row_lens + p.max_seqs;
    if (tid == 0) worst = INT_MAX;
    __syncthreads();
    for (int i = tid; i < n; i += PLAN) {
        const int d = dst[i], s = src ? src[i] : -1;
        if ((unsigned)d >= (unsigned)p.max_seqs || s < -1 || s >= p.max_seqs) note(&worst, i, Q3ASR_PAGES_BAD_INDEX);
        else mark[d] = i;
    }
    __syncthreads();
    for (int i = tid; i < n; i += PLAN) {
        const int d = dst[i];
        if ((unsigned)d < (unsigned)p.max_seqs && mark[d] != i) note(&worst, i, Q3ASR_PAGES_DUPLICATE);
    }
    __syncthreads();
    if (worst != INT_MAX) {   // the same for the whole workgroup
        if (tid == 0) pages_error(p.status, worst & 7, worst >> 3);
        return;
    }
    // the rows to come, from the table as it was; counts of the pages that come and go
    const int64_t total = (int64_t)n * width;
    for (int64_t e = tid; e < total; e += PLAN) {
        const int i = (int)(e / width), j = (int)(e - (int64_t)i * width);
        const int s = src ? src[i] : -1;
        const int now = s < 0 ? -1 : p.table[(int64_t)s * width + j], old = p.table[(int64_t)dst[i] * width + j];
        rows[e] = now;
        if ((unsigned)now < (unsigned)p.pages) atomicAdd(&p.refs[now], 1);
        if ((unsigned)old < (unsigned)p.pages) atomicSub(&p.refs[old], 1);
    }
    for (int i = tid; i < n; i += PLAN) {
        const int s = src ? src[i] : -1;
        row_lens[i] = s < 0 ? 0 : p.lens[s];
    }
    __syncthreads();
    for (int64_t e = tid; e < total; e += PLAN) {
        const int i = (int)(e / width), j = (int)(e - (int64_t)i * width);
        p.table[(int64_t)dst[i] * width + j] = rows[e];
    }
    for (int i = tid; i < n; i += PLAN) p.lens[dst[i]] = row_lens[i];
}

// ---- reserve ----
// What an entry of the list needs.
struct Need {
    int seq, fill, last, page, old_pages, new_pages;
    bool partly;   // adds to a page that is partly filled
};
__device__ __forceinline__ Need need_of(const Pages& p, int seq, int add) {
    Need r;
    r.seq = seq;
    const int len = p.lens[seq], pt = p.page_tokens;
    r.fill = len & (pt - 1);
    r.partly = r.fill > 0 && add > 0;
    r.old_pages = (len + pt - 1) / pt;
    r.new_pages = (int)(((int64_t)len + add + pt - 1) / pt);
    r.last = r.old_pages - 1;
    r.page = r.partly ? p.table[(int64_t)seq * p.max_seq_pages + r.last] : 0;
    return r;
}

__global__ __launch_bounds__(PLAN) void pages_reserve_kernel(Pages p, const int* seqs, const int* tokens, int n) {
    __shared__ int worst, scan[PLAN / 64], wave_free[PLAN / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, width = p.max_seq_pages, pt = p.page_tokens;
    const Layout l = layout(p.pages, p.max_seqs, width);
    int *mark = p.ws + l.rows, *need = p.ws + l.need, *copies = p.ws + l.copies, *free = p.ws + l.free;
    int *here = p.ws + l.per_page, *first = here + p.pages;
    if (tid == 0) {
        worst = INT_MAX;
        p.ws[0] = 0;
    }
    __syncthreads();
    for (int i = tid; i < n; i += PLAN) {
        const int s = seqs[i], add = tokens[i];
        if ((unsigned)s >= (unsigned)p.max_seqs || add < 0) {
            note(&worst, i, Q3ASR_PAGES_BAD_INDEX);
            continue;
        }
        mark[s] = i;
        const int len = p.lens[s];
        if (len < 0 || (int64_t)len + add > (int64_t)width * pt) {
            note(&worst, i, Q3ASR_PAGES_TOO_LONG);
            continue;
        }
        const Need r = need_of(p, s, add);
        if ((unsigned)r.page >= (unsigned)p.pages) note(&worst, i, Q3ASR_PAGES_BAD_INDEX);
        else if (r.partly) {
            here[r.page] = 0;
            first[r.page] = INT_MAX;
        }
    }
    __syncthreads();
    for (int i = tid; i < n; i += PLAN)
        if ((unsigned)seqs[i] < (unsigned)p.max_seqs && mark[seqs[i]] != i) note(&worst, i, Q3ASR_PAGES_DUPLICATE);
    __syncthreads();
    if (worst != INT_MAX) {
        if (tid == 0) pages_error(p.status, worst & 7, worst >> 3);
        return;
    }
    for (int i = tid; i < n; i += PLAN) {
        const Need r = need_of(p, seqs[i], tokens[i]);
        if (!r.partly) continue;
        atomicAdd(&here[r.page], 1);
        atomicMin(&first[r.page], i);
    }
    __syncthreads();
    // pages wanted: one for a copy, one for every page begun; ranks in the order of the list
    int64_t carry = 0;
    int copied = 0;
    for (int i0 = 0; i0 < n; i0 += PLAN) {
        const int i = i0 + tid;
        int want = 0, copy = 0;
        if (i < n) {
            const Need r = need_of(p, seqs[i], tokens[i]);
            if (r.partly) {
                const int refs = p.refs[r.page];
                copy = refs > 1 && !(counted(&here[r.page]) == refs && counted(&first[r.page]) == i);
            }
            want = copy + r.new_pages - r.old_pages;
        }
        int total, copies_total;
        const int before = block_scan(want, &total, scan);
        const int rank = block_scan(copy, &copies_total, scan);
        if (i < n) {
            // fewer than 2^30 pages are wanted before this entry, or the call is refused below
            need[i] = (int)(min(carry + before, (int64_t)0x3fffffff) << 1) | copy;
            if (copy) copies[3 * (copied + rank)] = i;
        }
        carry += total;
        copied += copies_total;
    }
    // the lowest `carry` free pages: every wave counts, then lists, a contiguous span of the pool
    const int span = ((p.pages + PLAN / 64 - 1) / (PLAN / 64) + 63) & ~63;
    const int s0 = wave * span, s1 = min(p.pages, s0 + span);
    int mine = 0;
    for (int q = s0 + lane; q < s1; q += 64) mine += p.refs[q] == 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o, 64);
    if (lane == 0) wave_free[wave] = mine;
    __syncthreads();
    int at = 0, all = 0;
    for (int w = 0; w < PLAN / 64; ++w) {
        at += w < wave ? wave_free[w] : 0;
        all += wave_free[w];
    }
    if (carry > all) {
        if (tid == 0) pages_error(p.status, Q3ASR_PAGES_NO_PAGES, n, (int)min(carry - all, (int64_t)INT_MAX));
        return;
    }
    for (int q0 = s0; q0 < s1 && at < carry; q0 += 64) {
        const bool is = q0 + lane < s1 && p.refs[q0 + lane] == 0;
        const unsigned long long m = __ballot(is);
        const int k = at + __popcll(m & ((1ull << lane) - 1));
        if (is && k < carry) free[k] = q0 + lane;
        at += __popcll(m);
    }
    __syncthreads();
    for (int64_t k = tid; k < carry; k += PLAN) p.refs[free[k]] = 1;
    // table entries of the new pages, by waves: one entry of the list at a time
    for (int i = wave; i < n; i += PLAN / 64) {
        const Need r = need_of(p, seqs[i], tokens[i]);
        const int start = (need[i] >> 1) + (need[i] & 1);
        for (int j = r.old_pages + lane; j < r.new_pages; j += 64)
            p.table[(int64_t)r.seq * width + j] = free[start + j - r.old_pages];
    }
    for (int k = tid; k < copied; k += PLAN) {
        const int i = copies[3 * k];
        const Need r = need_of(p, seqs[i], tokens[i]);
        const int to = free[need[i] >> 1];
        copies[3 * k] = r.page;
        copies[3 * k + 1] = to;
        copies[3 * k + 2] = r.fill;
        atomicSub(&p.refs[r.page], 1);
        p.table[(int64_t)r.seq * width + r.last] = to;
    }
    __syncthreads();
    for (int i = tid; i < n; i += PLAN) p.lens[seqs[i]] += tokens[i];
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

__global__ __launch_bounds__(256) void pages_renumber_kernel(Pages p) {
    if (p.ws[0] == 0) return;
    const Layout l = layout(p.pages, p.max_seqs, p.max_seq_pages);
    const int* to = p.ws + l.per_page;
    const int64_t n = (int64_t)p.max_seqs * p.max_seq_pages;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int q = p.table[i];
        if ((unsigned)q < (unsigned)p.pages && to[q] != q) p.table[i] = to[q];
    }
}

// ---- copies of page contents: one wave per (K or V, page, layer, head), a run of filled tokens that is contiguous on both sides ----
__global__ __launch_bounds__(256) void pages_copy_kernel(Pages p) {
    const int copies = p.ws[0];
    const int* list = p.ws + layout(p.pages, p.max_seqs, p.max_seq_pages).copies;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int runs = p.layers * p.kv_heads;
    const int64_t items = (int64_t)copies * runs * 2, head = (int64_t)p.page_tokens * p.head_dim;
    for (int64_t it = (int64_t)blockIdx.x * 4 + wave; it < items; it += (int64_t)gridDim.x * 4) {
        const int which = (int)(it & 1);
        const int k = (int)((it >> 1) / runs), run = (int)((it >> 1) - (int64_t)k * runs);
        const int layer = run / p.kv_heads, h = run - layer * p.kv_heads;
        const int from = list[3 * k], to = list[3 * k + 1], chunks = list[3 * k + 2] * (p.head_dim / 8);
        const int64_t base = (int64_t)layer * p.pages;
        bf16_t* pool = which ? p.kv[1] : p.kv[0];
        const uint4* a = (const uint4*)(pool + ((base + from) * p.kv_heads + h) * head);
        uint4* b = (uint4*)(pool + ((base + to) * p.kv_heads + h) * head);
        for (int c = lane; c < chunks; c += 64) b[c] = a[c];
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
    // the entry of the list that the row belongs to: the row's own number where every sequence has one row, else by halving
    int lo = min(row, n - 1), r0 = cu_rows[lo], r1 = cu_rows[lo + 1], seq = seqs[lo];
    if (row < r0 || row >= r1) {
        lo = 0;
        int hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (cu_rows[mid] <= row) lo = mid;
            else hi = mid;
        }
        r0 = cu_rows[lo];
        r1 = cu_rows[lo + 1];
        seq = seqs[lo];
    }
    bool twice = false;
    for (int i = tid; i < lo; i += 256) twice |= seqs[i] == seq;
    twice = __syncthreads_or(twice);
    int code = Q3ASR_PAGES_OK, page = 0, pos = 0;
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
void launch_copies(const Pages& p, int64_t most, hipStream_t s) {
    const int64_t items = most * p.layers * p.kv_heads * 2;
    if (items <= 0) return;
    ProfScope ps("pages_copy_kernel", 0, s);
    hipLaunchKernelGGL(pages_copy_kernel, dim3((int)std::min<int64_t>(cdiv(items, 4), 8 * device_cus())), dim3(256), 0, s, p);
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
    hipLaunchKernelGGL(pages_fork_kernel, dim3(1), dim3(PLAN), 0, s, p, dst, src, n);
    HIP_CHECK(hipGetLastError());
}

void launch_pages_reserve(const q3asr_kv_pages& c, const int* seqs, const int* tokens, int n, hipStream_t s) {
    const Pages p = device_pages(c);
    {
        ProfScope ps("pages_reserve_kernel", 4.0 * c.pages, s);
        hipLaunchKernelGGL(pages_reserve_kernel, dim3(1), dim3(PLAN), 0, s, p, seqs, tokens, n);
        HIP_CHECK(hipGetLastError());
    }
    launch_copies(p, n, s);
}

void launch_pages_compact(const q3asr_kv_pages& c, hipStream_t s) {
    const Pages p = device_pages(c);
    {
        ProfScope ps("pages_compact_kernel", 4.0 * c.pages, s);
        hipLaunchKernelGGL(pages_compact_kernel, dim3(1), dim3(PLAN), 0, s, p);
        HIP_CHECK(hipGetLastError());
    }
    const int64_t n = (int64_t)c.max_seqs * c.max_seq_pages;
    hipLaunchKernelGGL(pages_renumber_kernel, dim3((int)std::min<int64_t>((n + 255) / 256, 1024)), dim3(256), 0, s, p);
    HIP_CHECK(hipGetLastError());
    launch_copies(p, c.pages / 2, s);
}

void launch_pages_write(const q3asr_kv_pages& c, int layer, const bf16_t* k, int64_t k_ld, const bf16_t* v, int64_t v_ld,
                        const q3asr_attn_batch& b, hipStream_t s) {
    const Pages p = device_pages(c);
    ProfScope ps("pages_write_kernel", 8.0 * b.rows * c.kv_heads * c.head_dim, s);
    hipLaunchKernelGGL(pages_write_kernel, dim3(b.rows), dim3(256), 0, s, p, layer, k, k_ld, v, v_ld, b.seqs, b.cu_rows, b.n, b.rows);
    HIP_CHECK(hipGetLastError());
}
