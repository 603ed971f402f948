// A KV cache in pages that sequences share, and the attention over it (gfx950).
#pragma once
#include "../../include/q3asr.h"
#include "common.h"

int64_t pages_workspace(const q3asr_kv_pages& c);
void launch_pages_reset(const q3asr_kv_pages& c, hipStream_t s);
// src null: the sequences become empty
void launch_pages_fork(const q3asr_kv_pages& c, const int* dst, const int* src, int n, hipStream_t s);
void launch_pages_reserve(const q3asr_kv_pages& c, const int* seqs, const int* tokens, int n, hipStream_t s);
void launch_pages_compact(const q3asr_kv_pages& c, hipStream_t s);
void launch_pages_write(const q3asr_kv_pages& c, int layer, const bf16_t* k, int64_t k_ld, const bf16_t* v, int64_t v_ld,
                        const q3asr_attn_batch& b, hipStream_t s);
void launch_pages_clear_status(const q3asr_kv_pages& c, hipStream_t s);

int64_t paged_attention_workspace(const q3asr_kv_pages& c, const q3asr_attn_batch& b, int heads);
void launch_paged_attention(const q3asr_kv_pages& c, int layer, const bf16_t* q, int64_t q_ld, int heads, float scale,
                            const q3asr_attn_batch& b, bf16_t* out, int64_t o_ld, float* lse, void* workspace, hipStream_t s);

#ifdef __HIPCC__
// Keeps the first error: code in status[0], entry in status[1], pages short of in status[2].
__device__ __forceinline__ void pages_error(int* status, int code, int entry, int short_of = 0) {
    if (atomicCAS(&status[0], Q3ASR_PAGES_OK, code) == Q3ASR_PAGES_OK) {
        status[1] = entry;
        status[2] = short_of;
    }
}
#endif
