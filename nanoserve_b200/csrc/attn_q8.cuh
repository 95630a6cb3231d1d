// Arguments shared by the attention kernels over 8-bit pools.
#pragma once
#include "attn_plan.cuh"
#include "kv8.cuh"

namespace ns {

struct Q8Params {
    const void* q;                   // [n_tokens, n_heads, head_dim], bf16 or fp32
    const uint8_t *k_pool, *v_pool;  // one layer's codes
    const float *k_scale, *v_scale;  // [num_blocks, n_kv_heads] through the two scale strides
    const int32_t* block_tables;
    const int32_t* table_rows;       // may be null: sequence s uses row s
    const int32_t* seq_lens;
    const int32_t* cu_seqlens;       // may be null: sequence s owns exactly query row s
    void* out;
    uint8_t* ws;                     // AttnWorkspace (split partials, arrival counters, prefill items)
    WsLayout L;
    int64_t n_tokens, table_stride, q_stride, out_stride, blk_stride, pos_stride, head_stride, sc_blk_stride, sc_head_stride;
    int n_seqs, n_heads, n_kv_heads, group, head_dim, block_size, num_blocks, table_width;
    int block_shift;                 // log2(block_size) where that is a power of two, else -1 (scalar kernel only)
    float scale, scale_log2;         // softmax scale, and times log2(e)
    int only_prefill;                // 1: sequences of one token are another launch's
    int overlap_prefill;             // 1: the prefill kernel runs beside the decode kernel launched just before it
    int sm_count;
};

// Keys of sequence s: no more than its table row can name, never negative.
__device__ __forceinline__ int q8_len(const Q8Params& p, int s) {
    const long long cap = (long long)p.table_width * p.block_size;
    const int len = p.seq_lens[s];
    return len < 0 ? 0 : (len > cap ? (int)cap : len);
}

namespace q8 {

// The four codes of a word as f16: bytes 0 and 1, bytes 2 and 3.
template <typename KV> __device__ __forceinline__ void expand(uint32_t w, uint32_t& lo, uint32_t& hi);
template <> __device__ __forceinline__ void expand<KvInt8>(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t u = w ^ 0x80808080u;                     // 0 .. 255: u + 1024 is the f16 0x6400 | u
    const uint32_t bias = 0x64806480u;                      // 1024 + 128
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<const __half2*>(&bias));
    __half2 y = __hsub2(*reinterpret_cast<__half2*>(&b), *reinterpret_cast<const __half2*>(&bias));
    lo = *reinterpret_cast<uint32_t*>(&x);
    hi = *reinterpret_cast<uint32_t*>(&y);
}
template <> __device__ __forceinline__ void expand<KvE4m3>(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(lo), "=r"(hi) : "r"(w));
}

}  // namespace q8

}  // namespace ns
