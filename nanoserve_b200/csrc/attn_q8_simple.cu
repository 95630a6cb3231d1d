// Scalar ragged paged attention over 8-bit pools: one warp per (query token, query head), fp32 everywhere. Serves the head
// layouts and block sizes the tensor-core kernels do not cover, fp32 prefill chunks, and on-device cross-checks. A lane scores a key, the
// warp then adds up the values a dim per lane; bound by its scalar loads and multiply-adds.
#include "attn_q8.cuh"

namespace ns {

constexpr int kQ8SimpleWarps = 4;
constexpr int kQ8SimpleMaxHd = 256;

template <typename T, typename KV>
__global__ void __launch_bounds__(kQ8SimpleWarps * 32) ragged_attn_q8_simple_kernel(const Q8Params p) {
    __shared__ float q_sm[kQ8SimpleWarps][kQ8SimpleMaxHd];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int NH = p.n_heads, HD = p.head_dim;
    const int64_t unit = (int64_t)blockIdx.x * kQ8SimpleWarps + warp;
    if (unit >= p.n_tokens * NH) return;
    const int64_t t = unit / NH;
    const int h = (int)(unit - t * NH), g = h / p.group;

    int s = (int)t, j = 0, T_new = 1;
    if (p.cu_seqlens != nullptr) {
        if (t >= p.cu_seqlens[p.n_seqs] || t < p.cu_seqlens[0]) return;      // rows of no sequence stay as they are
        int lo = 0, hi = p.n_seqs;              // cu[lo] <= t < cu[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.cu_seqlens[mid] <= t) lo = mid; else hi = mid;
        }
        s = lo;
        j = (int)(t - p.cu_seqlens[s]);
        T_new = p.cu_seqlens[s + 1] - p.cu_seqlens[s];
    }
    if (p.only_prefill && T_new == 1) return;
    const int len = q8_len(p, s);
    const int n_keys = len - T_new + j + 1;     // causal: query j sees keys 0 .. ctx + j
    const T* qrow = reinterpret_cast<const T*>(p.q) + t * p.q_stride + (int64_t)h * HD;
    for (int d = lane; d < HD; d += 32) q_sm[warp][d] = to_f32<T>(qrow[d]);
    __syncwarp();
    const int32_t* table = p.block_tables + (int64_t)(p.table_rows ? p.table_rows[s] : s) * p.table_stride;

    float m = -INFINITY, l = 0.f;
    float acc[kQ8SimpleMaxHd / 32];
#pragma unroll
    for (int i = 0; i < kQ8SimpleMaxHd / 32; ++i) acc[i] = 0.f;
    for (int base = 0; base < n_keys; base += 32) {
        const int key = base + lane;
        float sc = -INFINITY, sv = 0.f;
        int64_t row_off = 0;
        bool ok = false;
        if (key < n_keys) {
            const int blk = table[key / p.block_size];
            ok = (unsigned)blk < (unsigned)p.num_blocks;
            if (ok) {
                row_off = (int64_t)blk * p.blk_stride + (int64_t)(key % p.block_size) * p.pos_stride + (int64_t)g * p.head_stride;
                const uint8_t* kr = p.k_pool + row_off;
                const int64_t so = (int64_t)blk * p.sc_blk_stride + (int64_t)g * p.sc_head_stride;
                float dot = 0.f;
                for (int d = 0; d < HD; ++d) dot = fmaf(q_sm[warp][d], KV::decode(kr[d]), dot);
                sc = dot * (p.scale * p.k_scale[so]);
                sv = p.v_scale[so];
            }
        }
        const float m_new = fmaxf(m, warp_max(sc));
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = expf(m - ref);
        const float pr = ok ? expf(sc - ref) : 0.f;
        l = l * alpha + warp_sum(pr);
        m = m_new;
#pragma unroll
        for (int i = 0; i < kQ8SimpleMaxHd / 32; ++i) acc[i] *= alpha;
        const float pv = pr * sv;
        const unsigned present = __ballot_sync(0xffffffffu, ok);
        for (int kk = 0; kk < 32; ++kk) {
            if (!((present >> kk) & 1u)) continue;
            const float pk = __shfl_sync(0xffffffffu, pv, kk);
            const int64_t ro = __shfl_sync(0xffffffffu, row_off, kk);
            const uint8_t* vr = p.v_pool + ro;
#pragma unroll
            for (int i = 0; i < kQ8SimpleMaxHd / 32; ++i) {
                const int d = lane + 32 * i;
                if (d < HD) acc[i] = fmaf(pk, KV::decode(vr[d]), acc[i]);
            }
        }
    }
    T* orow = reinterpret_cast<T*>(p.out) + t * p.out_stride + (int64_t)h * HD;
    const float inv = l == 0.f ? 0.f : 1.f / l;      // (a row that sees nothing is zero; a NaN stays one)
#pragma unroll
    for (int i = 0; i < kQ8SimpleMaxHd / 32; ++i) {
        const int d = lane + 32 * i;
        if (d < HD) orow[d] = from_f32<T>(acc[i] * inv);
    }
}

int launch_q8_simple(const Q8Params& p, int dtype, int pool_dtype, cudaStream_t st) {
    if (p.head_dim > kQ8SimpleMaxHd) return fail(NS_ERR_UNSUPPORTED, "attn_q8: head_dim %d > %d", p.head_dim, kQ8SimpleMaxHd);
    const int64_t units = p.n_tokens * p.n_heads;
    const unsigned grid = (unsigned)((units + kQ8SimpleWarps - 1) / kQ8SimpleWarps);
    const dim3 block(kQ8SimpleWarps * 32);
    if (dtype == NS_BF16) {
        if (pool_dtype == NS_INT8) ragged_attn_q8_simple_kernel<__nv_bfloat16, KvInt8><<<grid, block, 0, st>>>(p);
        else ragged_attn_q8_simple_kernel<__nv_bfloat16, KvE4m3><<<grid, block, 0, st>>>(p);
    } else {
        if (pool_dtype == NS_INT8) ragged_attn_q8_simple_kernel<float, KvInt8><<<grid, block, 0, st>>>(p);
        else ragged_attn_q8_simple_kernel<float, KvE4m3><<<grid, block, 0, st>>>(p);
    }
    return check_launch("ragged_attn_q8_simple");
}

}  // namespace ns
