// Rotary position tables in fp32, and the rotation of a step's Q and K fused with the store of K and V into one layer's
// paged pool: 16/32-bit pools (rows copied to their slots) and 8-bit pools (codes + one scale per block and KV head).
#include "kv8.cuh"

namespace ns {

// ------------------------------------------------------------------------------------------------ tables
// cos/sin[t][i] = factor * cos/sin(pos_t * f_i). The angle of a far position needs more than fp32: at position 10^6 an fp32
// angle is off by 0.03 rad. The product and its reduction to a fraction of a turn are in fp64 (exact to 2^-53 of the
// angle), and so are sincospi of the reduced angle and the factor: one rounding to fp32 at the end.
__global__ void __launch_bounds__(256) rope_tables_kernel(const int64_t* pos, const float* inv_freq,
                                                          double factor, float* cos_out, float* sin_out,
                                                          int64_t total, int half) {
    constexpr double kInvPi = 0.31830988618379067154;
    pdl_launch_dependents();
    pdl_wait();
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t t = i / half;
        const double half_turns = (double)pos[t] * (double)inv_freq[i - t * half] * kInvPi;
        double s, c;
        sincospi(half_turns - 2.0 * rint(0.5 * half_turns), &s, &c);
        cos_out[i] = (float)(c * factor);
        sin_out[i] = (float)(s * factor);
    }
}

// ------------------------------------------------------------------------------------------------ rotation
// Quotient of a 31-bit number by a fixed divisor: a multiplication and a shift instead of a division per item.
struct FastDiv {
    uint32_t mul = 0, shift = 0, div = 1;
    FastDiv() = default;
    explicit FastDiv(uint32_t d) : div(d) {
        while ((1ull << shift) < d) ++shift;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t quot(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct RopeAppendParams {
    const void *q, *k, *v;                    // rows of heads, head stride = head_dim
    int64_t q_stride, k_stride, v_stride;     // elements between tokens
    const float *cos, *sin;                   // [n_tokens, rot / 2]
    int rot, interleaved;
    void *q_out, *k_out, *v_out;              // dense, each may be null
    void *k_pool, *v_pool;                    // may be null
    float *k_scale, *v_scale;                 // 8-bit pools
    const int64_t* slots;
    int64_t n_tokens, n_slots;
    int n_heads, n_kv_heads, head_dim, block_size, block_shift;
    int64_t blk_stride, pos_stride, head_stride, sc_blk_stride, sc_head_stride;
    int kv_ctas, planes, chunk, overlap;      // 8-bit pools: CTAs of the append role, (head, K or V) planes, tokens per CTA of a
                                              // large step; two kernels side by side
    FastDiv by_cpr, by_groups;                // items of the other role: pieces per head, groups of heads per token
    int h0, h1, heads_per_item, pairs;        // heads [h0, h1) of q | k | v have work there; pairs: rotate_pairs takes them
};

template <typename T, int V> __device__ __forceinline__ void load_vec(const T* p, float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = to_f32<T>(p[0]);
    } else {
#pragma unroll
        for (int c = 0; c < V / Vec16<T>::N; ++c) {
            const Vec16<T> r = load16(p + c * Vec16<T>::N);
#pragma unroll
            for (int j = 0; j < Vec16<T>::N; ++j) x[c * Vec16<T>::N + j] = r.get(j);
        }
    }
}
template <typename T, int V> __device__ __forceinline__ void store_vec(T* p, const float (&x)[V]) {
    if constexpr (V == 1) {
        p[0] = from_f32<T>(x[0]);
    } else {
#pragma unroll
        for (int c = 0; c < V / Vec16<T>::N; ++c) {
            Vec16<T> r;
#pragma unroll
            for (int j = 0; j < Vec16<T>::N; ++j) r.set(j, x[c * Vec16<T>::N + j]);
            store16(p + c * Vec16<T>::N, r);
        }
    }
}

// cos / sin of the V dims starting at d0 of a rotated head, one value per dim (a pair shares its two).
template <int V> __device__ __forceinline__ void load_angles(const float* row, int rot, int interleaved, int d0, float (&a)[V]) {
    const int half = rot / 2;
    if (interleaved) {
        if constexpr (V == 1) {
            a[0] = row[d0 >> 1];
        } else {
#pragma unroll
            for (int c = 0; c < V / 8; ++c) {
                const float4 w = *reinterpret_cast<const float4*>(row + (d0 >> 1) + 4 * c);
                a[8 * c] = a[8 * c + 1] = w.x;
                a[8 * c + 2] = a[8 * c + 3] = w.y;
                a[8 * c + 4] = a[8 * c + 5] = w.z;
                a[8 * c + 6] = a[8 * c + 7] = w.w;
            }
        }
    } else {
        const float* p = row + (d0 < half ? d0 : d0 - half);
        if constexpr (V == 1) {
            a[0] = p[0];
        } else {
#pragma unroll
            for (int c = 0; c < V / 4; ++c) *reinterpret_cast<float4*>(&a[4 * c]) = *reinterpret_cast<const float4*>(p + 4 * c);
        }
    }
}

// The V dims starting at d0 of one rotated head: (a, b) -> (a c - b s, b c + a s), every product and every sum rounded to
// fp32 (no contraction: the codes of an 8-bit pool are then the same on every path).
template <typename T, int V>
__device__ __forceinline__ void rotate_vec(const T* head, int rot, int interleaved, int d0, const float (&c)[V], const float (&s)[V],
                                           float (&x)[V]) {
    load_vec<T, V>(head + d0, x);
    if (interleaved) {
        if constexpr (V == 1) {
            const float y = to_f32<T>(head[d0 ^ 1]);
            const float xc = __fmul_rn(x[0], c[0]), ys = __fmul_rn(y, s[0]);
            x[0] = (d0 & 1) ? __fadd_rn(xc, ys) : __fsub_rn(xc, ys);
        } else {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float a = x[j], b = x[j + 1];
                x[j] = __fsub_rn(__fmul_rn(a, c[j]), __fmul_rn(b, s[j]));
                x[j + 1] = __fadd_rn(__fmul_rn(b, c[j]), __fmul_rn(a, s[j]));
            }
        }
    } else {
        const int half = rot / 2;
        const bool lo = d0 < half;
        float y[V];
        load_vec<T, V>(head + (lo ? d0 + half : d0 - half), y);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float xc = __fmul_rn(x[j], c[j]), ys = __fmul_rn(y[j], s[j]);
            x[j] = lo ? __fsub_rn(xc, ys) : __fadd_rn(xc, ys);
        }
    }
}

// ------------------------------------------------------------------------------------------------ append, 8-bit pools
// A block's scale depends on every row of it that the call writes, so a block has ONE owner per plane (KV head, K or V): the
// warp of the first token of the call which lands in it (the leader), whatever order the tokens come in and however often a
// slot is named. The owner needs the block's members: for each row, the last token of the call that names it.
//   steps of up to kSmallStep tokens: a warp per (token, plane) looks through all slots itself; nothing is shared, no barrier.
//   larger steps: a CTA takes kAppendChunk tokens of a KV head, finds the leaders among them, and its threads look through all
//     slots once for all of its leaders' blocks.
// (A layer of 14 / 2 heads of 64, 256 tokens: 3.3 us in blocks of their own and 3.6 as one chunk, against 11 and 5.6 for the CTA form.
// The first form at 512 tokens: 4.4 and 4.6 against 11 and 5.8, but 9.0 and 8.0 against 12.0 and 7.4 for 28 / 4 heads of 128, and the
// registers that twice as many slots take cost every decode step 0.5 us.) What bounds the large form is latency: a CTA's chain of slot,
// row and code loads, in some rounds of six CTAs per SM; DRAM is 4 % busy. With 28 / 4 heads of 128, 2,048 tokens of one prompt take
// 12.6 us, 37 decode rows and four chunks of 1,021 24.8. Chunks of 16 tokens and 256 threads: 13.8 and 25.8; one CTA for four heads of
// a chunk, which looks through the slots once: 20.1 and 33.8.
constexpr int kSmallStep = 256;
constexpr int kAppendChunk = 8;               // tokens per CTA of a large step
constexpr int kAppendMaxBlock = 64;           // largest block size
constexpr int kMembers = kAppendChunk * kAppendMaxBlock;
constexpr int kAppendWarps = 8, kLargeThreads = 128;

// What the owner of a block does with its scale: the magnitude of the written rows, the old scale and whether the call writes the
// block's first row give the new one.
struct Rescale {
    float now, old, inv, ratio;
    bool fresh, dead;                          // dead: the scale is NaN, every written code is 0
    __device__ __forceinline__ bool grown() const { return !fresh && !(now == old); }
};
template <typename KV> __device__ __forceinline__ Rescale rescale(uint32_t amax, float old, bool fresh) {
    Rescale r;
    const float s_new = pow2_scale<KV>(amax);
    r.old = old;
    r.fresh = fresh;
    r.now = fresh ? s_new : (old != old || s_new != s_new) ? __int_as_float(0x7fffffff) : fmaxf(old, s_new);
    r.inv = 1.0f / r.now;
    r.ratio = old / r.now;
    r.dead = r.now != r.now;
    return r;
}
__device__ __forceinline__ void note_max(uint32_t& amax, float x) { amax = max(amax, (uint32_t)__float_as_int(x) & 0x7fffffffu); }

// Codes of 8 dims at dst: of a written row (x: its values), of a row the call does not write in a block it starts afresh, or of an
// older row under a scale that grew (was: its codes, requested before any of the block's stores).
__device__ __forceinline__ void old_codes(const uint8_t* src, int partner, uint2 (&was)[2]) {
    was[0] = *reinterpret_cast<const uint2*>(src);
    was[1] = *reinterpret_cast<const uint2*>(src + partner);
}
template <typename KV> __device__ __forceinline__ void put_codes8(uint8_t* dst, const Rescale& r, bool written, const float* x, uint2 was) {
    if (!written && !r.fresh && !r.grown()) return;
    uint2 w = make_uint2(0u, 0u);
    if (written) {
        if (!r.dead) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = __fmul_rn(x[j], r.inv);
            w = make_uint2(KV::encode4(y[0], y[1], y[2], y[3]), KV::encode4(y[4], y[5], y[6], y[7]));
        }
    } else if (!r.fresh && r.ratio < 1.f) {                // (a scale that became NaN, or grew from a NaN: code 0; ratio < 1: no overflow)
        auto again = [&](uint32_t v) -> uint32_t {
            float y[4];
            KV::decode4(KV::without_nan(v), y);
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = __fmul_rn(y[j], r.ratio);
            return KV::encode4(y[0], y[1], y[2], y[3]);
        };
        w = make_uint2(again(was.x), again(was.y));
    }
    *reinterpret_cast<uint2*>(dst) = w;
}
template <typename KV, int V> __device__ __forceinline__ void put_codes(uint8_t* dst, const Rescale& r, bool written, const float* x) {
    if constexpr (V == 8) {
        put_codes8<KV>(dst, r, written, x, !written && r.grown() ? *reinterpret_cast<const uint2*>(dst) : make_uint2(0u, 0u));
    } else {
        if (!written && !r.fresh && !r.grown()) return;
        *dst = (uint8_t)(written ? KV::encode(__fmul_rn(x[0], r.inv)) : r.fresh ? 0u : KV::encode(__fmul_rn(KV::decode(*dst), r.ratio)));
    }
}

// One block of one plane by one warp, any sizes. mem[row]: the token that writes the row, or -1. The rotated values are computed
// twice, for the magnitude and for the codes, from rows that the first pass left in the caches.
template <typename T, typename KV, int V>
__device__ __forceinline__ void append_block(const RopeAppendParams& p, int plane, int64_t blk, const int* mem) {
    const int lane = threadIdx.x & 31, head = plane >> 1, is_v = plane & 1, hd = p.head_dim, half = p.rot / 2;
    const T* src = reinterpret_cast<const T*>(is_v ? p.v : p.k) + (int64_t)head * hd;
    const int64_t src_stride = is_v ? p.v_stride : p.k_stride;
    uint8_t* pool = reinterpret_cast<uint8_t*>(is_v ? p.v_pool : p.k_pool) + head * p.head_stride + blk * p.blk_stride;
    float* sc = (is_v ? p.v_scale : p.k_scale) + head * p.sc_head_stride + blk * p.sc_blk_stride;
    const float old = *sc;
    const int cpr = hd / V, items = p.block_size * cpr;
    auto values = [&](int t, int d0, float (&x)[V]) {
        const T* row = src + t * src_stride;
        if (!is_v && d0 < p.rot) {
            float c[V], s[V];
            load_angles<V>(p.cos + (int64_t)t * half, p.rot, p.interleaved, d0, c);
            load_angles<V>(p.sin + (int64_t)t * half, p.rot, p.interleaved, d0, s);
            rotate_vec<T, V>(row, p.rot, p.interleaved, d0, c, s, x);
        } else {
            load_vec<T, V>(row + d0, x);
        }
    };
    uint32_t amax = 0;
#pragma unroll 2
    for (int i = lane; i < items; i += 32) {
        const int off = i / cpr, t = mem[off];
        if (t < 0) continue;
        float x[V];
        values(t, (i - off * cpr) * V, x);
#pragma unroll
        for (int j = 0; j < V; ++j) note_max(amax, x[j]);
    }
    const Rescale r = rescale<KV>(__reduce_max_sync(0xffffffffu, amax), old, mem[0] >= 0);
    __syncwarp();
    if (lane == 0 && !(r.now == old)) *sc = r.now;
#pragma unroll 2
    for (int i = lane; i < items; i += 32) {
        const int off = i / cpr, t = mem[off], d0 = (i - off * cpr) * V;
        float x[V];
        if (t >= 0) values(t, d0, x);
        put_codes<KV, V>(pool + (int64_t)off * p.pos_stride + d0, r, t >= 0, x);
    }
}

// The same for blocks of 16 rows of 64 or 128 dims, half layout, whole head rotated (the framework's models): a lane takes 8 dims of
// the low half of a row together with their partners, so each row is read once, and keeps the values for the codes.
template <typename T, typename KV, int HD>
__device__ __forceinline__ void append_block_pairs(const RopeAppendParams& p, int plane, int64_t blk, const int* mem) {
    constexpr int CPR = HD / 16, NI = 16 * CPR / 32;          // pairs of pieces per row, per lane
    const int lane = threadIdx.x & 31, head = plane >> 1, is_v = plane & 1;
    const T* src = reinterpret_cast<const T*>(is_v ? p.v : p.k) + (int64_t)head * HD;
    const int64_t src_stride = is_v ? p.v_stride : p.k_stride;
    uint8_t* pool = reinterpret_cast<uint8_t*>(is_v ? p.v_pool : p.k_pool) + head * p.head_stride + blk * p.blk_stride;
    float* sc = (is_v ? p.v_scale : p.k_scale) + head * p.sc_head_stride + blk * p.sc_blk_stride;
    const float old = *sc;
    const int row0 = lane / CPR, d0 = (lane % CPR) * 8;                            // row n * (32 / CPR) + row0 of item n
    float lo[NI][8], hi[NI][8];
    uint32_t amax = 0;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
        const int t = mem[n * (32 / CPR) + row0];
        if (t >= 0) {
            const T* row = src + t * src_stride + d0;
            load_vec<T, 8>(row, lo[n]);
            load_vec<T, 8>(row + HD / 2, hi[n]);
            if (!is_v) {
                const float* cr = p.cos + (int64_t)t * (HD / 2) + d0;
                const float* sr = p.sin + (int64_t)t * (HD / 2) + d0;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const float4 c4 = *reinterpret_cast<const float4*>(cr + 4 * w), s4 = *reinterpret_cast<const float4*>(sr + 4 * w);
                    const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float a = lo[n][4 * w + j], b = hi[n][4 * w + j];
                        lo[n][4 * w + j] = __fsub_rn(__fmul_rn(a, c[j]), __fmul_rn(b, s[j]));
                        hi[n][4 * w + j] = __fadd_rn(__fmul_rn(b, c[j]), __fmul_rn(a, s[j]));
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                note_max(amax, lo[n][j]);
                note_max(amax, hi[n][j]);
            }
        }
        if (n & 1) asm volatile("" ::: "memory");            // two rows' loads at a time: all of them would not fit the registers
    }
    const Rescale r = rescale<KV>(__reduce_max_sync(0xffffffffu, amax), old, mem[0] >= 0);
    __syncwarp();
    if (lane == 0 && !(r.now == old)) *sc = r.now;
    uint2 was[NI][2];
    if (r.grown()) {
#pragma unroll
        for (int n = 0; n < NI; ++n) old_codes(pool + (int64_t)(n * (32 / CPR) + row0) * p.pos_stride + d0, HD / 2, was[n]);
    }
#pragma unroll
    for (int n = 0; n < NI; ++n) {
        const int off = n * (32 / CPR) + row0;
        uint8_t* dst = pool + (int64_t)off * p.pos_stride + d0;
        const bool written = mem[off] >= 0;
        put_codes8<KV>(dst, r, written, lo[n], was[n][0]);
        put_codes8<KV>(dst + HD / 2, r, written, hi[n], was[n][1]);
    }
}

template <typename T, typename KV, int V>
__device__ __forceinline__ void append_any(const RopeAppendParams& p, int plane, int64_t blk, const int* mem) {
    if constexpr (V == 8) {
        if (p.pairs && p.block_size == 16 && p.head_dim == 64) return append_block_pairs<T, KV, 64>(p, plane, blk, mem);
        if (p.pairs && p.block_size == 16 && p.head_dim == 128) return append_block_pairs<T, KV, 128>(p, plane, blk, mem);
    }
    append_block<T, KV, V>(p, plane, blk, mem);
}

__device__ __forceinline__ int block_of(const RopeAppendParams& p, int64_t slot) {
    return (slot >= 0 && slot < p.n_slots) ? (int)(slot >> p.block_shift) : -1;
}

// A warp per (token, plane).
template <typename T, typename KV, int V> __device__ void append_small(const RopeAppendParams& p, int cta) {
    __shared__ int member[kAppendWarps][kAppendMaxBlock];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mask = p.block_size - 1;
    const int unit = cta * kAppendWarps + warp, n_tok = (int)p.n_tokens;
    const int t = unit / p.planes, plane = unit - t * p.planes;
    if (t >= n_tok) return;
    int blk[kSmallStep / 32], off[kSmallStep / 32];
#pragma unroll
    for (int k = 0; k < kSmallStep / 32; ++k) {
        const int i = k * 32 + lane;
        const int64_t slot = i < n_tok ? p.slots[i] : -1;
        blk[k] = block_of(p, slot);
        off[k] = (int)slot & mask;
    }
    int b = -1;
#pragma unroll
    for (int k = 0; k < kSmallStep / 32; ++k)
        if (k == t >> 5) b = blk[k];
    b = __shfl_sync(0xffffffffu, b, t & 31);
    if (b < 0) return;
    int* mem = member[warp];
    for (int i = lane; i < p.block_size; i += 32) mem[i] = -1;
    __syncwarp();
    bool first = true;
#pragma unroll
    for (int k = 0; k < kSmallStep / 32; ++k) {
        unsigned hit = __ballot_sync(0xffffffffu, blk[k] == b);
        if (hit == 0) continue;
        if (k * 32 + __ffs(hit) - 1 < t) first = false;        // an earlier token owns the block
        if (!first) break;
        if ((hit >> lane) & 1u) atomicMax(&mem[off[k]], k * 32 + lane);
    }
    if (!first) return;
    __syncwarp();
    append_any<T, KV, V>(p, plane, b, mem);
}

// The blocks of a CTA's candidates, K and V, by all of its warps: the layouts of append_block_pairs. A step is a warp's share of a
// unit (candidate, K or V): 32 pairs of pieces. First the magnitudes, then the scales, then the codes (the rotated values are
// computed again, from rows that the first pass left in the caches).
template <typename T, typename KV, int HD>
__device__ __forceinline__ void append_units(const RopeAppendParams& p, int head, int nc, const int* cand_block, const int* cand_dead, const int* member,
                                             uint32_t* unit_max, Rescale* unit_scale) {
    constexpr int CPR = HD / 16, NI = 16 * CPR / 32, B = 2, NW = kLargeThreads / 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row0 = lane / CPR, d0 = (lane % CPR) * 8;
    const int units = 2 * nc, steps = units * NI;
    float old = 0.f;
    auto scale_of = [&](int u) -> float* {
        return ((u & 1) ? p.v_scale : p.k_scale) + head * p.sc_head_stride + (int64_t)cand_block[u >> 1] * p.sc_blk_stride;
    };
    for (int u = tid; u < units; u += kLargeThreads) unit_max[u] = 0;
    if (tid < units) old = *scale_of(tid);
    __syncthreads();
    auto pair_values = [&](int t, bool is_v, float (&lo)[8], float (&hi)[8]) {
        const T* row = reinterpret_cast<const T*>(is_v ? p.v : p.k) + (int64_t)head * HD + t * (is_v ? p.v_stride : p.k_stride) + d0;
        load_vec<T, 8>(row, lo);
        load_vec<T, 8>(row + HD / 2, hi);
        if (is_v) return;
        const float* cr = p.cos + (int64_t)t * (HD / 2) + d0;
        const float* sr = p.sin + (int64_t)t * (HD / 2) + d0;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const float4 c4 = *reinterpret_cast<const float4*>(cr + 4 * w), s4 = *reinterpret_cast<const float4*>(sr + 4 * w);
            const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = lo[4 * w + j], b = hi[4 * w + j];
                lo[4 * w + j] = __fsub_rn(__fmul_rn(a, c[j]), __fmul_rn(b, s[j]));
                hi[4 * w + j] = __fadd_rn(__fmul_rn(b, c[j]), __fmul_rn(a, s[j]));
            }
        }
    };
#pragma unroll 2
    for (int st = warp; st < steps; st += NW) {
        const int u = st / NI, c = u >> 1, t = member[c * 16 + (st % NI) * (32 / CPR) + row0];
        if (cand_dead[c] || !__any_sync(0xffffffffu, t >= 0)) continue;
        uint32_t amax = 0;
        if (t >= 0) {
            float lo[8], hi[8];
            pair_values(t, u & 1, lo, hi);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                note_max(amax, lo[j]);
                note_max(amax, hi[j]);
            }
        }
        amax = __reduce_max_sync(0xffffffffu, amax);
        if (lane == 0) atomicMax(&unit_max[u], amax);
    }
    __syncthreads();
    for (int u = tid; u < units; u += kLargeThreads) {
        if (cand_dead[u >> 1]) continue;
        const float was = u == tid ? old : *scale_of(u);
        const Rescale r = rescale<KV>(unit_max[u], was, member[(u >> 1) * 16] >= 0);
        unit_scale[u] = r;
        if (!(r.now == was)) *scale_of(u) = r.now;
    }
    __syncthreads();
    for (int st0 = warp; st0 < steps; st0 += B * NW) {
        uint2 was[B][2];                                  // all loads of B steps before the first store
        float lo[B][8], hi[B][8];
        auto dst_of = [&](int c, int u, int off) -> uint8_t* {
            return reinterpret_cast<uint8_t*>((u & 1) ? p.v_pool : p.k_pool) + head * p.head_stride + cand_block[c] * p.blk_stride + off * p.pos_stride + d0;
        };
#pragma unroll
        for (int k = 0; k < B; ++k) {
            const int st = st0 + k * NW, u = st / NI, c = u >> 1, off = (st % NI) * (32 / CPR) + row0;
            if (st >= steps || cand_dead[c]) continue;
            const int t = member[c * 16 + off];
            if (t >= 0) pair_values(t, u & 1, lo[k], hi[k]);
            else if (unit_scale[u].grown()) old_codes(dst_of(c, u, off), HD / 2, was[k]);
        }
#pragma unroll
        for (int k = 0; k < B; ++k) {
            const int st = st0 + k * NW, u = st / NI, c = u >> 1, off = (st % NI) * (32 / CPR) + row0;
            if (st >= steps || cand_dead[c]) continue;
            const Rescale r = unit_scale[u];
            const bool written = member[c * 16 + off] >= 0;
            uint8_t* dst = dst_of(c, u, off);
            put_codes8<KV>(dst, r, written, lo[k], was[k][0]);
            put_codes8<KV>(dst + HD / 2, r, written, hi[k], was[k][1]);
        }
    }
}

// A CTA per (chunk of tokens, KV head): K and V share the search for the members.
template <typename T, typename KV, int V> __device__ void append_large(const RopeAppendParams& p, int cta) {
    __shared__ int member[kMembers];
    __shared__ int cand_block[kAppendChunk], cand_tok[kAppendChunk], cand_dead[kAppendChunk];
    __shared__ int key[4 * kAppendChunk], val[4 * kAppendChunk];          // block -> candidate, open addressing, a quarter full at most
    __shared__ int n_cand;
    __shared__ uint32_t filter;
    __shared__ uint32_t unit_max[2 * kAppendChunk];
    __shared__ Rescale unit_scale[2 * kAppendChunk];
    constexpr int kSlotsOfTable = 4 * kAppendChunk;
    const int tid = threadIdx.x, warp = tid >> 5;
    const int head = cta % p.n_kv_heads, bs = p.block_size, mask = bs - 1;
    const int t0 = (cta / p.n_kv_heads) * p.chunk, n_tok = (int)p.n_tokens;
    auto hash = [](int b) -> int { return (int)(((uint32_t)b * 2654435761u) >> 16) & (kSlotsOfTable - 1); };
    int64_t slot[8];                                                      // the first of all slots, asked for before anything else
    auto request = [&](int base) {
#pragma unroll
        for (int k = 0; k < 8; ++k) slot[k] = base + k * kLargeThreads < n_tok ? p.slots[base + k * kLargeThreads] : -1;
    };
    request(tid);
    if (tid == 0) n_cand = 0, filter = 0;
    for (int i = tid; i < p.chunk * bs; i += blockDim.x) member[i] = -1;
    for (int i = tid; i < kSlotsOfTable; i += blockDim.x) key[i] = -1;
    __syncthreads();
    if (tid < p.chunk && t0 + tid < n_tok) {
        const int t = t0 + tid, b = block_of(p, p.slots[t]);
        if (b >= 0 && (t == 0 || block_of(p, p.slots[t - 1]) != b)) {
            const int c = atomicAdd(&n_cand, 1);
            cand_block[c] = b;
            cand_tok[c] = t;
            cand_dead[c] = 0;
            atomicOr(&filter, 1u << (b & 31));
        }
    }
    __syncthreads();
    const int nc = n_cand;
    if (nc == 0) return;                                                  // (the chunk's blocks began in an earlier one)
    // Of two candidates with one block the earlier token's is the owner; the table keeps that one (ends: fewer entries than places).
    if (tid < nc) {
        const int b = cand_block[tid];
        for (int h = hash(b);; h = (h + 1) & (kSlotsOfTable - 1)) {
            const int was = atomicCAS(&key[h], -1, b);
            if (was == -1 || was == b) break;
        }
    }
    for (int i = tid; i < kSlotsOfTable; i += blockDim.x) val[i] = 0x7fffffff;
    __syncthreads();
    auto find = [&](int b) -> int {                                       // place of block b, -1 if it is no candidate's
        for (int h = hash(b);; h = (h + 1) & (kSlotsOfTable - 1)) {
            const int k = key[h];
            if (k == b) return h;
            if (k == -1) return -1;
        }
    };
    if (tid < nc) atomicMin(&val[find(cand_block[tid])], cand_tok[tid] << 8 | tid);      // (the token decides; kAppendChunk <= 256)
    __syncthreads();
    if (tid < nc && (val[find(cand_block[tid])] & 255) != tid) cand_dead[tid] = 1;
    __syncthreads();
    // Every CTA looks at every slot, so a slot that is nobody's must cost little: bit (block & 31) of `seen` turns most of them away.
    const uint32_t seen = filter;
    for (int base = tid; base < n_tok; base += 8 * kLargeThreads) {       // eight slots in flight
        if (base != tid) request(base);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (!((seen >> ((uint32_t)(slot[k] >> p.block_shift) & 31u)) & 1u)) continue;
            const int t = base + k * kLargeThreads, b = block_of(p, slot[k]);
            const int at = b < 0 ? -1 : find(b);
            if (at < 0) continue;
            const int c = val[at] & 255;
            if (t < cand_tok[c]) cand_dead[c] = 1;                        // an earlier token owns the block
            else atomicMax(&member[c * bs + ((int)slot[k] & mask)], t);
        }
    }
    __syncthreads();
    if constexpr (V == 8) {
        // Many candidates are blocks with a row or two each (decode rows): a warp takes a block's K or V as a whole, its loads all in
        // flight at once. (512 tokens in blocks of their own, 28 / 4 heads of 128: 12.4 us against 24.8 by all warps; 37 of those
        // before a 2,048-token chunk: 14.9 against 26.6.)
        if (p.pairs && bs == 16 && nc > 2 && (p.head_dim == 64 || p.head_dim == 128)) {
            for (int i = warp; i < 2 * nc; i += kLargeThreads / 32)
                if (!cand_dead[i >> 1]) append_any<T, KV, V>(p, 2 * head + (i & 1), cand_block[i >> 1], member + (i >> 1) * bs);
            return;
        }
        if (p.pairs && bs == 16 && p.head_dim == 64) return append_units<T, KV, 64>(p, head, nc, cand_block, cand_dead, member, unit_max, unit_scale);
        if (p.pairs && bs == 16 && p.head_dim == 128) return append_units<T, KV, 128>(p, head, nc, cand_block, cand_dead, member, unit_max, unit_scale);
    }
    for (int i = warp; i < 2 * nc; i += kLargeThreads / 32) {
        const int c = i >> 1;
        if (!cand_dead[c]) append_block<T, KV, V>(p, 2 * head + (i & 1), cand_block[c], member + c * bs);
    }
}

// ------------------------------------------------------------------------------------------------ the kernel
struct NoKv8 {};

// Offset of a token's row in a 16/32-bit pool, -1 if its slot is outside.
__device__ __forceinline__ int64_t pool_row(const RopeAppendParams& p, int64_t slot) {
    if (slot < 0 || slot >= p.n_slots) return -1;
    const int64_t b = p.block_shift >= 0 ? slot >> p.block_shift : slot / p.block_size;
    return b * p.blk_stride + (slot - b * p.block_size) * p.pos_stride;
}

// Half layout, whole head: a thread takes 8 dims of the low half and their partners for several heads, so each row is read once
// and the angles once per group of heads; all of its loads are in flight before the first is used.
template <typename T, bool kv8> __device__ __forceinline__ void rotate_pairs(const RopeAppendParams& p, int cta, int ctas) {
    constexpr int H = 2, W = 8 / Vec16<T>::N;        // heads per item; 16-byte words per 8 dims
    const int hd = p.head_dim, half = hd / 2, NH = p.n_heads, NKV = p.n_kv_heads;
    const bool pool16 = !kv8 && p.k_pool != nullptr;
    const uint32_t cpr = p.by_cpr.div, total = (uint32_t)p.n_tokens * p.by_groups.div * cpr;
    for (uint32_t i = cta * blockDim.x + threadIdx.x; i < total; i += ctas * blockDim.x) {
        const uint32_t tg = p.by_cpr.quot(i);
        const int d0 = (int)(i - tg * cpr) * 8;
        const int64_t t = p.by_groups.quot(tg);
        const int first = p.h0 + (int)(tg - (uint32_t)t * p.by_groups.div) * H;
        Vec16<T> lo[H][W], hi[H][W];
#pragma unroll
        for (int e = 0; e < H; ++e) {
            const int h = first + e;
            if (h >= p.h1) continue;
            const T* head = (h < NH         ? reinterpret_cast<const T*>(p.q) + t * p.q_stride + (int64_t)h * hd
                             : h < NH + NKV ? reinterpret_cast<const T*>(p.k) + t * p.k_stride + (int64_t)(h - NH) * hd
                                            : reinterpret_cast<const T*>(p.v) + t * p.v_stride + (int64_t)(h - NH - NKV) * hd) + d0;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                lo[e][w] = load16(head + w * Vec16<T>::N);
                hi[e][w] = load16(head + half + w * Vec16<T>::N);
            }
        }
        float c[8], s[8];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            *reinterpret_cast<float4*>(&c[4 * w]) = *reinterpret_cast<const float4*>(p.cos + t * half + d0 + 4 * w);
            *reinterpret_cast<float4*>(&s[4 * w]) = *reinterpret_cast<const float4*>(p.sin + t * half + d0 + 4 * w);
        }
        const int64_t row_off = pool16 ? pool_row(p, p.slots[t]) : -1;
#pragma unroll
        for (int e = 0; e < H; ++e) {
            const int h = first + e;
            if (h >= p.h1) continue;
            const bool is_q = h < NH, is_v = h >= NH + NKV;
            const int g = is_q ? h : is_v ? h - NH - NKV : h - NH;
            if (!is_v) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int w = j / Vec16<T>::N, k = j % Vec16<T>::N;
                    const float a = lo[e][w].get(k), b = hi[e][w].get(k);
                    lo[e][w].set(k, __fsub_rn(__fmul_rn(a, c[j]), __fmul_rn(b, s[j])));
                    hi[e][w].set(k, __fadd_rn(__fmul_rn(b, c[j]), __fmul_rn(a, s[j])));
                }
            }
            T* dense = reinterpret_cast<T*>(is_q ? p.q_out : is_v ? p.v_out : p.k_out);
            T* pool = !is_q && row_off >= 0 ? reinterpret_cast<T*>(is_v ? p.v_pool : p.k_pool) + row_off + g * p.head_stride + d0 : nullptr;
            if (dense != nullptr) dense += (t * (is_q ? NH : NKV) + g) * hd + d0;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (dense != nullptr) {
                    store16(dense + w * Vec16<T>::N, lo[e][w]);
                    store16(dense + half + w * Vec16<T>::N, hi[e][w]);
                }
                if (pool != nullptr) {
                    store16(pool + w * Vec16<T>::N, lo[e][w]);
                    store16(pool + half + w * Vec16<T>::N, hi[e][w]);
                }
            }
        }
    }
}

// Items are (token, V dims, group of heads): the angles of the V dims are loaded once per group.
template <typename T, bool kv8, int V> __device__ __forceinline__ void rotate_rows(const RopeAppendParams& p, int cta, int ctas) {
    if constexpr (V == 8) {
        if (p.pairs) {
            rotate_pairs<T, kv8>(p, cta, ctas);
            return;
        }
    }
    const int hd = p.head_dim, cpr = hd / V, half = p.rot / 2, NH = p.n_heads, NKV = p.n_kv_heads;
    const bool pool16 = !kv8 && p.k_pool != nullptr;
    const uint32_t total = (uint32_t)p.n_tokens * p.by_groups.div * cpr;
    for (uint32_t i = cta * blockDim.x + threadIdx.x; i < total; i += ctas * blockDim.x) {
        const uint32_t tg = p.by_cpr.quot(i);
        const int d0 = (int)(i - tg * cpr) * V;
        const int64_t t = p.by_groups.quot(tg);
        const int first = p.h0 + (int)(tg - (uint32_t)t * p.by_groups.div) * p.heads_per_item;
        float c[V], s[V];
        const bool rotated = d0 < p.rot;
        if (rotated) {
            load_angles<V>(p.cos + t * half, p.rot, p.interleaved, d0, c);
            load_angles<V>(p.sin + t * half, p.rot, p.interleaved, d0, s);
        }
        const int64_t row_off = pool16 ? pool_row(p, p.slots[t]) : -1;
        for (int e = 0; e < p.heads_per_item; ++e) {
            const int h = first + e;
            if (h >= p.h1) break;
            const bool is_q = h < NH, is_v = h >= NH + NKV;
            const int g = is_q ? h : is_v ? h - NH - NKV : h - NH;
            const T* head = (is_q   ? reinterpret_cast<const T*>(p.q) + t * p.q_stride
                             : is_v ? reinterpret_cast<const T*>(p.v) + t * p.v_stride
                                    : reinterpret_cast<const T*>(p.k) + t * p.k_stride) + (int64_t)g * hd;
            float x[V];
            if (rotated && !is_v) rotate_vec<T, V>(head, p.rot, p.interleaved, d0, c, s, x);
            else load_vec<T, V>(head + d0, x);
            T* dense = reinterpret_cast<T*>(is_q ? p.q_out : is_v ? p.v_out : p.k_out);
            if (dense != nullptr) store_vec<T, V>(dense + (t * (is_q ? NH : NKV) + g) * hd + d0, x);
            if (!is_q && row_off >= 0) {
                T* pool = reinterpret_cast<T*>(is_v ? p.v_pool : p.k_pool);
                store_vec<T, V>(pool + row_off + g * p.head_stride + d0, x);
            }
        }
    }
}

// 16/32-bit pools, and the queries of a large step over an 8-bit pool.
template <typename T, bool kv8, int V> __global__ void __launch_bounds__(kAppendWarps * 32, 4) rope_rows_kernel(const RopeAppendParams p) {
    if (!p.overlap) pdl_launch_dependents();
    pdl_wait();
    if (p.overlap) pdl_launch_dependents();       // the append kernel of the same call may start: it reads the same inputs
    rotate_rows<T, kv8, V>(p, blockIdx.x, gridDim.x);
}
// A small step over an 8-bit pool, in one launch: CTAs [0, kv_ctas) append, the others take the queries.
template <typename T, typename KV, int V> __global__ void __launch_bounds__(kAppendWarps * 32, 2) rope_append_small_kernel(const RopeAppendParams p) {
    pdl_launch_dependents();
    pdl_wait();
    if ((int)blockIdx.x < p.kv_ctas) append_small<T, KV, V>(p, blockIdx.x);
    else rotate_rows<T, true, V>(p, blockIdx.x - p.kv_ctas, gridDim.x - p.kv_ctas);
}
// The append of a large step. It runs beside rope_rows_kernel, which was launched just before it and lets it start once the
// call's inputs exist; it completes after that kernel, so that the next one waits for both.
template <typename T, typename KV, int V> __global__ void __launch_bounds__(kLargeThreads, 6) append_large_kernel(const RopeAppendParams p) {
    if (!p.overlap) {
        pdl_launch_dependents();
        pdl_wait();
    }
    append_large<T, KV, V>(p, blockIdx.x);
    if (p.overlap) pdl_wait();
}

template <typename T, typename KV, int V> static int launch_rope_append(RopeAppendParams p, cudaStream_t st) {
    constexpr bool kv8 = !std::is_same<KV, NoKv8>::value;
    const dim3 threads(kAppendWarps * 32);
    int sms = device_sm_count();
    if (sms <= 0) sms = 148;
    p.planes = 2 * p.n_kv_heads;
    p.h0 = p.q_out != nullptr ? 0 : p.n_heads;
    p.h1 = (p.v_out || (!kv8 && p.k_pool)) ? p.n_heads + 2 * p.n_kv_heads : p.k_out ? p.n_heads + p.n_kv_heads : p.n_heads;
    p.pairs = V == 8 && !p.interleaved && p.rot == p.head_dim;
    p.heads_per_item = p.pairs ? 2 : 4;
    const int64_t groups = p.h1 > p.h0 ? (p.h1 - p.h0 + p.heads_per_item - 1) / p.heads_per_item : 0, cpr = p.head_dim / (p.pairs ? 2 * V : V);
    const int64_t items = p.n_tokens * groups * cpr;
    NS_REQUIRE(items < ((int64_t)1 << 31), NS_ERR_UNSUPPORTED, "rope_append: %lld tokens", (long long)p.n_tokens);
    if (groups > 0) {
        p.by_cpr = FastDiv((uint32_t)cpr);
        p.by_groups = FastDiv((uint32_t)groups);
    }
    int64_t ctas = (items + threads.x - 1) / threads.x;
    if (ctas > sms * 12) ctas = sms * 12;
    cudaError_t e = cudaSuccess;
    if constexpr (!kv8) {
        if (ctas > 0) e = launch_pdl(rope_rows_kernel<T, false, V>, dim3((unsigned)ctas), threads, 0, st, p);
    } else if (p.n_tokens <= kSmallStep) {
        p.kv_ctas = (int)((p.n_tokens * p.planes + kAppendWarps - 1) / kAppendWarps);
        e = launch_pdl(rope_append_small_kernel<T, KV, V>, dim3((unsigned)(ctas + p.kv_ctas)), threads, 0, st, p);
    } else {
        p.chunk = kAppendChunk;
        const int64_t n = (p.n_tokens + p.chunk - 1) / p.chunk * p.n_kv_heads;
        NS_REQUIRE(n < (1 << 30), NS_ERR_UNSUPPORTED, "rope_append: %lld tokens", (long long)p.n_tokens);
        p.overlap = ctas > 0 ? 1 : 0;
        if (ctas > 0) e = launch_pdl(rope_rows_kernel<T, true, V>, dim3((unsigned)ctas), threads, 0, st, p);
        if (e == cudaSuccess) e = launch_pdl(append_large_kernel<T, KV, V>, dim3((unsigned)n), dim3(kLargeThreads), 0, st, p);
    }
    if (e != cudaSuccess) return fail(NS_ERR_CUDA, "rope_append: launch failed: %s", cudaGetErrorString(e));
    return NS_OK;
}

template <typename T, int V> static int dispatch_pool(const RopeAppendParams& p, int pool_dtype, cudaStream_t st) {
    if (pool_dtype == NS_INT8) return launch_rope_append<T, KvInt8, V>(p, st);
    if (pool_dtype == NS_E4M3) return launch_rope_append<T, KvE4m3, V>(p, st);
    return launch_rope_append<T, NoKv8, V>(p, st);
}

// ------------------------------------------------------------------------------------------------ values of an 8-bit pool
// V dims per thread, one 16-byte store (two would leave every lane half of a 32-byte sector at a time); bound by the stores, the codes
// are a fifth of the traffic to fp32. Quotients by multiplication, not by three 64-bit divisions per thread. (An append of 61 rows and
// its pools read back, three launches: 7.3 -> 5.8 us by the two together.)
template <typename T, typename KV, int V>
__global__ void __launch_bounds__(256) kv_values_kernel(const uint8_t* pool, const float* scale, T* out, uint32_t total, FastDiv by_cpr,
                                                        FastDiv by_heads, FastDiv by_block, int64_t blk_stride, int64_t pos_stride,
                                                        int64_t head_stride, int64_t sc_blk, int64_t sc_head) {
    pdl_launch_dependents();
    pdl_wait();
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < total; i += gridDim.x * blockDim.x) {
        const uint32_t rh = by_cpr.quot(i), row = by_heads.quot(rh), b = by_block.quot(row);
        const uint32_t d0 = (i - rh * by_cpr.div) * V, h = rh - row * by_heads.div, off = row - b * by_block.div;
        const uint8_t* src = pool + b * blk_stride + off * pos_stride + h * head_stride + d0;
        const float s = scale[b * sc_blk + h * sc_head];
        float x[V];
        if constexpr (V == 1) {
            x[0] = KV::decode(src[0]) * s;
        } else {
#pragma unroll
            for (int c = 0; c < V / 4; ++c) {
                float y[4];
                KV::decode4(reinterpret_cast<const uint32_t*>(src)[c], y);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[4 * c + j] = y[j] * s;
            }
        }
        store_vec<T, V>(out + (int64_t)i * V, x);
    }
}

template <typename T, typename KV, int V>
static int launch_kv_values(const uint8_t* pool, const float* scale, T* out, int64_t blocks, int bs, int nkv, int hd, int64_t s0, int64_t s1,
                            int64_t s2, int64_t c0, int64_t c1, cudaStream_t st) {
    int sms = device_sm_count();
    if (sms <= 0) sms = 148;
    const int64_t per_block = (int64_t)bs * nkv * (hd / V), most = 0x7fffffffll / per_block;      // blocks of a launch: items in 31 bits
    NS_REQUIRE(most > 0, NS_ERR_UNSUPPORTED, "kv_values: blocks of %lld values", (long long)(per_block * V));
    for (int64_t b0 = 0; b0 < blocks; b0 += most) {
        const int64_t n = blocks - b0 < most ? blocks - b0 : most, items = n * per_block;
        int64_t ctas = (items + 255) / 256;
        if (ctas > sms * 8) ctas = sms * 8;
        const cudaError_t e = launch_pdl(kv_values_kernel<T, KV, V>, dim3((unsigned)ctas), dim3(256), 0, st, pool + b0 * s0, scale + b0 * c0,
                                         out + b0 * per_block * V, (uint32_t)items, FastDiv((uint32_t)(hd / V)), FastDiv((uint32_t)nkv),
                                         FastDiv((uint32_t)bs), s0, s1, s2, c0, c1);
        if (e != cudaSuccess) return fail(NS_ERR_CUDA, "kv_values: launch failed: %s", cudaGetErrorString(e));
    }
    return NS_OK;
}

}  // namespace ns

using namespace ns;

extern "C" int ns_rope_tables(const int64_t* positions, const float* inv_freq, double factor, float* cos_out, float* sin_out,
                              int64_t n_tokens, int32_t half, void* stream) {
    NS_REQUIRE(n_tokens >= 0 && half >= 0, NS_ERR_INVALID_ARG, "rope_tables: bad shape");
    if (n_tokens == 0 || half == 0) return NS_OK;
    NS_REQUIRE(positions && inv_freq && cos_out && sin_out, NS_ERR_INVALID_ARG, "rope_tables: null pointer");
    int sms = device_sm_count();
    if (sms <= 0) sms = 148;
    int64_t ctas = (n_tokens * half + 255) / 256;
    if (ctas > sms * 8) ctas = sms * 8;
    cudaError_t e = launch_pdl(rope_tables_kernel, dim3((unsigned)ctas), dim3(256), 0, (cudaStream_t)stream, positions, inv_freq, factor,
                               cos_out, sin_out, n_tokens * half, half);
    if (e != cudaSuccess) return fail(NS_ERR_CUDA, "rope_tables: launch failed: %s", cudaGetErrorString(e));
    return NS_OK;
}

extern "C" int ns_rope_append(const void* q, const void* k, const void* v, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                              const float* cos, const float* sin, int32_t rot_dim, int32_t interleaved, void* q_out, void* k_out,
                              void* v_out, void* k_pool, void* v_pool, float* k_scale, float* v_scale, const int64_t* slots,
                              int64_t n_tokens, int64_t n_slots, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                              int32_t block_size, int64_t pool_block_stride, int64_t pool_pos_stride, int64_t pool_head_stride,
                              int64_t scale_block_stride, int64_t scale_head_stride, int dtype, int pool_dtype, void* stream) {
    NS_REQUIRE(n_tokens >= 0 && n_heads >= 0 && n_kv_heads > 0 && head_dim > 0, NS_ERR_INVALID_ARG, "rope_append: bad shape");
    NS_REQUIRE(dtype == NS_BF16 || dtype == NS_F32, NS_ERR_UNSUPPORTED, "rope_append: dtype %d", dtype);
    NS_REQUIRE(rot_dim >= 0 && rot_dim % 2 == 0 && rot_dim <= head_dim, NS_ERR_INVALID_ARG,
               "rope_append: rotary dim %d must be even and at most head_dim %d", rot_dim, head_dim);
    NS_REQUIRE((k_pool == nullptr) == (v_pool == nullptr), NS_ERR_INVALID_ARG, "rope_append: need both pools or none");
    const bool kv8 = k_pool != nullptr && (pool_dtype == NS_INT8 || pool_dtype == NS_E4M3);
    NS_REQUIRE(k_pool == nullptr || kv8 || pool_dtype == dtype, NS_ERR_UNSUPPORTED, "rope_append: pool dtype %d with activations of dtype %d",
               pool_dtype, dtype);
    if (n_tokens == 0) return NS_OK;
    NS_REQUIRE(k && v && (q || n_heads == 0 || !q_out), NS_ERR_INVALID_ARG, "rope_append: null pointer");
    NS_REQUIRE(rot_dim == 0 || (cos && sin), NS_ERR_INVALID_ARG, "rope_append: rotary dim %d without tables", rot_dim);
    if (k_pool != nullptr) {
        NS_REQUIRE(slots, NS_ERR_INVALID_ARG, "rope_append: pools given without slots");
        NS_REQUIRE(block_size > 0 && n_slots >= 0, NS_ERR_INVALID_ARG, "rope_append: bad pool shape");
    }
    if (kv8) {
        NS_REQUIRE(k_scale && v_scale, NS_ERR_INVALID_ARG, "rope_append: an 8-bit pool needs its scales");
        NS_REQUIRE(block_size <= kAppendMaxBlock && (block_size & (block_size - 1)) == 0, NS_ERR_UNSUPPORTED,
                   "rope_append: 8-bit pools take blocks of 1, 2, 4 ... %d tokens, not %d", kAppendMaxBlock, block_size);
        NS_REQUIRE(n_tokens < (1 << 23) && n_slots < ((int64_t)1 << 31), NS_ERR_UNSUPPORTED, "rope_append: %lld tokens / %lld slots",
                   (long long)n_tokens, (long long)n_slots);
    }
    RopeAppendParams p = {};
    p.q = q; p.k = k; p.v = v; p.q_stride = q_stride; p.k_stride = k_stride; p.v_stride = v_stride;
    p.cos = cos; p.sin = sin; p.rot = rot_dim; p.interleaved = interleaved ? 1 : 0;
    p.q_out = n_heads > 0 ? q_out : nullptr; p.k_out = k_out; p.v_out = v_out; p.k_pool = k_pool; p.v_pool = v_pool;
    p.k_scale = k_scale; p.v_scale = v_scale; p.slots = slots; p.n_tokens = n_tokens; p.n_slots = n_slots;
    p.n_heads = n_heads; p.n_kv_heads = n_kv_heads; p.head_dim = head_dim; p.block_size = block_size > 0 ? block_size : 1;
    while ((1 << p.block_shift) < p.block_size) ++p.block_shift;
    if ((1 << p.block_shift) != p.block_size) p.block_shift = -1;         // (16/32-bit pools only)
    p.blk_stride = pool_block_stride; p.pos_stride = pool_pos_stride; p.head_stride = pool_head_stride;
    p.sc_blk_stride = scale_block_stride; p.sc_head_stride = scale_head_stride;
    const int kind = k_pool == nullptr ? dtype : pool_dtype;
    cudaStream_t st = (cudaStream_t)stream;
    // 8 dims at a time where every 8-dim piece of every buffer is 16-byte aligned (8-byte for codes) and rotated pieces lie
    // wholly on one side of a pair; one dim at a time otherwise.
    const int64_t e = dtype == NS_F32 ? 4 : 8;            // elements per 16 bytes
    uintptr_t a = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)v_out | (uintptr_t)cos | (uintptr_t)sin;
    bool wide = head_dim % 8 == 0 && (a & 15) == 0 && k_stride % e == 0 && v_stride % e == 0 && (q_stride % e == 0 || n_heads == 0) &&
                (interleaved ? rot_dim % 8 == 0 : rot_dim % 16 == 0);
    if (k_pool != nullptr) {
        const int64_t pe = kv8 ? 8 : e;
        wide = wide && (((uintptr_t)k_pool | (uintptr_t)v_pool) & (kv8 ? 7 : 15)) == 0 && pool_block_stride % pe == 0 &&
               pool_pos_stride % pe == 0 && pool_head_stride % pe == 0;
    }
    if (dtype == NS_BF16) return wide ? dispatch_pool<__nv_bfloat16, 8>(p, kind, st) : dispatch_pool<__nv_bfloat16, 1>(p, kind, st);
    return wide ? dispatch_pool<float, 8>(p, kind, st) : dispatch_pool<float, 1>(p, kind, st);
}

extern "C" int ns_kv_values(const void* pool, const float* scale, void* out, int64_t num_blocks, int32_t block_size, int32_t n_kv_heads,
                            int32_t head_dim, int64_t pool_block_stride, int64_t pool_pos_stride, int64_t pool_head_stride,
                            int64_t scale_block_stride, int64_t scale_head_stride, int dtype, int pool_dtype, void* stream) {
    NS_REQUIRE(num_blocks >= 0 && block_size > 0 && n_kv_heads > 0 && head_dim > 0, NS_ERR_INVALID_ARG, "kv_values: bad shape");
    NS_REQUIRE(dtype == NS_BF16 || dtype == NS_F32, NS_ERR_UNSUPPORTED, "kv_values: output dtype %d", dtype);
    NS_REQUIRE(pool_dtype == NS_INT8 || pool_dtype == NS_E4M3, NS_ERR_UNSUPPORTED, "kv_values: pool dtype %d is not an 8-bit one", pool_dtype);
    if (num_blocks == 0) return NS_OK;
    NS_REQUIRE(pool && scale && out, NS_ERR_INVALID_ARG, "kv_values: null pointer");
    cudaStream_t st = (cudaStream_t)stream;
    const bool wide = head_dim % 8 == 0 && ((uintptr_t)out & 15) == 0 && ((uintptr_t)pool & 7) == 0 && pool_block_stride % 8 == 0 &&
                      pool_pos_stride % 8 == 0 && pool_head_stride % 8 == 0;
#define NS_GO(T, KV)                                                                                                                          \
    return wide ? launch_kv_values<T, KV, 16 / (int)sizeof(T)>((const uint8_t*)pool, scale, (T*)out, num_blocks, block_size, n_kv_heads, head_dim,              \
                                             pool_block_stride, pool_pos_stride, pool_head_stride, scale_block_stride, scale_head_stride, st) \
                : launch_kv_values<T, KV, 1>((const uint8_t*)pool, scale, (T*)out, num_blocks, block_size, n_kv_heads, head_dim,              \
                                             pool_block_stride, pool_pos_stride, pool_head_stride, scale_block_stride, scale_head_stride, st)
    if (dtype == NS_BF16) {
        if (pool_dtype == NS_INT8) NS_GO(__nv_bfloat16, KvInt8);
        NS_GO(__nv_bfloat16, KvE4m3);
    }
    if (pool_dtype == NS_INT8) NS_GO(float, KvInt8);
    NS_GO(float, KvE4m3);
#undef NS_GO
}
