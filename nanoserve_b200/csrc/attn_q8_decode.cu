// Decode attention over 8-bit pools: every sequence of one query token, any number of query heads per KV head.
//
// Work   : a UNIT is (sequence, KV head, eight of its query heads); its keys are 16-token TILES. All tiles of the step in
//          unit order form one list that is cut evenly over the CTAs (one per SM) and, inside a CTA, evenly over the warps:
//          every warp streams the same number of tiles whatever the lengths. The cuts need no plan: each CTA scans the
//          sequence lengths itself. A CTA cut that falls near a unit's end moves onto it (no cross-CTA join then).
// Warp   : tiles go straight from global memory into registers, in the fragment layout of the matrix instructions, kDepth
//          tiles deep; nothing is staged through shared memory. The k index of an mma is free as long as both operands
//          agree, so a lane's 16-byte (K) / 8- or 16-byte (V) piece of a token's row IS its fragment share:
//            S^T[16 tokens x 8 heads] = K[16 x HD] . Q^T      A = K (lane: rows g and g + 8, dims 16 t .. 16 t + 15)
//            O^T[HD x 8 heads]       += V^T[HD x 16] . P^T    A = V^T (lane: tokens 2t, 2t+1, 2t+8, 2t+9, dims HD/8 g ..)
//          (g = lane / 4, t = lane % 4; m16n8k16, f16 operands, fp32 accumulators.) Eight heads are the n extent, so no half of
//          an instruction is empty, and P^T comes from S^T's accumulator by a register transpose (movmatrix).
// Codes  : int8 -> f16 by placing the byte under the exponent of 1024 and subtracting 1152; e4m3 by the hardware conversion:
//          both exact. Q is scaled by a power of two per head so that its largest element lies in [1, 2): f16 then holds a
//          bf16 q exactly (parts below 2^-17 of the largest aside). fp32 q is a sum of two f16 (22 bits), and so is P then.
// Softmax: s = q.k * (scale log2 e * 2^e_q * sk). The V scale joins the exponent: x = s + log2 sv, p = 2^(x - m) multiplies
//          V's codes and p / sv enters the denominator: P is then relative to the largest CONTRIBUTION and f16 keeps 11 bits
//          of everything that matters, however far apart the blocks' scales are. m follows the maximum of x lazily: it moves when
//          some x exceeds it by 2^8. Statistics and sums are fp32.
// Join   : pieces of a unit meet in shared memory (warps of a CTA, in order), then through fp32 partials in the workspace,
//          where the last CTA to arrive (one counter, nobody waits) joins them in CTA order: the result does not depend on
//          the order of arrival.
// Bound  : the stream itself runs at the copy rate (12 K cycles for 304 KB per SM); 8 K cycles before the first key is multiplied and
//          10 K of joins after the last are dependent loads. 48 rows U[128, 8192] of 14 / 2 heads of 64: 22.4 us, 45 MB (6.9 us at
//          the copy rate); 64 rows U[256, 4608] of 28 / 4 heads of 128: 38.2 us, 144 MB (22.0); 2 rows of 131 K keys of 12 / 2 heads
//          of 128: 41.3 us, 134 MB (20.5).
// Cuts   : a CTA takes at least two tiles per warp (one row of 300 keys: 7.3 us; at least one: 8.3; at least four: 7.1, and no
//          difference elsewhere). A cut moves onto a unit's end that is nearer than a join costs, or than half a share: 64 rows of
//          28 heads 38.0 us, 128 rows U[512, 4096] of 14 heads 27.8, 32 rows of 1,000 keys 10.9. By up to a quarter of a share: 39.8, 28.7,
//          12.4 (2 rows of 131 K: 40.5 against 41.5); by up to half: 43.4 for the first; not at all: 40.9, and 10.4 against 7.3 for
//          the row of 300 keys.
#include "attn_q8.cuh"

namespace ns {

namespace q8 {

constexpr float kLazy = 8.f;               // the exponent's reference may lag the maximum by this many powers of two
constexpr float kMinScale = 7.8886090522101181e-31f;    // 2^-100: a smaller V scale (zero included) counts as this
constexpr int kMaxSeqs = 8192;             // sequences per launch (prefix, length and table row of each in shared memory)

// Tiles a CTA streams in the time that a join across CTAs costs it (about 4 K cycles at 25 bytes per cycle and SM).
template <int HD> constexpr int kJoinTiles = HD == 64 ? 48 : 24;

template <int HD> struct Cfg;
template <> struct Cfg<64> { static constexpr int kWarps = 16, kDepth = 3; };
template <> struct Cfg<128> { static constexpr int kWarps = 12, kDepth = 2; };

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// One tile of a unit as a lane holds it.
template <int HD> struct Tile {
    static constexpr int KW = HD / 64, VW = HD / 32;        // 16-byte pieces per K row, words per V row
    uint4 k[2][KW];
    uint32_t v[4][VW];
};

// Streaming loads past L1: every byte is used once. (Not the read-only path: with programmatic launches the kernel before
// this one may still have been writing the pool when this one started.)
__device__ __forceinline__ uint4 ld16(const uint8_t* p) { return __ldcg(reinterpret_cast<const uint4*>(p)); }

}  // namespace q8

template <int HD, typename KV, bool F32>
__global__ void __launch_bounds__(q8::Cfg<HD>::kWarps * 32, 1) decode_q8_kernel(const Q8Params p, const int s_begin, const int n_rows,
                                                                               const int min_tiles) {
    using namespace q8;
    constexpr int NW = Cfg<HD>::kWarps, D = Cfg<HD>::kDepth, KW = HD / 64, VW = HD / 32, RS = HD + 4, THREADS = NW * 32;
    constexpr int QN = F32 ? 2 : 1;                          // f16 terms of q and of P
    extern __shared__ __align__(16) uint8_t smem_q8[];
    float* const slots = reinterpret_cast<float*>(smem_q8);              // [NW][2][8][RS] pieces of units
    float4* const tile_info = reinterpret_cast<float4*>(slots + NW * 2 * 8 * RS);   // [NW][2][32] {sk, log2 sv, 1 / sv, present}
    int* const prefix = reinterpret_cast<int*>(tile_info + NW * 64);     // [n_rows + 1] tiles (per unit of the row) before row r
    int* const row_len = prefix + n_rows + 1;                            // keys; -1: not a decode row
    int* const row_tab = row_len + n_rows;
    __shared__ int warp_total[NW], has_empty, n_chain, n_open;
    __shared__ int4 chain[2 * NW];         // units with pieces in this CTA: {row, vhead, first warp | slot << 8 | last warp << 16, kind}
    __shared__ int4 open_unit[2];          // units over several CTAs: [0] began in an earlier one, [1] begins here {row, vhead, first CTA, parts}
    __shared__ int open_last[2];

    // A mixed call's prefill kernel, launched next, does not wait for this one (it reads the same inputs and writes other rows):
    // it may start only once the inputs exist, that is after this kernel's own wait.
    if (!p.overlap_prefill) pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int G = gridDim.x, cta = blockIdx.x;
    const int sub = (p.group + 7) >> 3, VH = p.n_kv_heads * sub;
    if (tid == 0) has_empty = n_chain = n_open = 0;
    if (tid < 2) {
        open_unit[tid].w = 0;
        open_last[tid] = 0;
    }
    pdl_wait();
    if (p.overlap_prefill) pdl_launch_dependents();

    // ---- tiles before each row
    int total = 0;
    for (int base = 0; base < n_rows; base += THREADS) {
        const int r = base + tid, s = s_begin + r;
        int nt = 0, len = -1;
        if (r < n_rows) {
            int T = 1, q0 = s;
            if (p.cu_seqlens != nullptr) {
                q0 = p.cu_seqlens[s];
                T = p.cu_seqlens[s + 1] - q0;
            }
            const int tab = p.table_rows != nullptr ? p.table_rows[s] : s;
            len = q8_len(p, s);
            if (T != 1 || q0 < 0 || q0 >= p.n_tokens) len = -1;
            nt = len > 0 ? (len + 15) >> 4 : 0;
            row_len[r] = len;
            row_tab[r] = tab;
        }
        int inc = nt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int n = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += n;
        }
        if (base > 0) __syncthreads();                    // warp_total has been read
        if (lane == 31) warp_total[warp] = inc;
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const int v = warp_total[w];
            before += w < warp ? v : 0;
            all += v;
        }
        if (r < n_rows) prefix[r] = total + before + inc - nt;
        if (len == 0) has_empty = 1;
        total += all;
    }
    if (tid == 0) prefix[n_rows] = total;
    __syncthreads();
    const int W = total * VH;
    if (has_empty)                                        // rows without keys: zeros
        for (int r = cta; r < n_rows; r += G)
            if (row_len[r] == 0) {
                const int64_t q0 = p.cu_seqlens != nullptr ? p.cu_seqlens[s_begin + r] : s_begin + r;
                for (int e = tid; e < p.n_heads * HD; e += THREADS) {
                    if (F32) reinterpret_cast<float*>(p.out)[q0 * p.out_stride + e] = 0.f;
                    else reinterpret_cast<__nv_bfloat16*>(p.out)[q0 * p.out_stride + e] = __float2bfloat16_rn(0.f);
                }
            }
    if (W == 0) return;
    // row that holds tile x of the list: the last r with prefix[r] * VH <= x (empty rows share their successor's prefix). By one lane
    // for itself, or by a warp for one x: 32 rows are compared at once.
    auto row_of = [&](int x) -> int {
        int lo = 0, hi = n_rows;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] * VH <= x) lo = mid; else hi = mid;
        }
        return lo;
    };
    auto warp_row_of = [&](int x) -> int {
        int lo = 0, hi = n_rows, step = 1;                // prefix[lo] VH <= x; rows lo + step, lo + 2 step ... below hi are compared
        while (step * 32 < n_rows) step *= 32;
        for (;; step >>= 5) {
            const int r = lo + (lane + 1) * step;
            lo += step * __popc(__ballot_sync(0xffffffffu, r < hi && prefix[r] * VH <= x));
            if (step == 1) return lo;
        }
    };
    // First tile of CTA c: an even cut, moved onto the end or the start of a unit that is near (no cross-CTA join then).
    const int per = max((W + G - 1) / G, min_tiles), slack = min(per >> 1, kJoinTiles<HD>);
    auto even_cut = [&](int c) -> int {
        const long long want = (long long)c * per;
        return want >= W ? W : (int)want;
    };
    auto moved_cut = [&](int x, int r) -> int {           // r: row of x
        if (x > 0 && x < W) {
            const int nt = prefix[r + 1] - prefix[r], start = prefix[r] * VH;
            const int lo = start + (int)((unsigned)(x - start) / (unsigned)nt) * nt, hi = lo + nt;
            if (x - lo <= hi - x) {
                if (x - lo <= slack) x = lo;
            } else if (hi - x <= slack) {
                x = hi;
            }
        }
        return x;
    };
    auto cta_cut = [&](int c) -> int {
        const int x = even_cut(c);
        return moved_cut(x, row_of(x));
    };
    // every warp for itself: lane 0 the CTA's first tile, lane 1 the next CTA's
    const int e0 = even_cut(cta), e1 = even_cut(cta + 1), r0 = warp_row_of(e0), r1 = warp_row_of(e1);
    int c0 = moved_cut(lane & 1 ? e1 : e0, lane & 1 ? r1 : r0);
    const int c1 = __shfl_sync(0xffffffffu, c0, 1);
    c0 = __shfl_sync(0xffffffffu, c0, 0);
    const int n_mine = c1 - c0;
    if (n_mine <= 0) return;
    auto warp_cut = [&](int w) -> int { return c0 + (int)((unsigned)(n_mine * w) / (unsigned)NW); };
    const int a = warp_cut(warp), b = warp_cut(warp + 1);

    // ---- this warp's tiles
    if (a < b) {
        int r = warp_row_of(a), nt = prefix[r + 1] - prefix[r], us = prefix[r] * VH;
        int vh = (int)((unsigned)(a - us) / (unsigned)nt);
        us += vh * nt;
        int x = a;
        while (x < b) {
            const int len = row_len[r], kvh = vh / sub, h0 = (vh - kvh * sub) * 8, heads = min(8, p.group - h0);
            const int64_t q0 = p.cu_seqlens != nullptr ? p.cu_seqlens[s_begin + r] : s_begin + r;
            const int32_t* table = p.block_tables + (int64_t)row_tab[r] * p.table_stride;
            const int j0 = x - us, j1 = min(us + nt, b) - us;               // tiles [j0, j1) of the unit
            const uint8_t* kb = p.k_pool + kvh * p.head_stride + 16 * t;
            const uint8_t* vb = p.v_pool + kvh * p.head_stride + (HD / 8) * g;
            const float* ksc = p.k_scale + kvh * p.sc_head_stride;
            const float* vsc = p.v_scale + kvh * p.sc_head_stride;

            // Q's raw rows and the first block ids are requested together; K, V and the scales follow as soon as the ids are there, and
            // Q is converted while they travel. Lane (g, t) holds head g, dims 64 w + 16 t .. + 15, as B fragments.
            constexpr int QV = F32 ? 4 : 2;                   // 16-byte pieces per 16 dims
            uint4 qraw[KW * QV];
#pragma unroll
            for (int w = 0; w < KW; ++w)
#pragma unroll
                for (int c = 0; c < QV; ++c) {
                    const int64_t o = q0 * p.q_stride + (int64_t)(kvh * p.group + h0 + min(g, heads - 1)) * HD + 64 * w + 16 * t;
                    qraw[w * QV + c] = F32 ? *reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p.q) + o + 4 * c)
                                           : *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.q) + o + 8 * c);
                }
            // block ids of 32 tiles at a time, one per lane, the next 32 requested a batch ahead; their scales go to shared memory
            auto raw_id = [&](int base) -> int { return base + lane < j1 ? table[(base + lane) * 16 >> p.block_shift] : -1; };
            float4* const info = tile_info + warp * 64;
            int id_base = j0, id = raw_id(j0), id_next = raw_id(j0 + 32);
            if ((unsigned)id >= (unsigned)p.num_blocks) id = -1;
            float sk, sv;
            auto load_scales = [&]() {
                sk = id >= 0 ? ksc[(int64_t)id * p.sc_blk_stride] : 0.f;
                sv = id >= 0 ? vsc[(int64_t)id * p.sc_blk_stride] : 1.f;
            };
            auto put_scales = [&]() {                         // (the older batch of the two in `info` may still be read)
                const float svf = sv < kMinScale ? kMinScale : sv;
                info[(((id_base - j0) >> 5) & 1) * 32 + lane] = make_float4(sk, __log2f(svf), __fdividef(1.f, svf), id >= 0 ? 1.f : 0.f);
                __syncwarp();
            };
            Tile<HD> ring[D];
            const int64_t row_k = g * p.pos_stride, row_k8 = 8 * p.pos_stride, row_v = 2 * t * p.pos_stride;
            auto load = [&](Tile<HD>& T, int j) {
                if (j - id_base >= 32) {
                    id_base = j;
                    id = (unsigned)id_next >= (unsigned)p.num_blocks ? -1 : id_next;
                    id_next = raw_id(j + 32);
                    load_scales();
                    put_scales();
                }
                const int blk = __shfl_sync(0xffffffffu, id, j - id_base);
                int64_t off = (int64_t)max(blk, 0) * p.blk_stride;
                if (p.block_size != 16) off += (int64_t)((j * 16) & (p.block_size - 1)) * p.pos_stride;
                const uint8_t* ks = kb + off + row_k;
                const uint8_t* vs = vb + off + row_v;
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int w = 0; w < KW; ++w) T.k[e][w] = ld16(ks + e * row_k8 + 64 * w);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint8_t* src_v = vs + (e & 1) * p.pos_stride + (e >> 1) * row_k8;
                    if constexpr (HD == 64) {
                        const uint2 v = __ldcg(reinterpret_cast<const uint2*>(src_v));
                        T.v[e][0] = v.x;
                        T.v[e][1] = v.y;
                    } else {
                        const uint4 v = ld16(src_v);
                        T.v[e][0] = v.x;
                        T.v[e][1] = v.y;
                        T.v[e][2] = v.z;
                        T.v[e][3] = v.w;
                    }
                }
            };
#pragma unroll
            for (int d = 0; d < D; ++d)
                if (j0 + d < j1) load(ring[d], j0 + d);
            load_scales();

            uint32_t qf[QN][4 * KW][2];
            float f0, f1;                                     // score factors of heads 2t and 2t + 1
            {
                float qx[16 * KW];
#pragma unroll
                for (int i = 0; i < 16 * KW; ++i) {
                    if constexpr (F32) {
                        const uint4 u = qraw[i >> 2];
                        qx[i] = __uint_as_float((i & 3) == 0 ? u.x : (i & 3) == 1 ? u.y : (i & 3) == 2 ? u.z : u.w);
                    } else {
                        const uint4 u = qraw[i >> 3];
                        const uint32_t word = ((i >> 1) & 3) == 0 ? u.x : ((i >> 1) & 3) == 1 ? u.y : ((i >> 1) & 3) == 2 ? u.z : u.w;
                        qx[i] = __uint_as_float((i & 1) ? (word & 0xffff0000u) : (word << 16));
                    }
                }
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < 16 * KW; ++i) top = fmaxf(top, fabsf(qx[i]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                int e = (int)((uint32_t)__float_as_int(top) >> 23) - 127;     // NaN elements stay NaN whatever e is
                e = top == 0.f || e > 127 ? 0 : min(max(e, -126), 126);
                const float mult = __int_as_float((127 - e) << 23), back = __int_as_float((127 + e) << 23);
#pragma unroll
                for (int i = 0; i < 16 * KW; ++i) qx[i] *= mult;
#pragma unroll
                for (int ks = 0; ks < 4 * KW; ++ks)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float u = qx[4 * ks + 2 * c], v = qx[4 * ks + 2 * c + 1];
                        const uint32_t hi = pack_f16x2(u, v);
                        qf[0][ks][c] = hi;
                        if (F32) {
                            const float2 r2 = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                            qf[QN - 1][ks][c] = pack_f16x2(u - r2.x, v - r2.y);
                        }
                    }
                f0 = p.scale_log2 * __shfl_sync(0xffffffffu, back, 8 * t);
                f1 = p.scale_log2 * __shfl_sync(0xffffffffu, back, 8 * t + 4);
            }
            put_scales();

            float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
            float o[HD / 16][4];
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

            auto compute = [&](Tile<HD>& T, int j) {
                const float4 ti = info[(j - j0) & 63];
                const int valid = ti.w != 0.f ? min(16, len - 16 * j) : 0;
                float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    const uint32_t ka[4] = {T.k[0][w].x, T.k[0][w].y, T.k[0][w].z, T.k[0][w].w};
                    const uint32_t kc[4] = {T.k[1][w].x, T.k[1][w].y, T.k[1][w].z, T.k[1][w].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t a0, a1, a2, a3;
                        expand<KV>(ka[i], a0, a2);
                        expand<KV>(kc[i], a1, a3);
#pragma unroll
                        for (int n = 0; n < QN; ++n) mma_f16(s, a0, a1, a2, a3, qf[n][4 * w + i][0], qf[n][4 * w + i][1]);
                    }
                }
                const float k0 = f0 * ti.x, k1 = f1 * ti.x;
                float x0 = fmaf(s[0], k0, ti.y), x1 = fmaf(s[1], k1, ti.y), x2 = fmaf(s[2], k0, ti.y), x3 = fmaf(s[3], k1, ti.y);
                if (valid < 16) {                           // the row's last tile, or a block that is not there
                    if (g >= valid) x0 = x1 = -INFINITY;
                    if (g + 8 >= valid) x2 = x3 = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (2 * t + (e & 1) + 8 * (e >> 1) >= valid) {
#pragma unroll
                            for (int w = 0; w < VW; ++w) T.v[e][w] = 0u;      // 0 x NaN must not reach the sum
                        }
                }
                if (__any_sync(0xffffffffu, x0 > m0 + kLazy || x2 > m0 + kLazy || x1 > m1 + kLazy || x3 > m1 + kLazy)) {
                    float n0 = fmaxf(x0, x2), n1 = fmaxf(x1, x3);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, d));
                        n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, d));
                    }
                    n0 = fmaxf(m0, n0);
                    n1 = fmaxf(m1, n1);
                    const float al0 = n0 == -INFINITY ? 1.f : ex2(m0 - n0), al1 = n1 == -INFINITY ? 1.f : ex2(m1 - n1);
                    m0 = n0;
                    m1 = n1;
                    l0 *= al0;
                    l1 *= al1;
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i) {
                        o[i][0] *= al0;
                        o[i][1] *= al1;
                        o[i][2] *= al0;
                        o[i][3] *= al1;
                    }
                }
                const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
                const float p0 = ex2(x0 - r0), p1 = ex2(x1 - r1), p2 = ex2(x2 - r0), p3 = ex2(x3 - r1);
                l0 = fmaf(p0 + p2, ti.z, l0);
                l1 = fmaf(p1 + p3, ti.z, l1);
                uint32_t pb[QN][2];
                {
                    const uint32_t u = pack_f16x2(p0, p1), v = pack_f16x2(p2, p3);
                    pb[0][0] = transpose8x8(u);
                    pb[0][1] = transpose8x8(v);
                    if (F32) {
                        const float2 a2 = __half22float2(*reinterpret_cast<const __half2*>(&u)), b2 = __half22float2(*reinterpret_cast<const __half2*>(&v));
                        pb[QN - 1][0] = transpose8x8(pack_f16x2(p0 - a2.x, p1 - a2.y));
                        pb[QN - 1][1] = transpose8x8(pack_f16x2(p2 - b2.x, p3 - b2.y));
                    }
                }
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    // dims 4w .. 4w+3 of this lane: tokens 2t, 2t+1 (lo) and 2t+8, 2t+9 (hi), one dim per f16 pair
                    uint32_t d0l, d1l, d2l, d3l, d0h, d1h, d2h, d3h;
                    expand<KV>(__byte_perm(T.v[0][w], T.v[1][w], 0x5140), d0l, d1l);
                    expand<KV>(__byte_perm(T.v[0][w], T.v[1][w], 0x7362), d2l, d3l);
                    expand<KV>(__byte_perm(T.v[2][w], T.v[3][w], 0x5140), d0h, d1h);
                    expand<KV>(__byte_perm(T.v[2][w], T.v[3][w], 0x7362), d2h, d3h);
#pragma unroll
                    for (int n = 0; n < QN; ++n) {
                        mma_f16(o[2 * w], d0l, d1l, d0h, d1h, pb[n][0], pb[n][1]);
                        mma_f16(o[2 * w + 1], d2l, d3l, d2h, d3h, pb[n][0], pb[n][1]);
                    }
                }
            };
            for (int j = j0; j < j1; j += D) {
#pragma unroll
                for (int d = 0; d < D; ++d)
                    if (j + d < j1) {
                        compute(ring[d], j + d);
                        if (j + d + D < j1) load(ring[d], j + d + D);
                    }
            }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, d);
                l1 += __shfl_xor_sync(0xffffffffu, l1, d);
            }
            // ---- whole unit in this warp: write it; else leave the piece in shared memory
            if (j0 == 0 && j1 == nt) {
                const float i0 = l0 == 0.f ? 0.f : 1.f / l0, i1 = l1 == 0.f ? 0.f : 1.f / l1;
                const int64_t ob = q0 * p.out_stride + (int64_t)(kvh * p.group + h0) * HD + (HD / 8) * g;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (2 * t + e >= heads) continue;
                    const float inv = e ? i1 : i0;
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        const float4 v = make_float4(o[2 * w][e] * inv, o[2 * w][2 + e] * inv, o[2 * w + 1][e] * inv, o[2 * w + 1][2 + e] * inv);
                        const int64_t at = ob + (int64_t)(2 * t + e) * HD + 4 * w;
                        if (F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = v;
                        else *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + at) =
                                 make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
                    }
                }
            } else {
                const int slot = us < a ? 0 : 1;              // 0: the unit began before this warp's range
                float* dst = slots + (warp * 2 + slot) * 8 * RS;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float* row = dst + (2 * t + e) * RS + (HD / 8) * g;
#pragma unroll
                    for (int w = 0; w < VW; ++w)
                        *reinterpret_cast<float4*>(row + 4 * w) = make_float4(o[2 * w][e], o[2 * w][2 + e], o[2 * w + 1][e], o[2 * w + 1][2 + e]);
                    if (g == 0) *reinterpret_cast<float2*>(dst + (2 * t + e) * RS + HD) = make_float2(e ? m1 : m0, e ? l1 : l0);
                }
                if (lane == 0 && x == max(us, c0)) {          // the first warp of the unit in this CTA lists the unit
                    int last = warp;
                    const int end = min(us + nt, c1);
                    while (warp_cut(last + 1) < end) ++last;
                    const int kind = us >= c0 ? (us + nt <= c1 ? 1 : 3) : 2;      // 1 whole, 2 began in an earlier CTA, 3 begins here and ends in a later one
                    chain[atomicAdd(&n_chain, 1)] = make_int4(r, vh, warp | slot << 8 | last << 16, kind);
                    if (kind >= 2) {
                        open_unit[kind - 2] = make_int4(r, vh, 0, 1);
                        atomicAdd(&n_open, 1);
                    }
                }
            }
            x = us + j1;
            us += nt;
            if (++vh == VH) {
                vh = 0;
                do { ++r; } while (r < n_rows && prefix[r + 1] == prefix[r]);
                if (r < n_rows) nt = prefix[r + 1] - prefix[r];
            }
        }
    }
    __syncthreads();

    // ---- join the pieces of this CTA's warps: (unit, head) items over the warps; a lane is a piece for the weights and HD / 32
    // columns for the sums
    constexpr int C = HD / 32;
    float* const partials = reinterpret_cast<float*>(p.ws + p.L.partials);       // [CTA][2][8][RS]
    for (int item = warp; item < n_chain * 8; item += NW) {
        const int4 ch = chain[item >> 3];
        const int h = item & 7, kvh = ch.y / sub, h0 = (ch.y - kvh * sub) * 8;
        if (h >= min(8, p.group - h0)) continue;
        const int w0 = ch.z & 0xff, slot = (ch.z >> 8) & 0xff, w1 = ch.z >> 16;
        const float* const piece0 = slots + ((w0 * 2 + slot) * 8 + h) * RS;      // of the first warp; the others' are their slot 0
        float2 ml = make_float2(-INFINITY, 0.f);
        if (w0 + lane <= w1 && warp_cut(w0 + lane) < warp_cut(w0 + lane + 1)) 
            ml = *reinterpret_cast<const float2*>((lane == 0 ? piece0 : slots + ((w0 + lane) * 16 + h) * RS) + HD);
        const float m = warp_max(ml.x);
        const float wt = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
        const float l = warp_sum(ml.y == 0.f ? 0.f : wt * ml.y);
        float acc[C];
#pragma unroll
        for (int i = 0; i < C; ++i) acc[i] = 0.f;
        // four pieces' columns are requested before the first is used (a piece without tiles, or one that weighs nothing, is skipped:
        // its slot may hold anything)
#pragma unroll 1
        for (int k0 = 0; k0 <= w1 - w0; k0 += 4) {
            float v[4][C], f[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                f[k] = __shfl_sync(0xffffffffu, wt, k0 + k);              // (lanes past the last piece: 0)
                const float* src = (k0 + k == 0 ? piece0 : slots + ((w0 + k0 + k) * 16 + h) * RS) + C * lane;
#pragma unroll
                for (int i = 0; i < C; i += 2) {
                    const float2 u = f[k] != 0.f ? *reinterpret_cast<const float2*>(src + i) : make_float2(0.f, 0.f);
                    v[k][i] = u.x;
                    v[k][i + 1] = u.y;
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < C; ++i) acc[i] = fmaf(f[k], v[k][i], acc[i]);
        }
        if (ch.w == 1) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int64_t q0 = p.cu_seqlens != nullptr ? p.cu_seqlens[s_begin + ch.x] : s_begin + ch.x;
            const int64_t at = q0 * p.out_stride + (int64_t)(kvh * p.group + h0 + h) * HD + C * lane;
#pragma unroll
            for (int i = 0; i < C; i += 2) {
                if (F32) *reinterpret_cast<float2*>(reinterpret_cast<float*>(p.out) + at + i) = make_float2(acc[i] * inv, acc[i + 1] * inv);
                else *reinterpret_cast<uint32_t*>(reinterpret_cast<__nv_bfloat16*>(p.out) + at + i) = pack_bf16x2(acc[i] * inv, acc[i + 1] * inv);
            }
        } else {
            float* dst = partials + ((size_t)(cta * 2 + (ch.w == 3)) * 8 + h) * RS;
#pragma unroll
            for (int i = 0; i < C; i += 2) __stcg(reinterpret_cast<float2*>(dst + C * lane + i), make_float2(acc[i], acc[i + 1]));
            if (lane == 0) __stcg(reinterpret_cast<float2*>(dst + HD), make_float2(m, l));
        }
    }

    // ---- units over several CTAs: the last one to arrive joins the pieces in CTA order. Warps 0 and 1 count the arrivals (the
    // barrier orders the CTA's partials before them, the atomic releases them and acquires the others').
    if (n_open == 0) return;
    __syncthreads();
    int* const counters = reinterpret_cast<int*>(p.ws + p.L.q8_counters);
    if (warp < 2 && open_unit[warp].w != 0) {
        const int4 u = open_unit[warp];
        const int nt = prefix[u.x + 1] - prefix[u.x], us = prefix[u.x] * VH + u.y * nt, ue = us + nt;
        // CTAs that hold the unit's first and last tile: a cut moves by less than half a share, so they are among the neighbours of
        // the even ones (lanes 0..3 try the first, 4..7 the last)
        const int c = min((lane < 4 ? us : ue - 1) / per - 1 + (lane & 3), G);
        const int cut = lane < 8 && c >= 0 ? cta_cut(c) : 0;
        const unsigned first = __ballot_sync(0xffffffffu, lane < 4 && (c < 0 || cut <= us)), last = __ballot_sync(0xffffffffu, lane >= 4 && lane < 8 && (c < 0 || cut < ue));
        const int f = us / per - 1 + __popc(first) - 1, l = (ue - 1) / per - 1 + __popc(last) - 1;
        if (lane == 0) {
            int before;
            asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(&counters[f]) : "memory");
            if (before == l - f) {
                counters[f] = 0;
                open_unit[warp] = make_int4(u.x, u.y, f, l - f + 1);
                open_last[warp] = 1;
            }
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
        if (!open_last[k]) continue;
        const int4 u = open_unit[k];
        const int f = u.z, parts = u.w;
        const int kvh = u.y / sub, h0 = (u.y - kvh * sub) * 8, heads = min(8, p.group - h0);
        // thread = (share of the pieces, head, four columns); piece i lies in CTA f + i, the first CTA's is its "begins here" piece.
        // B pieces' statistics and columns are requested at once.
        constexpr int E4 = 8 * HD / 4, GR = THREADS / E4, B = GR > 1 ? 8 : 16;
        static_assert(GR >= 1, "one float4 column per thread at least");
        const int e = tid % E4, gr = tid / E4, h = e / (HD / 4), c4 = e % (HD / 4);
        float m = -INFINITY, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (gr < GR && h < heads)
            for (int i0 = gr; i0 < parts; i0 += B * GR) {
                float2 ml[B];
                float4 v[B];
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    const int q = i0 + i * GR;
                    const float* src = partials + ((size_t)((f + q) * 2 + (q == 0)) * 8 + h) * RS;
                    ml[i] = q < parts ? __ldcg(reinterpret_cast<const float2*>(src + HD)) : make_float2(-INFINITY, 0.f);
                    v[i] = q < parts ? __ldcg(reinterpret_cast<const float4*>(src) + c4) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                float mn = m;
#pragma unroll
                for (int i = 0; i < B; ++i) mn = fmaxf(mn, ml[i].x);
                const float ref = mn == -INFINITY ? 0.f : mn, al = ex2(m - ref);
                m = mn;
                l *= al;
                acc.x *= al;
                acc.y *= al;
                acc.z *= al;
                acc.w *= al;
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    const float wt = ml[i].x == -INFINITY ? 0.f : ex2(ml[i].x - ref);
                    l = fmaf(wt, ml[i].y, l);
                    acc.x = fmaf(wt, v[i].x, acc.x);
                    acc.y = fmaf(wt, v[i].y, acc.y);
                    acc.z = fmaf(wt, v[i].z, acc.z);
                    acc.w = fmaf(wt, v[i].w, acc.w);
                }
            }
        if (GR > 1) {                                        // the shares meet in shared memory, in order
            float* const red = slots;                        // [THREADS][6]: nothing else lives there any more
            if (gr > 0) {
                float* mine = red + tid * 6;
                mine[0] = acc.x, mine[1] = acc.y, mine[2] = acc.z, mine[3] = acc.w, mine[4] = m, mine[5] = l;
            }
            __syncthreads();
            if (gr == 0)
                for (int i = 1; i < GR; ++i) {
                    const float* o = red + (tid + i * E4) * 6;
                    const float mn = fmaxf(m, o[4]), ref = mn == -INFINITY ? 0.f : mn, wa = ex2(m - ref), wb = ex2(o[4] - ref);
                    acc.x = acc.x * wa + o[0] * wb;
                    acc.y = acc.y * wa + o[1] * wb;
                    acc.z = acc.z * wa + o[2] * wb;
                    acc.w = acc.w * wa + o[3] * wb;
                    l = l * wa + o[5] * wb;
                    m = mn;
                }
        }
        if (gr == 0 && h < heads) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int64_t q0 = p.cu_seqlens != nullptr ? p.cu_seqlens[s_begin + u.x] : s_begin + u.x;
            const int64_t at = q0 * p.out_stride + (int64_t)(kvh * p.group + h0 + h) * HD + 4 * c4;
            if (F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            else *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + at) =
                     make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
        }
        __syncthreads();
    }
}

// Layouts the decode kernel takes; everything else is the scalar kernel's.
bool q8_decode_supported(const Q8Params& p, int dtype) {
    const int64_t qa = dtype == NS_F32 ? 4 : 8;
    if (p.head_dim != 64 && p.head_dim != 128) return false;
    if (p.block_size < 16 || p.block_shift < 0) return false;
    if (((uintptr_t)p.k_pool | (uintptr_t)p.v_pool | (uintptr_t)p.q) & 15) return false;
    if (((uintptr_t)p.out & (dtype == NS_F32 ? 15 : 7)) || p.out_stride % 4 || p.q_stride % qa) return false;
    if (p.blk_stride % 16 || p.pos_stride % 16 || p.head_stride % 16) return false;
    const int64_t tiles = (int64_t)p.table_width * (p.block_size / 16) * p.n_kv_heads * ((p.group + 7) / 8);
    return tiles * (p.n_seqs < q8::kMaxSeqs ? p.n_seqs : q8::kMaxSeqs) < ((int64_t)1 << 30);
}

template <int HD, typename KV, bool F32> static int launch_decode_q8(const Q8Params& p, cudaStream_t st) {
    constexpr int NW = q8::Cfg<HD>::kWarps;
    int grid = p.sm_count;
    const int cap = (int)((int64_t)kMaxDecodeCtas * 2 * p.n_heads * (HD + 4) / (2 * 8 * (HD + 4)));      // CTAs the partials hold
    if (grid > cap) grid = cap;
    if (grid > kMaxDecodeCtas) grid = kMaxDecodeCtas;
    for (int s0 = 0; s0 < p.n_seqs; s0 += q8::kMaxSeqs) {
        const int n = p.n_seqs - s0 < q8::kMaxSeqs ? p.n_seqs - s0 : q8::kMaxSeqs;
        const size_t smem = (size_t)NW * 2 * 8 * (HD + 4) * 4 + (size_t)NW * 64 * 16 + (size_t)(3 * n + 1) * 4;
        static SmemOptIn optin;
        if (optin.needs(smem)) {
            cudaError_t e = cudaFuncSetAttribute(decode_q8_kernel<HD, KV, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e != cudaSuccess) return fail(NS_ERR_CUDA, "decode_q8: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
            optin.done(smem);
        }
        // at least two tiles per warp: splitting further costs a cross-CTA join and saves less (figures above)
        cudaError_t e = launch_pdl(decode_q8_kernel<HD, KV, F32>, dim3((unsigned)grid), dim3(NW * 32), smem, st, p, s0, n, 2 * NW);
        if (e != cudaSuccess) return fail(NS_ERR_CUDA, "decode_q8: launch failed: %s", cudaGetErrorString(e));
    }
    return NS_OK;
}

int launch_q8_decode(const Q8Params& p, int dtype, int pool_dtype, cudaStream_t st) {
#define NS_GO(HD)                                                                                                                \
    if (dtype == NS_F32) return pool_dtype == NS_INT8 ? launch_decode_q8<HD, KvInt8, true>(p, st) : launch_decode_q8<HD, KvE4m3, true>(p, st); \
    return pool_dtype == NS_INT8 ? launch_decode_q8<HD, KvInt8, false>(p, st) : launch_decode_q8<HD, KvE4m3, false>(p, st)
    if (p.head_dim == 64) { NS_GO(64); }
    NS_GO(128);
#undef NS_GO
}

}  // namespace ns
