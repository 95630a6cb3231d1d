// Prefill-chunk attention over 8-bit pools on the 5th-generation tensor cores (tcgen05), accumulators in tensor memory.
//
// Work item = (sequence, 32 query tokens, eight query heads of a KV head): two UMMA tiles A and B of 128 rows (row r of a tile =
// token r / 8, head r % 8) against the same key tiles of 64.
//   S[128 x 64]  = Q[128 x HD] . K_tile[64 x HD]^T      f16 operands, fp32 accumulators
//   O[128 x HD] += P[128 x 64] . V_tile[64 x HD]
// The codes become f16 on their way into shared memory (exact for int8 and e4m3, so K and V are never rounded): six converting
// warps read 16-byte pieces of the pool's rows, one tile ahead, and store them in the swizzled layout the UMMA descriptors
// expect; both Q tiles use them. Rows past the sequence and blocks outside the pool become zeros there. Scales stay out of the
// operands:
//   x = s * (scale log2 e * 2^e_q * sk) + log2 sv,   P = 2^(x - m),   l += sum(P) / sv   per block of 16 keys
// (Q is scaled by a power of two per row, P is relative to the row's largest contribution; see attn_q8_decode.cu.)
// Four warpgroups, 512 threads, one CTA per SM (all 512 columns of its tensor memory):
//   warps 0-3, 4-7   softmax and output of tiles A and B, one thread per row; 176 registers
//   warps 8, 9       issue the tcgen05.mma of tile A, of tile B: the warp runs converged on uniform values, one elected lane issues
//                    (a lone lane, with its operands moved to uniform registers one by one: 310 us against 307, mixed 68 against 64)
//   warps 10-15      convert K and V tiles. 80 registers a thread: 2 (176 + 80) 128 = 128 * 512, what the block was launched with
// Pipeline per tile: S runs two key tiles ahead in two buffers; P(kt) goes back into the columns that S(kt) was read from and is the
// A operand from there, so it never passes through shared memory (in shared memory, double buffered: 356 us against 322). S(kt + 2)
// overwrites it after PV(kt): one warp issues both, and the tensor cores keep its order. O stays in tensor memory and is rescaled only
// when a row's reference has to move; A and B fill each other's gaps. Barriers are asked for ahead of the wait. Every mbarrier wait is
// bounded: on expiry the CTA counts an error in the plan header (ns_collect_status), skips its stores, frees its tensor memory and
// returns.
// What bounds it (2,048 tokens on 6,001 keys, 28 / 4 heads of 128: 302 us, 682 TFLOP/s of the rows that exist; 256 items on 148 SMs
// are two rounds, the second three quarters full, and seven of eight head slots are used): with
// the softmax and the conversion cut out the same chain of waits and products takes 208 us, with the softmax alone cut out 239, with
// the conversion alone cut out 298. Q is read again for every 64 keys, which makes 48 cycles of shared memory for 32 of arithmetic in Q.K
// (scores of 128 keys, double buffered, and O would need 384 of the 256 columns a tile has; single-buffered: 445 us). Two softmax warpgroups per tile taking turns, with the scores read twice so that 768
// threads fit the registers: 372 us.
#include "attn_q8.cuh"
#include "tc_common.cuh"

namespace ns {

namespace q8p {

using namespace tc;

constexpr int kRows = 128, kKeys = 64, kThreads = 512, kConv = 192;    // rows of a Q tile, keys per tile, threads, converting threads
constexpr int kTokens = 2 * kPrefillTileTokens;                        // query tokens per item
constexpr int kConvWarps = kConv / 32;
constexpr int kRegsSoftmax = 176, kRegsOther = 80;
constexpr int kSplitTiles = 8;      // key tiles from which an item is split
constexpr int kScaleRing = 8;       // a converter is at most five tiles ahead of the slowest softmax thread
template <int HD> struct Depth {
    static constexpr int K = 4, V = 4;
    // mbarriers: S0 S1, PV0 PV1, P0 P1 ready of each Q tile | K full | V full | K free | V free | scales of a key tile
    static constexpr int BarS = 0, BarPV = 4, BarPReady = 8, BarKFull = 12, BarVFull = BarKFull + K, BarKFree = BarVFull + V,
                         BarVFree = BarKFree + K, BarScale = BarVFree + V, Bars = BarScale + kScaleRing;
};
constexpr int kTailBytes = 1152;    // mbarriers, two words, the scale ring [8][3][4], the NaN-key ring [8][6]
constexpr float kLazy = 8.f;
constexpr float kMinScale = 7.8886090522101181e-31f;    // 2^-100

// Instruction descriptor for kind::f16: fp32 accumulate, f16 A and B, M = 128, N = n.
__host__ __device__ constexpr uint32_t instr_desc(bool b_mn_major, int n) {
    return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    // (no memory clobber: only the fence before the barrier arrival orders these stores, and loads may move across them)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d));
}
// Largest of three (NaN operands are passed over, as by fmaxf).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t cluster_ctas() {
    uint32_t n;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
    return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctaid.x;" : "=r"(r));
    return r;
}
// All threads of the cluster's CTAs that have not exited (no role waits here for another without a limit of its own before).
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_address(uint32_t saddr, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    return a;
}
__device__ __forceinline__ void st_cluster16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// One lane of a converged warp, the same one at every call.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// Every lane's generic-proxy stores become visible to the tensor cores, then one arrival for the warp.
__device__ __forceinline__ void warp_arrive(uint32_t mbar_saddr) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(mbar_saddr);
}
// Named barriers 1 and 2: a tile's softmax threads and its issuing warp meet once, when Q is in place.
__device__ __forceinline__ void q_ready_barrier(int tile) { asm volatile("bar.sync %0, %1;" ::"r"(1 + tile), "r"(kRows + 32) : "memory"); }

}  // namespace q8p

// SPLIT: the CTAs of a cluster share an item, each with its part of the keys.
template <int HD, typename KV, bool SPLIT>
__global__ void __launch_bounds__(q8p::kThreads, 1) prefill_q8_kernel(const Q8Params p) {
    using namespace q8p;
    using D = Depth<HD>;
    constexpr int kStagesK = D::K, kStagesV = D::V;
    constexpr int ATOMS = HD / 64;
    constexpr int Q_BYTES = kRows * 128 * ATOMS, KV_BYTES = kKeys * 128 * ATOMS;
    constexpr uint32_t COL_TILE = 2 * kKeys + HD, COL_O = 2 * kKeys, TMEM_COLS = 512;      // per Q tile: S0, S1, O
    static_assert(D::Bars * 8 + 16 + kScaleRing * (48 + 8 * kConvWarps) <= kTailBytes, "the tail holds the barriers, two words and the rings");
    // V codes that are NaN (e4m3 only): 0 x NaN would reach rows that must not see the key, so the operand gets 0 there and the
    // key goes on a list: the score of a row that does see it becomes NaN (its whole output row then is).
    constexpr bool kNanCodes = std::is_same<KV, KvE4m3>::value;
    extern __shared__ __align__(1024) uint8_t smem_raw[];

    const PlanHeader* hdr = reinterpret_cast<const PlanHeader*>(p.ws + p.L.header);
    const int sub = (p.group + 7) >> 3;
    int item_idx, vh;
    {
        // the plan lists tiles of 16 tokens, heaviest first: the even ones of a sequence stand for a pair, the odd ones for nothing
        const int n_items = hdr->n_prefill_items, n_vh = p.n_kv_heads * sub;
        const int lin = SPLIT ? (int)(blockIdx.x / cluster_ctas()) : (int)blockIdx.x;
        item_idx = lin / n_vh;
        vh = lin - item_idx * n_vh;
        if (item_idx >= n_items) {
            pdl_wait();                           // the grid must not complete before the decode kernel it overlaps
            return;
        }
    }
    const int2 item = reinterpret_cast<const int2*>(p.ws + p.L.prefill_items)[item_idx];
    const int s = item.x, q_start = item.y;
    if (s < 0 || s >= p.n_seqs || (q_start & kPrefillTileTokens)) {      // (s: a plan of another batch)
        pdl_wait();
        return;
    }
    const int g = vh / sub, h0 = (vh - g * sub) * 8, heads = min(8, p.group - h0);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int q0 = p.cu_seqlens[s];
    const int T = p.cu_seqlens[s + 1] - q0;
    const int len = q8_len(p, s);
    const int ctx = len - T;
    const int32_t* table = p.block_tables + (int64_t)(p.table_rows ? p.table_rows[s] : s) * p.table_stride;
    const int kv_end = min(len, ctx + min(q_start + kTokens, T));
    const int n_q = T - q_start > kPrefillTileTokens ? 2 : 1;                // Q tiles
    int n_tiles = kv_end > 0 ? (kv_end + kKeys - 1) / kKeys : 0, tile0 = 0;   // this CTA's key tiles: tile0 .. tile0 + n_tiles - 1
    int parts = 1, part = 0;
    if (SPLIT) {
        part = (int)cluster_rank();
        if (n_tiles >= kSplitTiles) {
            parts = (int)cluster_ctas();
            tile0 = (int)((unsigned)(n_tiles * part) / (unsigned)parts);
            n_tiles = (int)((unsigned)(n_tiles * (part + 1)) / (unsigned)parts) - tile0;
        } else if (part > 0) {                    // a short item is the first CTA's alone
            pdl_wait();
            return;
        }
    }

    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    const uint32_t sQ0 = base, sK = sQ0 + 2 * Q_BYTES, sV = sK + kStagesK * KV_BYTES;
    const uint32_t bar0 = sV + kStagesV * KV_BYTES;
    auto bar = [&](int i) -> uint32_t { return bar0 + 8u * (uint32_t)i; };
    volatile uint32_t* tail_words = reinterpret_cast<volatile uint32_t*>(smem_raw + (bar0 - raw) + D::Bars * 8);
    volatile uint32_t& tmem_slot = tail_words[0];
    volatile uint32_t& abort_flag = tail_words[1];
    float* const scale_ring = reinterpret_cast<float*>(smem_raw + (bar0 - raw) + ((D::Bars * 8 + 8 + 15) & ~15));   // [ring][sk | lv | 1/sv][4]
    uint64_t* const nan_ring = reinterpret_cast<uint64_t*>(scale_ring + kScaleRing * 12);       // [ring][converting warp], bit = key of the tile
    uint32_t dyn_bytes;
    asm volatile("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dyn_bytes));
    if (bar0 - raw + kTailBytes > dyn_bytes) {    // the array did not start where the launcher's size assumes: never expected
        if (tid == 0) atomicAdd(&reinterpret_cast<PlanHeader*>(p.ws + p.L.header)->errors, 1);
        pdl_wait();
        return;
    }
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < D::Bars; ++i) {
            // K and V free: one commit per Q tile that read them
            const uint32_t count = i >= D::BarScale ? (kNanCodes ? kConvWarps : 2) : i >= D::BarKFree ? n_q : i >= D::BarVFull ? kConvWarps : i >= D::BarKFull ? 4
                                   : i >= D::BarPReady ? kRows / 32 : 1;
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar(i)), "r"(count) : "memory");
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        abort_flag = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bar0 + D::Bars * 8), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    bool ok = true;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
        if (warp < 10) {
            // The whole warp runs the loop with warp-uniform values and one elected lane issues: descriptors and addresses then stay
            // in uniform registers, where the instruction wants them.
            const int w = __shfl_sync(0xffffffffu, warp, 0) - 8;
            q_ready_barrier(w);
            if (w < n_q) {
                const uint32_t sQ = sQ0 + w * Q_BYTES, t_tile = __shfl_sync(0xffffffffu, tmem, 0) + w * COL_TILE;
                const int tiles = __shfl_sync(0xffffffffu, n_tiles, 0);
                const bool leader = elect_one();
                constexpr uint32_t idesc_s = instr_desc(false, kKeys), idesc_pv = instr_desc(true, HD);
                const uint64_t dQ = smem_desc(sQ, 16, 1024), dK = smem_desc(sK, 16, 1024);
                const uint64_t dV = smem_desc(sV, kKeys * 128, 1024);
                auto wait = [&](int i, uint32_t parity) -> bool {
                    return __all_sync(0xffffffffu, mbar_wait_or_abort(bar(i), parity, tail_words + 1));
                };
                auto issue_s = [&](int kt, bool there) {
                    const int sk = kt % kStagesK;
                    if (!there && !wait(D::BarKFull + sk, (uint32_t)((kt / kStagesK) & 1))) { ok = false; return; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t k0 = dK + (uint64_t)((sk * KV_BYTES) >> 4);
                    const uint32_t d = t_tile + (uint32_t)((kt & 1) * kKeys);
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk) {
                            const uint32_t a_off = (uint32_t)(((kk >> 2) * (kRows * 128) + (kk & 3) * 32) >> 4);
                            const uint32_t b_off = (uint32_t)(((kk >> 2) * (kKeys * 128) + (kk & 3) * 32) >> 4);
                            tc::mma_f16(d, dQ + a_off, k0 + b_off, idesc_s, kk > 0);
                        }
                        mma_commit(bar(D::BarS + 2 * w + (kt & 1)));
                        mma_commit(bar(D::BarKFree + sk));
                    }
                    __syncwarp();
                };
                auto issue_pv = [&](int kt, bool there) {
                    const int sv = kt % kStagesV;
                    if (!there && !wait(D::BarVFull + sv, (uint32_t)((kt / kStagesV) & 1))) { ok = false; return; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t t_p = t_tile + (uint32_t)((kt & 1) * kKeys);      // P(kt) lies where S(kt) was
                    const uint64_t v0 = dV + (uint64_t)((sv * KV_BYTES) >> 4);
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < kKeys / 16; ++kk)
                            tc::mma_f16_ts(t_tile + COL_O, t_p + (uint32_t)(kk * 8), v0 + (uint32_t)((kk * 2048) >> 4), idesc_pv,
                                           (kt > 0 || kk > 0) ? 1u : 0u);
                        mma_commit(bar(D::BarPV + 2 * w + (kt & 1)));
                        mma_commit(bar(D::BarVFree + sv));
                    }
                    __syncwarp();
                };
                if (tiles > 0) issue_s(0, false);
                if (tiles > 1) issue_s(1, false);
                for (int kt = 0; kt < tiles && ok; ++kt) {
                    // V and K are usually there long before P: one wait in turn instead of three
                    const bool v_there = __all_sync(0xffffffffu, mbar_test(bar(D::BarVFull + kt % kStagesV), (uint32_t)((kt / kStagesV) & 1)));
                    const bool k_there = __all_sync(0xffffffffu, mbar_test(bar(D::BarKFull + (kt + 2) % kStagesK), (uint32_t)(((kt + 2) / kStagesK) & 1)));
                    if (!wait(D::BarPReady + 2 * w + (kt & 1), (uint32_t)((kt >> 1) & 1))) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    issue_pv(kt, v_there);
                    if (kt + 2 < tiles) issue_s(kt + 2, k_there);
                }
                if (!ok) abort_flag = 1;
            }
        } else {
            // ---- converting warps. A piece is 16 codes of a row (one lane), an item 32 consecutive pieces: ROWS rows of one block. The
            // first four warps take a block of the tile each: its K items and its last V item; the other two the remaining V
            // items of two blocks each. A warp's addresses are then a base per block and constant steps: what bounds these warps is
            // the number of their instructions (they share the issue slots with the softmax).
            constexpr int CPR = HD / 16, ROWS = 32 / CPR, PER = 16 / ROWS;       // pieces per row, rows per item, items per block
            const int cw = warp - 10;
            // Eight lanes of a store (one pass over the 32 banks) hold four pieces of two neighbouring rows: their even 16-byte chunks
            // are swizzled to all eight places. (Eight pieces of one row would meet in four: 16 codes make two chunks, and the two
            // halves of a 128-dim head lie at the same banks.)
            const int row_in = CPR == 4 ? lane >> 2 : ((lane >> 2) & 1) | ((lane >> 4) << 1);
            const int piece = CPR == 4 ? lane & 3 : (lane & 3) | ((lane >> 1) & 4);
            auto row_lanes = [](int r) -> uint32_t { return CPR == 4 ? 0xfu << (4 * r) : 0xf0fu << (4 * (r & 1) + 16 * (r >> 1)); };
            const bool k_warp = cw < 4;
            const int b0 = k_warp ? cw : 2 * (cw - 4);                           // this warp's (first) block
            constexpr int VK = HD == 64 ? 1 : 2, VV = PER - VK, NV = 2 * VV;      // V items of a K warp; of a block left to a V warp; of a V warp
            const uint8_t* kb = p.k_pool + g * p.head_stride + piece * 16 + row_in * p.pos_stride;
            const uint8_t* vb = p.v_pool + g * p.head_stride + piece * 16 + row_in * p.pos_stride;
            const int64_t step = ROWS * p.pos_stride;
            const uint32_t piece_off = (uint32_t)((piece >> 2) * (kKeys * 128) + row_in * 128), chunk0 = (uint32_t)((piece & 3) * 2);
            uint4 kr[PER], vr[NV];
            // the table entry of keys 16 b .. of a tile, -1 past the last visible key; it is requested a whole tile before it is looked at
            auto fetch_raw = [&](int kt, int b) -> int {
                const int key = (tile0 + kt) * kKeys + 16 * b;
                return kt < n_tiles && key < kv_end ? table[key >> p.block_shift] : -1;
            };
            auto locate = [&](int kt, int b, int& raw) -> int64_t {              // offset of the block's first key in a pool; raw -1: absent
                int64_t off = (int64_t)raw * p.blk_stride;
                if (p.block_size != 16) off += (int64_t)(((tile0 + kt) * kKeys + 16 * b) & (p.block_size - 1)) * p.pos_stride;
                if ((unsigned)raw >= (unsigned)p.num_blocks) raw = -1;
                return off;
            };
            // items n0 .. of a block into r: a block that is there and full takes plain loads (the usual case, and warp-uniform)
            auto load_items = [&](const uint8_t* pool, int64_t off, int id, int kt, int b, int n0, auto count, uint4* r) {
                const uint8_t* src = pool + off;
                const int left = len - ((tile0 + kt) * kKeys + 16 * b);                    // keys of the block
                if (id >= 0 && left >= 16) {
#pragma unroll
                    for (int n = 0; n < decltype(count)::value; ++n) r[n] = __ldcg(reinterpret_cast<const uint4*>(src + (n0 + n) * step));
                } else {
#pragma unroll
                    for (int n = 0; n < decltype(count)::value; ++n)
                        r[n] = id >= 0 && (n0 + n) * ROWS + row_in < left ? __ldcg(reinterpret_cast<const uint4*>(src + (n0 + n) * step))
                                                                         : make_uint4(0u, 0u, 0u, 0u);
                }
            };
            auto store_item = [&](uint32_t tile, int b, int n, const uint4& w) { // 16 codes -> two 16-byte pieces of f16
                const uint32_t dst = tile + piece_off + b * (16 * 128) + n * (ROWS * 128), r7 = (uint32_t)((n * ROWS + row_in) & 7);
                uint32_t x, y, z, u;
                q8::expand<KV>(w.x, x, y);
                q8::expand<KV>(w.y, z, u);
                st_shared16(dst + ((chunk0 ^ r7) << 4), x, y, z, u);
                q8::expand<KV>(w.z, x, y);
                q8::expand<KV>(w.w, z, u);
                st_shared16(dst + (((chunk0 + 1) ^ r7) << 4), x, y, z, u);
            };
            // V item m of this warp: block and item inside it
            auto v_block = [&](int m) -> int { return k_warp ? b0 : b0 + m / VV; };
            auto v_item = [&](int m) -> int { return k_warp ? VV + m : m % VV; };
            const int n_v = k_warp ? VK : NV;
            int id0 = fetch_raw(0, b0), id1 = k_warp ? -1 : fetch_raw(0, b0 + 1);
            int raw0 = fetch_raw(1, b0), raw1 = k_warp ? -1 : fetch_raw(1, b0 + 1);
            float sk = 0.f, sv = 1.f;
            using std::integral_constant;
            auto load_tile_k = [&](int kt, int64_t off0) { load_items(kb, off0, id0, kt, b0, 0, integral_constant<int, PER>(), kr); };
            auto load_tile_v = [&](int kt, int64_t off0, int64_t off1) {
                if (k_warp) {
                    load_items(vb, off0, id0, kt, b0, VV, integral_constant<int, VK>(), vr);
                } else {
                    load_items(vb, off0, id0, kt, b0, 0, integral_constant<int, VV>(), vr);
                    load_items(vb, off1, id1, kt, b0 + 1, 0, integral_constant<int, VV>(), vr + VV);
                }
            };
            // scales: lanes 0 and 1 of the two V warps, a block each (the K warps are the slower ones)
            const bool scale_lane = !k_warp && lane < 2;
            int its_id = -1;
            auto load_scales = [&]() {
                its_id = lane == 0 ? id0 : id1;
                if (scale_lane && its_id >= 0) {
                    const int64_t o = (int64_t)its_id * p.sc_blk_stride + (int64_t)g * p.sc_head_stride;
                    sk = p.k_scale[o];
                    sv = p.v_scale[o];
                }
            };
            {
                const int64_t off0 = locate(0, b0, id0), off1 = locate(0, b0 + 1, id1);
                if (n_tiles > 0) {
                    if (k_warp) load_tile_k(0, off0);
                    load_tile_v(0, off0, off1);
                    load_scales();
                }
            }
            bool k_free = true;                                                  // asked for a tile ahead
            for (int kt = 0; kt < n_tiles; ++kt) {
                const int st_k = kt % kStagesK, st_v = kt % kStagesV;
                const bool v_free = kt < kStagesV || mbar_test(bar(D::BarVFree + st_v), (uint32_t)((kt / kStagesV - 1) & 1));
                int64_t off0 = 0, off1 = 0;
                if (k_warp) {
                    if (!k_free)
                        ok = mbar_wait_or_abort(bar(D::BarKFree + st_k), (uint32_t)((kt / kStagesK - 1) & 1), tail_words + 1);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
#pragma unroll
                    for (int n = 0; n < PER; ++n) store_item(sK + st_k * KV_BYTES, b0, n, kr[n]);
                    warp_arrive(bar(D::BarKFull + st_k));
                }
                id0 = raw0;
                id1 = raw1;
                off0 = locate(kt + 1, b0, id0);
                off1 = locate(kt + 1, b0 + 1, id1);
                raw0 = fetch_raw(kt + 2, b0);
                raw1 = k_warp ? -1 : fetch_raw(kt + 2, b0 + 1);
                if (k_warp) load_tile_k(kt + 1, off0);
                if (!v_free)
                    ok = mbar_wait_or_abort(bar(D::BarVFree + st_v), (uint32_t)((kt / kStagesV - 1) & 1), tail_words + 1);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                if (kNanCodes) {
                    auto carry = [](uint32_t w) -> uint32_t { return (w & 0x7f7f7f7fu) + 0x01010101u; };     // bit 7 of a NaN byte is set
                    auto nan_of = [&](uint32_t w) -> uint32_t { return carry(w) & 0x80808080u; };
                    uint32_t any = 0;
#pragma unroll
                    for (int m = 0; m < NV; ++m)
                        if (m < n_v) any |= (carry(vr[m].x) | carry(vr[m].y)) | (carry(vr[m].z) | carry(vr[m].w));
                    uint64_t keys = 0;
                    if (__any_sync(0xffffffffu, (any & 0x80808080u) != 0)) {
#pragma unroll
                        for (int m = 0; m < NV; ++m) {
                            if (m >= n_v) continue;
                            const uint32_t fx = nan_of(vr[m].x), fy = nan_of(vr[m].y), fz = nan_of(vr[m].z), fw = nan_of(vr[m].w);
                            const uint32_t lanes = __ballot_sync(0xffffffffu, (fx | fy | fz | fw) != 0);
                            vr[m].x &= ~((fx >> 7) * 0xffu);
                            vr[m].y &= ~((fy >> 7) * 0xffu);
                            vr[m].z &= ~((fz >> 7) * 0xffu);
                            vr[m].w &= ~((fw >> 7) * 0xffu);
                            for (int r = 0; r < ROWS; ++r)
                                if (lanes & row_lanes(r)) keys |= 1ull << (16 * v_block(m) + v_item(m) * ROWS + r);
                        }
                    }
                    if (lane == 0) nan_ring[(kt % kScaleRing) * kConvWarps + cw] = keys;
                }
                if (!k_warp) {
                    // log2 and reciprocal by the approximate instructions (2^-22, far below P's 11 bits)
                    const float svf = sv < kMinScale ? kMinScale : sv;
                    if (scale_lane) {
                        float* e = scale_ring + (kt % kScaleRing) * 12 + b0 + lane;
                        e[0] = its_id >= 0 ? sk : 0.f;
                        e[4] = its_id >= 0 ? __log2f(svf) : -INFINITY;
                        e[8] = its_id >= 0 ? __fdividef(1.f, svf) : 0.f;
                    }
                    load_scales();
                    __syncwarp();
                }
                if (lane == 0 && (!k_warp || kNanCodes)) mbar_arrive(bar(D::BarScale + kt % kScaleRing));
#pragma unroll
                for (int m = 0; m < NV; ++m)
                    if (m < n_v) store_item(sV + st_v * KV_BYTES, v_block(m), v_item(m), vr[m]);
                warp_arrive(bar(D::BarVFull + st_v));
                if (k_warp) k_free = kt + 1 < kStagesK || mbar_test(bar(D::BarKFree + (kt + 1) % kStagesK), (uint32_t)(((kt + 1) / kStagesK - 1) & 1));
                load_tile_v(kt + 1, off0, off1);
            }
            if (!ok) abort_flag = 1;
        }
        if (SPLIT && parts > 1) {                  // the two meetings of the softmax threads below
            cluster_sync();
            cluster_sync();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        const int w = warp >> 2, row = tid & (kRows - 1);                  // Q tile, its row
        const uint32_t sQ = sQ0 + w * Q_BYTES;
        const uint32_t t_lane = tmem + w * COL_TILE + ((uint32_t)(32 * (warp & 3)) << 16);     // this warp's 32 lanes; lane = row
        const int tok = q_start + w * kPrefillTileTokens + (row >> 3), hh = row & 7;
        const bool row_ok = tok < T && hh < heads && q0 + tok >= 0 && q0 + tok < p.n_tokens;
        // Q row: scaled by a power of two so that its largest element lies in [1, 2), as f16
        float f_row;
        {
            const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(p.q) + (int64_t)(row_ok ? q0 + tok : 0) * p.q_stride +
                                       (int64_t)(row_ok ? g * p.group + h0 + hh : 0) * HD;
            float top = 0.f;
            if (row_ok)
                for (int c = 0; c < HD / 8; ++c) {
                    const Vec16<__nv_bfloat16> v = load16(src + 8 * c);
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v.get(i)));
                }
            int e = (int)((uint32_t)__float_as_int(top) >> 23) - 127;
            e = top == 0.f || e > 127 ? 0 : min(max(e, -126), 126);
            const float mult = __int_as_float((127 - e) << 23);
            f_row = p.scale_log2 * __int_as_float((127 + e) << 23);
            for (int c = 0; c < HD / 8; ++c) {
                uint32_t u[4] = {0u, 0u, 0u, 0u};
                if (row_ok) {
                    const Vec16<__nv_bfloat16> v = load16(src + 8 * c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) u[i] = pack_f16x2(v.get(2 * i) * mult, v.get(2 * i + 1) * mult);
                }
                st_shared16(sQ + (c >> 3) * (kRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4), u[0], u[1], u[2], u[3]);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        q_ready_barrier(w);
        const int limit = ctx + tok;      // last key this row may see
        const uint32_t t_o = t_lane + COL_O;
        const volatile uint32_t* abort_now = tail_words + 1;
        float m_run = -INFINITY, l_run = 0.f;
        const int my_tiles = w < n_q ? n_tiles : 0;
        bool ready = false;                // S and the scales of the next tile: asked for while this tile's exponentials are computed
        for (int kt = 0; kt < my_tiles; ++kt) {
            // The scales of tile kt were written before its S was issued: their barrier is only looked at. (A warp gives up as a whole:
            // its tensor-memory accesses and votes are warp-wide.)
            if (!__all_sync(0xffffffffu, ready)) {
                ok = mbar_wait_or_abort(bar(D::BarS + 2 * w + (kt & 1)), (uint32_t)((kt >> 1) & 1), abort_now) &&
                     mbar_wait_or_abort(bar(D::BarScale + kt % kScaleRing), (uint32_t)((kt / kScaleRing) & 1), abort_now);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t s_src = t_lane + (uint32_t)((kt & 1) * kKeys);
            const int key_base = (tile0 + kt) * kKeys;
            const bool masked = key_base + kKeys - 1 > ctx + q_start + w * kPrefillTileTokens;      // else every row sees every key of the tile
            uint32_t sr[2][32];
            tmem_ld32_issue(s_src, sr[0]);
            tmem_ld32_issue(s_src + 32, sr[1]);
            const float* ring = scale_ring + (kt % kScaleRing) * 12;
            const float4 sk4 = *reinterpret_cast<const float4*>(ring), lv4 = *reinterpret_cast<const float4*>(ring + 4),
                         iv4 = *reinterpret_cast<const float4*>(ring + 8);
            uint64_t keys = 0;                                             // NaN keys of the tile
            if (kNanCodes) {
                const ulonglong2* nr = reinterpret_cast<const ulonglong2*>(nan_ring + (kt % kScaleRing) * kConvWarps);
                const ulonglong2 n0 = nr[0], n1 = nr[1], n2 = nr[2];
                keys = n0.x | n0.y | n1.x | n1.y | n2.x | n2.y;
            }
            const float fac[4] = {f_row * sk4.x, f_row * sk4.y, f_row * sk4.z, f_row * sk4.w};
            const float lv[4] = {lv4.x, lv4.y, lv4.z, lv4.w}, isv[4] = {iv4.x, iv4.y, iv4.z, iv4.w};
            tmem_ld_wait();
            // x = s * factor + log2(sv), two at a time
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const int b = 2 * hf + (i >> 4);
                    float x0, x1;
                    unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(sr[hf][i]), __uint_as_float(sr[hf][i + 1])), pack_f32x2(fac[b], fac[b]),
                                           pack_f32x2(lv[b], lv[b])), x0, x1);
                    sr[hf][i] = __float_as_uint(x0);
                    sr[hf][i + 1] = __float_as_uint(x1);
                }
            if (kNanCodes) {
                if (keys != 0) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if ((keys >> (32 * hf + i)) & 1ull) sr[hf][i] = 0x7fffffffu;
                }
            }
            if (masked) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (key_base + 32 * hf + i > limit) sr[hf][i] = 0xff800000u;
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int i = 0; i < 32; i += 2)
                    mx4[(i >> 1) & 3] = max3(mx4[(i >> 1) & 3], __uint_as_float(sr[hf][i]), __uint_as_float(sr[hf][i + 1]));
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            const bool move = __any_sync(0xffffffffu, mx > m_run + kLazy);
            if (move && kt > 0) {                                          // the output is rewritten: PV(kt - 1) has to be over
                ok = __all_sync(0xffffffffu, mbar_wait_or_abort(bar(D::BarPV + 2 * w + ((kt - 1) & 1)), (uint32_t)(((kt - 1) >> 1) & 1), abort_now));
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            }
            if (move) {
                const float m_new = fmaxf(m_run, mx);
                const float alpha = m_new == -INFINITY ? 1.f : ex2(m_run - m_new);
                m_run = m_new;
                l_run *= alpha;
                if (kt > 0) {
#pragma unroll
                    for (int c = 0; c < HD / 32; ++c) {
                        uint32_t r[32];
                        tmem_ld32_issue(t_o + 32 * c, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                        tmem_st32(t_o + 32 * c, r);
                    }
                    tmem_st_wait();
                }
            }
            const float m_ref = m_run == -INFINITY ? 0.f : m_run;
            const uint64_t neg_m2 = pack_f32x2(-m_ref, -m_ref);
            uint32_t pp[32];                                               // the row's P, two f16 each
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                float v[32];
#pragma unroll
                for (int q = 0; q < 2; ++q) {                              // a block of 16 keys: one V scale
                    uint64_t ps2[2] = {0ull, 0ull};
#pragma unroll
                    for (int i = 16 * q; i < 16 * q + 16; i += 2) {
                        float x0, x1;
                        unpack_f32x2(add_f32x2(pack_f32x2(__uint_as_float(sr[hf][i]), __uint_as_float(sr[hf][i + 1])), neg_m2), x0, x1);
                        v[i] = ex2(x0);
                        v[i + 1] = ex2(x1);
                        ps2[(i >> 1) & 1] = add_f32x2(ps2[(i >> 1) & 1], pack_f32x2(v[i], v[i + 1]));
                    }
                    float a0, a1, b0, b1;
                    unpack_f32x2(ps2[0], a0, a1);
                    unpack_f32x2(ps2[1], b0, b1);
                    const float sum = (a0 + a1) + (b0 + b1);
                    l_run = sum == 0.f ? l_run : fmaf(sum, isv[2 * hf + q], l_run);      // (a block the row does not see may have any scale)
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) pp[16 * hf + i] = pack_f16x2(v[2 * i], v[2 * i + 1]);
            }
            ready = mbar_test(bar(D::BarS + 2 * w + ((kt + 1) & 1)), (uint32_t)(((kt + 1) >> 1) & 1)) &
                    mbar_test(bar(D::BarScale + (kt + 1) % kScaleRing), (uint32_t)(((kt + 1) / kScaleRing) & 1));
            tmem_st32(s_src, pp);                                          // over S(kt), which this warp has read
            tmem_st_wait();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (!ok) break;
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(D::BarPReady + 2 * w + (kt & 1)));
        }
        if (!ok) abort_flag = 1;
        // ---- the row's output: after the last PV, 32 columns at a time
        const bool have_o = my_tiles > 0 && ok;                             // (a wait of another role that ran out makes this one run out too)
        if (have_o) {
            ok = __all_sync(0xffffffffu, mbar_wait_or_abort(bar(D::BarPV + 2 * w + ((n_tiles - 1) & 1)), (uint32_t)(((n_tiles - 1) >> 1) & 1), abort_now));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        __nv_bfloat16* out_row = reinterpret_cast<__nv_bfloat16*>(p.out) + (int64_t)(row_ok ? q0 + tok : 0) * p.out_stride +
                                 (int64_t)(row_ok ? g * p.group + h0 + hh : 0) * HD;
        bool store = row_ok;
        float inv = l_run == 0.f ? 0.f : 1.f / l_run;
        // A split item: every CTA finishes 256 / parts of the rows. The others send it {O, m, l} of these into its K and V
        // buffers, which nothing reads any more once both sides' last PV is over; then it joins them, its own first, the others in
        // the order of their ranks.
        constexpr int RS = HD + 4;
        const int rows_of = 2 * kRows / (SPLIT ? parts : 1), R = w * kRows + row, owner = R / rows_of;
        float own_w = 1.f, w_of[3] = {0.f, 0.f, 0.f};                       // weights of the parts
        const float* const got = reinterpret_cast<const float*>(smem_raw + (sK - raw)) + (R - owner * rows_of) * RS;   // of source i: + i rows_of RS
        if (SPLIT && parts > 1) {
            static_assert(2 * kRows * 3 / 4 * RS * 4 <= (kStagesK + kStagesV) * KV_BYTES, "what the others send fits the K and V buffers");
            cluster_sync();
            if (__any_sync(0xffffffffu, owner != part)) {                   // (rows_of is a multiple of 32: the same for a whole warp)
                const uint32_t dst = cluster_address(sK + (uint32_t)((((part < owner ? part : part - 1) * rows_of + R - owner * rows_of) * RS) * 4), owner);
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) {
                    if (!have_o || !ok) break;
                    uint32_t r[32];
                    tmem_ld32_issue(t_o + 32 * c, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 8; ++e) st_cluster16(dst + (32 * c + 4 * e) * 4, r[4 * e], r[4 * e + 1], r[4 * e + 2], r[4 * e + 3]);
                }
                // (a CTA that gave up makes these rows NaN; a part without a visible key has O = 0 that was perhaps never written: its weight is 0)
                st_cluster16(dst + HD * 4, __float_as_uint(m_run), ok ? __float_as_uint(l_run) : 0x7fffffffu, 0u, 0u);
            }
            cluster_sync();
            store = row_ok && owner == part;
            if (store) {
                float top = m_run;
                for (int i = 0; i < parts - 1; ++i) top = fmaxf(top, got[i * rows_of * RS + HD]);
                const float ref = top == -INFINITY ? 0.f : top;
                // weight of a part; 0 only for one without a visible key, so that NaN comes through
                auto weight = [&](float m, float l) { return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(m - ref); };
                own_w = weight(m_run, l_run);
                float l = l_run * own_w;
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    if (i >= parts - 1) continue;
                    const float m_i = got[i * rows_of * RS + HD], l_i = got[i * rows_of * RS + HD + 1];
                    w_of[i] = weight(m_i, l_i);
                    if (m_i == -INFINITY && l_i == 0.f) w_of[i] = -1.f;     // nothing to read
                    else l = fmaf(l_i, w_of[i], l);
                }
                inv = l == 0.f ? 0.f : 1.f / l;
            }
        }
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
            float v[32];
            if (ok && have_o) {                                            // (warp-uniform)
                uint32_t r[32];
                tmem_ld32_issue(t_o + 32 * c, r);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = 0.f;
            }
            if (SPLIT && parts > 1 && store) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] *= own_w;
#pragma unroll
                for (int j = 0; j < 3; ++j) {
                    if (j >= parts - 1 || w_of[j] < 0.f) continue;
                    const float4* o = reinterpret_cast<const float4*>(got + j * rows_of * RS + 32 * c);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float4 x = o[e];
                        v[4 * e] = fmaf(x.x, w_of[j], v[4 * e]);
                        v[4 * e + 1] = fmaf(x.y, w_of[j], v[4 * e + 1]);
                        v[4 * e + 2] = fmaf(x.z, w_of[j], v[4 * e + 2]);
                        v[4 * e + 3] = fmaf(x.w, w_of[j], v[4 * e + 3]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= inv;
            if (ok && store) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint4 o;
                    o.x = pack_bf16x2(v[8 * e + 0], v[8 * e + 1]);
                    o.y = pack_bf16x2(v[8 * e + 2], v[8 * e + 3]);
                    o.z = pack_bf16x2(v[8 * e + 4], v[8 * e + 5]);
                    o.w = pack_bf16x2(v[8 * e + 6], v[8 * e + 7]);
                    *reinterpret_cast<uint4*>(out_row + 32 * c + 8 * e) = o;
                }
            }
        }
        if (!ok) abort_flag = 1;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (abort_flag && tid == 0)        // a wait expired: count it where the host can read it (ns_collect_status)
        atomicAdd(&reinterpret_cast<PlanHeader*>(p.ws + p.L.header)->errors, 1);
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    pdl_wait();                        // complete only after the decode kernel this one ran beside
}

bool q8_prefill_supported(const Q8Params& p, int dtype) {
    return dtype == NS_BF16 && ((uintptr_t)p.out & 15) == 0 && p.out_stride % 8 == 0;      // beside what the decode kernel asks for
}

// NS_ERR_UNSUPPORTED: the kernel was not built with the register count its split needs; the scalar kernel serves then.
template <int HD, typename KV, bool SPLIT> static int launch_prefill_q8_as(const Q8Params& p, int max_items, int parts, cudaStream_t st) {
    constexpr int atoms = HD / 64;
    using D = q8p::Depth<HD>;
    // tiles + tail; 1 KB of slack for the 1024-byte alignment
    constexpr int smem = 2 * q8p::kRows * 128 * atoms + (D::K + D::V) * q8p::kKeys * 128 * atoms + q8p::kTailBytes + 1024;
    static_assert(smem <= 227 * 1024, "one CTA's shared memory");
    const auto kernel = prefill_q8_kernel<HD, KV, SPLIT>;
    static SmemOptIn optin;
    if (optin.needs((size_t)smem)) {
        // setmaxnreg moves registers between the warpgroups within what the block was launched with: it must be all of 128 a thread
        cudaFuncAttributes attr;
        cudaError_t e = cudaFuncGetAttributes(&attr, kernel);
        if (e != cudaSuccess) return fail(NS_ERR_CUDA, "prefill_q8: cannot query the kernel: %s", cudaGetErrorString(e));
        if (attr.numRegs * q8p::kThreads < 2 * (q8p::kRegsSoftmax + q8p::kRegsOther) * 128) return NS_ERR_UNSUPPORTED;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return fail(NS_ERR_CUDA, "prefill_q8: cannot reserve %d bytes of shared memory: %s", smem, cudaGetErrorString(e));
        optin.done((size_t)smem);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(max_items * p.n_kv_heads * ((p.group + 7) / 8) * parts));
    cfg.blockDim = dim3(q8p::kThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = SPLIT ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess) return fail(NS_ERR_CUDA, "prefill_q8: launch failed: %s", cudaGetErrorString(e));
    return NS_OK;
}
// An item is split over its keys where the items leave most SMs without one: by four while four parts of each fit one wave, else by
// two. (512 tokens on 4,096 keys, 14 heads of 64, 32 items: 83 us whole, 50 in two parts, 33 in four; 28 heads of 128, 64
// items: 105 / 64 / 86. 1,024 tokens on 1,024 keys, 128 items of the latter: 55 / 66 / 111 - a second wave costs more than it
// saves, a CTA takes 6 us to start and to finish. Items below kSplitTiles stay whole; the clusters cost those 0.8 us.)
template <int HD, typename KV> static int launch_prefill_q8_hd(const Q8Params& p, int max_items, cudaStream_t st) {
    const int64_t items = p.n_tokens / q8p::kTokens * p.n_kv_heads * ((p.group + 7) / 8);
    const int parts = 4 * items <= p.sm_count ? 4 : 2 * items <= p.sm_count ? 2 : 1;
    return parts > 1 ? launch_prefill_q8_as<HD, KV, true>(p, max_items, parts, st) : launch_prefill_q8_as<HD, KV, false>(p, max_items, 1, st);
}

int launch_q8_prefill(const Q8Params& p, int pool_dtype, int max_items, cudaStream_t st) {
    if (p.head_dim == 64)
        return pool_dtype == NS_INT8 ? launch_prefill_q8_hd<64, KvInt8>(p, max_items, st) : launch_prefill_q8_hd<64, KvE4m3>(p, max_items, st);
    return pool_dtype == NS_INT8 ? launch_prefill_q8_hd<128, KvInt8>(p, max_items, st) : launch_prefill_q8_hd<128, KvE4m3>(p, max_items, st);
}

}  // namespace ns
