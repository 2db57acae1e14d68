// Attention over the 4-bit KV cache for prompts, on tcgen05 (kind::f16, FP32 accumulators in tensor memory), keeping FP32's accuracy.
//
// A block has 128 columns of a KV head (a column is a query head at a position) and walks the rows, 64 at a time:
//     S [128 columns x 64 rows] = Q K'^T,   P = 2^(S f - m + 14),   O [128 columns x values] += P V'
// K' = ks (n - 8) and V' = vs (n - 8) are held values, an 11-bit scale times a 4-bit code: 15 bits, which two fp16 pieces hold exactly. Q and P are
// two pieces of 11 bits. Each product is three instructions a step, high.high + low.high + high.low; low.low is 2^-23 of the result.
// (On mma.sync the scales stay FP32 factors outside the products, two instructions a step, but their rate is a third; 16
// columns share an unpacked row there, 128 here.)
//
// Warps: 8 softmax, two threads a column; 4 that turn key codes into the pieces of K', 4 for V' (transposed: the rows are the
// contraction); 1 issues the products, 1 the copies. All but P is double buffered, and S of the next rows is computed while the softmax is at these.
// The instruction cuts its sums off, towards zero, at every step: outputs after 16000 rows were 5.7e-5 off in one accumulator, 2.3e-6 after 2048. So after a run
// of PK_RUN times 64 rows its outputs are added, rounded, to sums: half of them in tensor memory, beside one place for P, half in shared memory (all of them there, in steps
// of 16: 160 us instead of 143).
// What bounds it: 2048 positions of 32 heads of 128 values over 8 take 139 us with the preparing launch, replayed, of which the products would be 62 at the measured rate. Per 64 rows
// the softmax's chain (load, maximum, exponentials, pieces, store: 1500 cycles without exponentials and dequantisers) and shared memory (values of K' and V' written and read,
// sums of runs) are longer than the products' 1600 cycles: leaving two of three products out gained 1 %, leaving both dequantisers out 15 %.
// A V' of a group with a NaN scale would reach columns that do not see the row (0 * NaN), so it is zeros, and the first row of a NaN in each of a row's groups is
// remembered: columns see rows from the first on, so those that see that one give NaN in the group's outputs. (A NaN in K' reaches its own row's scores alone.)
#include "kv4.cuh"
#include "tc_common.cuh"
#include <algorithm>

namespace {

constexpr int PK_ROWS = 64, PK_COLS = 128, PK_RAW = 3, PK_RUN = 3;
constexpr int PK_KEY_WARP = 8, PK_VALUE_WARP = 12, PK_MMA_WARP = 16, PK_TMA_WARP = 17, PK_THREADS = 18 * 32;
constexpr float PK_LOW = -3.0e38f, PK_SLACK = 1.9f;            // see kv4_attn.cu

struct PkParams {
    Kv4 c; Kv4Columns t; Kv4Place at;
    const unsigned char* image; const float* qc;
    float* out; float2* stat;
    int tiles;                                                 // of 128 columns, a KV head
    int* err;
};
template <int NG> struct PkSmem {
    static constexpr int KB = NG / 2, HD = 32 * NG;            // KB: blocks of 64 values, a swizzled row of 128 bytes each
    static constexpr int IMAGE = 2 * KB * 16384, KEYS = 2 * KB * 8192, VALUES = 2 * HD * 128, RAW_BYTES = PK_ROWS * 36 * NG;
    static constexpr int K = 0, V = K + 2 * KEYS, RAW = V + 2 * VALUES;
    static constexpr int SUM = RAW + PK_RAW * RAW_BYTES, TOTAL = SUM + HD * PK_COLS * 2;         // SUM [value / 4][column] float4, of the upper half of the values
};
struct PkShared {
    unsigned long long q_full, raw_full[PK_RAW], raw_empty[PK_RAW], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], s_empty[2], p_full[2], pv_done[2], drained;
    uint32_t tmem_base;
    int abort_flag;
    float meet[2][PK_COLS];                                    // maxima, at last sums, of a column's two threads
    int nan_from[4];                                           // first row whose value scale of this group is NaN
};

__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// whether any thread of the pair of warps says so
__device__ __forceinline__ bool pair_any(int id, bool x) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"(id), "r"((uint32_t)x) : "memory");
    return r;
}
__device__ __forceinline__ void pair_sync(int id) { asm volatile("barrier.cta.sync %0, 64;" :: "r"(id) : "memory"); }
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 half2_of(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }

// The eight codes of a word less their bias of 8, as pairs 0 and 4, 1 and 5, 2 and 6, 3 and 7: under the exponent of 1024 a code n is the fp16 1024 + n
__device__ __forceinline__ void codes_of(uint32_t w, __half2 (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t n;                                            // (w >> 4 i & mask) | base as one instruction
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(n) : "r"(w >> (4 * i)), "r"(0x000F000Fu), "r"(0x64006400u));
        f[i] = __hsub2(half2_of(n), half2_of(0x64086408u));
    }
}
// codes times scales as two pieces, exact together
__device__ __forceinline__ void held_pieces(const __half2 f, const __half2 scale, uint32_t& high, uint32_t& low) {
    const __half2 h = __hmul2(f, scale);
    high = bits(h);
    low = bits(__hfma2(f, scale, __hneg2(h)));
}
__device__ __forceinline__ bool is_nan(uint32_t half_bits) { return (half_bits & 0x7FFFu) > 0x7C00u; }

// Piece t of a key row (the values 8t..8t+7 of every group) into the operand image: rows of 128 bytes, 16-byte pieces swizzled, blocks of 64 values
// `block` bytes apart, the low pieces `part` bytes behind the high ones. scales: the row's keys'.
template <int NG>
__device__ __forceinline__ void place_key(unsigned char* to, int block, int part, int r, int t, const uint32_t (&w)[NG], const uint32_t (&scales)[NG / 2]) {
#pragma unroll
    for (int j = 0; j < NG; j++) {
        const uint32_t s = j & 1 ? scales[j / 2] >> 16 : scales[j / 2] & 0xFFFFu;
        const __half2 s2 = half2_of(s | s << 16);
        __half2 f[4];
        codes_of(w[j], f);
        uint4 high, low;
        held_pieces(f[0], s2, high.x, low.x); held_pieces(f[1], s2, high.y, low.y); held_pieces(f[2], s2, high.z, low.z); held_pieces(f[3], s2, high.w, low.w);
        const int piece = t * NG + j;
        unsigned char* at = to + (piece >> 3) * block + r * 128 + (((piece & 7) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(at) = high;
        *reinterpret_cast<uint4*>(at + part) = low;
    }
}
template <int N> __device__ __forceinline__ void load_words(uint32_t (&d)[N], const unsigned char* s) {
    if constexpr (N == 4) { const uint4 v = *reinterpret_cast<const uint4*>(s); d[0] = v.x; d[1] = v.y; d[2] = v.z; d[3] = v.w; }
    else if constexpr (N == 1) d[0] = *reinterpret_cast<const uint32_t*>(s);
    else { const uint2 v = *reinterpret_cast<const uint2*>(s); d[0] = v.x; d[1] = v.y; }
}

template <int NG>
__global__ void __launch_bounds__(PK_THREADS, 1) kv4_prompt_kernel(const PkParams p) {
    using S = PkSmem<NG>;
    extern __shared__ __align__(1024) unsigned char smem[];
    PkShared* sh = reinterpret_cast<PkShared*>(smem + S::TOTAL);
    volatile int* abort_flag = &sh->abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kvh = blockIdx.x % p.c.n_kv, tile = p.tiles - 1 - blockIdx.x / p.c.n_kv, unit = kvh * p.tiles + tile, c0 = tile * PK_COLS;          // most rows first
    if (tid == 0) {
        auto init = [&](unsigned long long& b, int n) { mbar_init(smem_u32(&b), n); };
        init(sh->q_full, 8); init(sh->drained, 1);
        for (int i = 0; i < PK_RAW; i++) { init(sh->raw_full[i], 1); init(sh->raw_empty[i], 8); }
        for (int i = 0; i < 2; i++) {
            init(sh->k_full[i], 4); init(sh->k_empty[i], 1); init(sh->v_full[i], 4); init(sh->v_empty[i], 1);
            init(sh->s_full[i], 1); init(sh->s_empty[i], 8); init(sh->p_full[i], 8); init(sh->pv_done[i], 1);
        }
        sh->abort_flag = 0;
        for (int j = 0; j < NG; j++) sh->nan_from[j] = 0x7FFFFFFF;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (warp == PK_MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&sh->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        pdl_launch_dependents();                               // not before this block holds its tensor memory: see linear_tc.cu
    }
    pdl_wait();
    int row0, pos0;
    const bool there = kv4_place(p.at, p.t.B, p.c.max_rows, p.err, row0, pos0);
    const int rows = there ? row0 + min(p.t.B - 1, (c0 + PK_COLS - 1) / p.t.group) + 1 : 0, n = (rows + PK_ROWS - 1) / PK_ROWS;
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_o = sh->tmem_base, tmem_s = tmem_o + S::HD, tmem_p = tmem_s + 2 * PK_ROWS, tmem_sum = tmem_p + PK_ROWS, tmem_q = tmem_sum + 64;          // 128 + 2 x 64 + 64 + 64 + 128 columns

    if (warp == PK_TMA_WARP) {
        if (elect_one() && n) {
            asm volatile("fence.proxy.async.global;" ::: "memory");
            const size_t plane = p.c.row(kvh, 0);
            int s = 0; uint32_t ph = 1;
            for (int i = 0; i < n; i++) {
                if (!mbar_wait(smem_u32(&sh->raw_empty[s]), ph, abort_flag, 1)) break;
                const int r = i * PK_ROWS, have = min(PK_ROWS, (rows - r + 7) & ~7);            // whole groups of 8 rows, which the planes have
                const uint32_t bar = smem_u32(&sh->raw_full[s]), to = smem_u32(smem + S::RAW + s * S::RAW_BYTES);
                mbar_expect_tx(bar, (uint32_t)have * 36 * NG);
                bulk_load(to, p.c.k + (plane + r) * (16 * NG), (uint32_t)have * 16 * NG, bar);
                bulk_load(to + PK_ROWS * 16 * NG, p.c.v + (plane + r) * (16 * NG), (uint32_t)have * 16 * NG, bar);
                bulk_load(to + PK_ROWS * 32 * NG, p.c.scale + (plane + r) * (2 * NG), (uint32_t)have * 4 * NG, bar);
                if (++s == PK_RAW) { s = 0; ph ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp == PK_MMA_WARP) {
        if (elect_one() && n) {
            constexpr uint32_t idesc = (1u << 4) | (8u << 24);                                    // FP32 accumulators, fp16 operands, 128 rows
            constexpr uint32_t idesc_s = idesc | ((PK_ROWS / 8) << 17), idesc_o = idesc | ((S::HD / 8) << 17);
            bool ok = mbar_wait(smem_u32(&sh->q_full), 0u, abort_flag, 2);
            auto scores = [&](int i) {
                const int b = i & 1;
                const uint32_t ph = (uint32_t)(i >> 1) & 1u;
                if (!mbar_wait(smem_u32(&sh->k_full[b]), ph, abort_flag, 3) || !mbar_wait(smem_u32(&sh->s_empty[b]), ph ^ 1u, abort_flag, 4)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t k = smem_desc_sw128(smem_u32(smem + S::K + b * S::KEYS));
#pragma unroll
                for (int m = 0; m < 3; m++)                                                       // low.high, high.low, high.high: small sums first, which lose least
#pragma unroll
                    for (int st = 0; st < S::HD / 16; st++)
                        mma_f16_ts(tmem_s + b * PK_ROWS, tmem_q + (m == 0) * (S::HD / 2) + st * 8, k + (((m == 1) * S::KB + st / 4) * 8192 >> 4) + st % 4 * 2, idesc_s, m || st ? 1u : 0u);
                mma_commit(smem_u32(&sh->k_empty[b]));
                mma_commit(smem_u32(&sh->s_full[b]));
                return true;
            };
            ok = ok && scores(0);
            for (int i = 0; i < n && ok; i++) {
                if (i + 1 < n) ok = scores(i + 1);
                const int b = i & 1;
                const uint32_t ph = (uint32_t)(i >> 1) & 1u;
                ok = ok && mbar_wait(smem_u32(&sh->v_full[b]), ph, abort_flag, 5) && mbar_wait(smem_u32(&sh->p_full[b]), ph, abort_flag, 6);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t v = smem_desc_sw128(smem_u32(smem + S::V + b * S::VALUES));
                const uint32_t more = i % PK_RUN ? 1u : 0u;
#pragma unroll
                for (int m = 0; m < 3; m++)
#pragma unroll
                    for (int st = 0; st < PK_ROWS / 16; st++)
                        mma_f16_ts(tmem_o, tmem_p + (m == 0) * (PK_ROWS / 2) + st * 8, v + ((m == 1) * S::HD * 128 >> 4) + st * 2, idesc_o, m || st ? 1u : more);
                mma_commit(smem_u32(&sh->v_empty[b]));
                mma_commit(smem_u32(&sh->pv_done[b]));
            }
            mma_commit(smem_u32(&sh->drained));
            mbar_wait(smem_u32(&sh->drained), 0u, abort_flag, 7);
        }
        __syncwarp();
    } else if (warp >= PK_KEY_WARP) {
        // 96 registers a thread at the launch: 256 x 72 + 256 x 120 + 64 x 96 are the 576 x 96 there
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const bool keys = warp < PK_VALUE_WARP;
        const int w = warp & 3;
        int s = 0; uint32_t ph = 0;
        for (int i = 0; i < n; i++) {
            const int b = i & 1;
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->raw_full[s]), ph, abort_flag, 8) &&
                                         mbar_wait(smem_u32(keys ? &sh->k_empty[b] : &sh->v_empty[b]), (uint32_t)((i >> 1) & 1) ^ 1u, abort_flag, 9))) break;
            const unsigned char* raw = smem + S::RAW + s * S::RAW_BYTES;
            const unsigned char* scales = raw + PK_ROWS * 32 * NG;
            if (keys) {
                // lanes: eight rows by the four pieces; the swizzle spreads the rows' pieces over the banks
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int r = 8 * (w + 4 * u) + (lane & 7), t = lane >> 3;
                    uint32_t k[NG], sc[NG / 2];
                    load_words<NG>(k, raw + r * 16 * NG + t * 4 * NG);
                    load_words<NG / 2>(sc, scales + r * 4 * NG);
                    place_key<NG>(smem + S::K + b * S::KEYS, 8192, S::KB * 8192, r, t, k, sc);
                }
            } else {
                // lanes: four pairs of rows by the eight pieces of a row; transposed, value 32 j + 4 g + i is line (4 j + i) 8 + g of 64 rows
#pragma unroll 1
                for (int u = 0; u < 2; u++) {
                    const int chunk = w + 4 * u, g = lane >> 2, a = 8 * chunk + 2 * (lane & 3);
                    uint32_t va[NG / 2], vb[NG / 2], sa[NG], sb[NG];
                    if constexpr (NG == 4) {
                        load_words<2>(va, raw + PK_ROWS * 16 * NG + a * 16 * NG + g * 2 * NG);
                        load_words<2>(vb, raw + PK_ROWS * 16 * NG + (a + 1) * 16 * NG + g * 2 * NG);
                    } else {
                        va[0] = *reinterpret_cast<const uint32_t*>(raw + PK_ROWS * 16 * NG + a * 16 * NG + g * 2 * NG);
                        vb[0] = *reinterpret_cast<const uint32_t*>(raw + PK_ROWS * 16 * NG + (a + 1) * 16 * NG + g * 2 * NG);
                    }
                    load_words<NG>(sa, scales + a * 4 * NG);
                    load_words<NG>(sb, scales + (a + 1) * 4 * NG);
                    uint32_t nan = 0;
#pragma unroll
                    for (int j = NG / 2; j < NG; j++) nan |= bits(__hisnan2(half2_of(sa[j]))) | bits(__hisnan2(half2_of(sb[j])));
                    if (nan || (i + 1) * PK_ROWS > rows) {     // no rows behind the last one, no NaN
                        auto keep = [&](uint32_t s, int r, int j) {                             // the scales of groups j and j + 1 of a row
                            if (r >= rows) return 0u;
                            if (is_nan(s)) { atomicMin(&sh->nan_from[j], r); s &= 0xFFFF0000u; }
                            if (is_nan(s >> 16)) { atomicMin(&sh->nan_from[j + 1], r); s &= 0xFFFFu; }
                            return s;
                        };
#pragma unroll
                        for (int j = NG / 2; j < NG; j++) {
                            sa[j] = keep(sa[j], i * PK_ROWS + a, 2 * j - NG);
                            sb[j] = keep(sb[j], i * PK_ROWS + a + 1, 2 * j - NG);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < NG; j++) {
                        const __half2 s2 = half2_of(__byte_perm(sa[(NG + j) / 2], sb[(NG + j) / 2], j & 1 ? 0x7632 : 0x5410));
                        __half2 f[4];
                        codes_of(__byte_perm(va[j / 2], vb[j / 2], j & 1 ? 0x7632 : 0x5410), f);
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            uint32_t high, low;
                            held_pieces(f[q], s2, high, low);
                            unsigned char* at = smem + S::V + b * S::VALUES + ((4 * j + q) * 8 + g) * 128 + ((chunk ^ g) << 4) + (lane & 3) * 4;
                            *reinterpret_cast<uint32_t*>(at) = high;
                            *reinterpret_cast<uint32_t*>(at + S::HD * 128) = low;
                        }
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");                        // the tensor cores read these stores
            __syncwarp();
            if (lane == 0) { mbar_arrive(smem_u32(keys ? &sh->k_full[b] : &sh->v_full[b])); mbar_arrive(smem_u32(&sh->raw_empty[s])); }
            if (++s == PK_RAW) { s = 0; ph ^= 1; }
        }
    } else {
        // A column has two threads, of warps w and w + 4: each has 32 of the rows, half of the queries' copy and of the outputs.
        asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
        const int quarter = warp & 3, half = warp >> 2, own = quarter * 32 + lane, c = c0 + own, b_col = c / p.t.group;
        const bool on = b_col < p.t.B;
        const int lim = row0 + b_col, lim0 = row0 + (c0 + quarter * 32) / p.t.group;             // last rows that this column, the warp's first column, see
        const float f = on ? __ldcg(p.qc + (size_t)unit * PK_COLS + own) : 0.0f;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        // the queries' pieces into tensor memory: the scores' A operand (from shared memory it would be read again for every 64 rows, and with what the
        // dequantisers write that is more than shared memory gives)
        if (n) {
            const unsigned char* image = p.image + (size_t)unit * S::IMAGE + own * 128 + half * S::KB * 16384;
#pragma unroll 1
            for (int kb = 0; kb < S::KB; kb++) {
                uint32_t x[32];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint4 v = __ldcg(reinterpret_cast<const uint4*>(image + kb * 16384 + ((e ^ (own & 7)) << 4)));
                    x[4 * e] = v.x; x[4 * e + 1] = v.y; x[4 * e + 2] = v.z; x[4 * e + 3] = v.w;
                }
                tmem_st32(tmem_q + lanes + half * (S::HD / 2) + kb * 32, x);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh->q_full));
        }
        float4* sums = reinterpret_cast<float4*>(smem + S::SUM) + own;
        float m = PK_LOW, l = 0.0f, aged = 1.0f;               // aged: what the sums of earlier runs are to be multiplied by
        bool wide = false, alive = true;                       // not alive: a wait gave up; the barriers of the pair are still both warps'
        for (int i = 0; i < n; i++) {
            const int from = i * PK_ROWS + half * 32;
            const int b = i & 1;
            const uint32_t ph = (uint32_t)(i >> 1) & 1u, ph_last = (uint32_t)((i - 1) >> 1) & 1u;
            const bool begins = i % PK_RUN == 0;
            alive = alive && __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->s_full[b]), ph, abort_flag, 10));
            uint32_t s[32];
            float top = PK_LOW, corr = 1.0f;
            if (alive) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                tmem_ld32(tmem_s + lanes + b * PK_ROWS + half * 32, s);
                tmem_wait_ld(s);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh->s_empty[b]));
                if (from + 31 > lim0) {
#pragma unroll
                    for (int u = 0; u < 32; u++) if (from + u > lim) s[u] = 0xFF800000u;
                }
                float t4[4] = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
#pragma unroll
                for (int u = 0; u < 32; u++) t4[u & 3] = fmaxf(t4[u & 3], __uint_as_float(s[u]));
                top = fmaxf(PK_LOW, fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * f);
            }
            if (pair_any(1 + quarter, top > m + PK_SLACK)) {
                sh->meet[half][own] = top;
                pair_sync(1 + quarter);
                const float now = fmaxf(m, fmaxf(top, sh->meet[half ^ 1][own]));
                corr = ex2(m - now);
                m = now;
                l *= corr;
                aged *= corr;
                wide = fabsf(now) > 524288.0f;
                alive = alive && (begins || __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->pv_done[b ^ 1]), ph_last, abort_flag, 12)));
                if (alive && !begins) {
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                    for (int d = half * (S::HD / 2); d < (half + 1) * (S::HD / 2); d += 32) {
                        const uint32_t at = tmem_o + lanes + d;
                        uint32_t o[32];
                        tmem_ld32(at, o);
                        tmem_wait_ld(o);
#pragma unroll
                        for (int u = 0; u < 32; u++) o[u] = __float_as_uint(__uint_as_float(o[u]) * corr);
                        tmem_st32(at, o);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
            }
            if (!alive) continue;
            const float off = 14.0f - m;
            if (__any_sync(0xffffffffu, wide)) {               // beyond 2^19 a fused product would show the maximum's own rounding
#pragma unroll
                for (int u = 0; u < 32; u++) s[u] = __float_as_uint(ex2((__fmul_rn(__uint_as_float(s[u]), f) - m) + 14.0f));
            } else {
#pragma unroll
                for (int u = 0; u < 32; u++) s[u] = __float_as_uint(ex2(fmaf(__uint_as_float(s[u]), f, off)));
            }
            float l4[4] = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
            for (int u = 0; u < 32; u++) l4[u & 3] += __uint_as_float(s[u]);
            l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
            uint32_t high[16], low[16];                        // 32 rows: 16 columns of tensor memory a piece
#pragma unroll
            for (int u = 0; u < 16; u++) {
                const float a = __uint_as_float(s[2 * u]), z = __uint_as_float(s[2 * u + 1]);
                const __half2 x = __floats2half2_rn(a, z);
                const float2 back = __half22float2(x);
                high[u] = bits(x);
                low[u] = bits(__floats2half2_rn(a - back.x, z - back.y));
            }
            alive = !i || __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->pv_done[b ^ 1]), ph_last, abort_flag, 11));       // P has been read, and outputs are whole
            if (!alive) continue;
            tmem_st16(tmem_p + lanes + 16 * half, high);
            tmem_st16(tmem_p + lanes + PK_ROWS / 2 + 16 * half, low);
            if (begins && i) {                                 // a run has ended
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                for (int d = 0; d < S::HD / 2; d += 32) {
                    uint32_t o[32];
                    tmem_ld32(tmem_o + lanes + half * (S::HD / 2) + d, o);
                    if (half == 0) {
                        uint32_t old[32];
                        tmem_ld32(tmem_sum + lanes + d, old);
                        tmem_wait_ld(o);
                        tmem_wait_ld(old);
#pragma unroll
                        for (int u = 0; u < 32; u++) old[u] = __float_as_uint(fmaf(__uint_as_float(o[u]), corr, i > PK_RUN ? __uint_as_float(old[u]) * aged : 0.0f));
                        tmem_st32(tmem_sum + lanes + d, old);
                    } else {
                        float4 old[8];
#pragma unroll
                        for (int u = 0; u < 8; u++) old[u] = i > PK_RUN ? sums[(d / 4 + u) * PK_COLS] : make_float4(0.f, 0.f, 0.f, 0.f);
                        tmem_wait_ld(o);
#pragma unroll
                        for (int u = 0; u < 8; u++)
                            sums[(d / 4 + u) * PK_COLS] = make_float4(fmaf(__uint_as_float(o[4 * u]), corr, old[u].x * aged), fmaf(__uint_as_float(o[4 * u + 1]), corr, old[u].y * aged),
                                                                      fmaf(__uint_as_float(o[4 * u + 2]), corr, old[u].z * aged), fmaf(__uint_as_float(o[4 * u + 3]), corr, old[u].w * aged));
                    }
                }
                aged = 1.0f;
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh->p_full[b]));
        }
        pair_sync(1 + quarter);                                // the last maxima are read
        sh->meet[half][own] = l;
        pair_sync(1 + quarter);
        l += sh->meet[half ^ 1][own];
        if (n && alive && __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->pv_done[(n - 1) & 1]), (uint32_t)((n - 1) >> 1) & 1u, abort_flag, 13)) &&
            __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->v_full[(n - 1) & 1]), (uint32_t)((n - 1) >> 1) & 1u, abort_flag, 14))) {          // what was said of the values' NaN
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const float inv = 1.0f / l;
            float* to = p.out + ((size_t)b_col * p.t.n_heads + (size_t)kvh * p.t.group + c % p.t.group) * S::HD;
            const bool vec = ((uintptr_t)p.out & 15) == 0;
#pragma unroll 1
            for (int j = half * (NG / 2); j < (half + 1) * (NG / 2); j++) {
                float o[32];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t x[16];
                    tmem_ld16(tmem_o + lanes + 32 * j + 16 * h, x);
                    const int d = 32 * (j - half * (NG / 2)) + 16 * h;                             // of the thread's half
                    float old[16];
                    if (n <= PK_RUN) {
#pragma unroll
                        for (int u = 0; u < 16; u++) old[u] = 0.0f;
                    } else if (half == 0) {
                        uint32_t y[16];
                        tmem_ld16(tmem_sum + lanes + d, y);
#pragma unroll
                        for (int u = 0; u < 16; u++) old[u] = __uint_as_float(y[u]);
                    } else {
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const float4 y = sums[(d / 4 + u) * PK_COLS];
                            old[4 * u] = y.x; old[4 * u + 1] = y.y; old[4 * u + 2] = y.z; old[4 * u + 3] = y.w;
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 16; u++) o[16 * h + u] = fmaf(old[u], aged, __uint_as_float(x[u]));
                }
                if (!on) continue;
                const float by = lim < sh->nan_from[j] ? inv : __uint_as_float(0x7FFFFFFFu);
#pragma unroll
                for (int g = 0; g < 8; g++) {
                    const float4 x = make_float4(o[g] * by, o[8 + g] * by, o[16 + g] * by, o[24 + g] * by);
                    float* at = to + 32 * j + 4 * g;
                    if (vec) *reinterpret_cast<float4*>(at) = x;
                    else { at[0] = x.x; at[1] = x.y; at[2] = x.z; at[3] = x.w; }
                }
            }
            if (on && !half && p.stat) p.stat[(size_t)unit * PK_COLS + own] = make_float2(m, log2f(l) - 14.0f);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == PK_MMA_WARP) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem_o), "r"(512u) : "memory");
    }
    if (tid == 0 && sh->abort_flag) {
        *p.err = IBCU_KV4_WAIT_ERR;
        for (int i = 0; i < 1000; i++) __nanosleep(1000);      // copies still on their way into this block's shared memory land before it goes
    }
}

// Attention that the rows draw: S^T [128 rows x 128 columns] = K' Q^T again, two threads a row, which add up its softmax weights over the columns that
// see it. A block for 128 rows, a KV head and a part of the column tiles; K' is made once and stays in tensor memory, the columns' images come through a ring. Writes
// parts [part][KV head][max_rows].
constexpr int PW_SUM_WARPS = 8, PW_MMA_WARP = 8, PW_TMA_WARP = 9, PW_THREADS = 10 * 32;
template <int NG> struct PwSmem {
    static constexpr int KB = NG / 2, IMAGE = 2 * KB * 16384, STAGE = IMAGE + 2048, DEPTH = 3;   // a tile's image, 128 factors, 128 pairs of its softmax
    static constexpr int TOTAL = DEPTH * STAGE;
};
struct PwShared { unsigned long long full[3], empty[3], d_full[2], d_empty[2], k_full, drained; uint32_t tmem_base; int abort_flag; float half[128]; };

template <int NG>
__global__ void __launch_bounds__(PW_THREADS, 1) kv4_prompt_weight_kernel(const PkParams p, float* __restrict__ parts, int n_parts) {
    using S = PwSmem<NG>;
    extern __shared__ __align__(1024) unsigned char smem[];
    PwShared* sh = reinterpret_cast<PwShared*>(smem + S::TOTAL);
    volatile int* abort_flag = &sh->abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kvh = blockIdx.x % p.c.n_kv, own_part = blockIdx.x / p.c.n_kv % n_parts;
    const int r0 = blockIdx.x / (p.c.n_kv * n_parts) * 128;    // rows that most tiles see first
    if (tid == 0) {
        auto init = [&](unsigned long long& b, int n) { mbar_init(smem_u32(&b), n); };
        for (int i = 0; i < S::DEPTH; i++) { init(sh->full[i], 1); init(sh->empty[i], PW_SUM_WARPS + 1); }
        for (int i = 0; i < 2; i++) { init(sh->d_full[i], 1); init(sh->d_empty[i], PW_SUM_WARPS); }
        init(sh->k_full, 4); init(sh->drained, 1);
        sh->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (warp == PW_MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&sh->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        pdl_launch_dependents();
    }
    pdl_wait();
    int row0, pos0;
    const bool there = kv4_place(p.at, p.t.B, p.c.max_rows, p.err, row0, pos0);
    const int R = there ? row0 + p.t.B : 0, first = max(0, r0 - row0) * p.t.group / PK_COLS + own_part;       // tiles that see a row of the block, every n_parts-th
    const int n = r0 < R && first < p.tiles ? (p.tiles - first + n_parts - 1) / n_parts : 0;
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sh->tmem_base, tmem_k = tmem + 2 * PK_COLS;                            // two accumulators, then high and low pieces of K'
    if (warp == PW_TMA_WARP) {
        if (elect_one() && n) {
            asm volatile("fence.proxy.async.global;" ::: "memory");
            int s = 0; uint32_t ph = 1;
            for (int i = 0; i < n; i++) {
                if (!mbar_wait(smem_u32(&sh->empty[s]), ph, abort_flag, 1)) break;
                const size_t unit = (size_t)kvh * p.tiles + first + i * n_parts;
                const uint32_t bar = smem_u32(&sh->full[s]), to = smem_u32(smem + s * S::STAGE);
                mbar_expect_tx(bar, S::IMAGE + 512 + 1024);
                for (int e = 0; e < S::IMAGE; e += 16384) bulk_load(to + e, p.image + unit * S::IMAGE + e, 16384, bar);
                bulk_load(to + S::IMAGE, p.qc + unit * PK_COLS, 512, bar);
                bulk_load(to + S::IMAGE + 512, p.stat + unit * PK_COLS, 1024, bar);
                if (++s == S::DEPTH) { s = 0; ph ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp == PW_MMA_WARP) {
        if (elect_one() && n) {
            constexpr uint32_t idesc = (1u << 4) | (8u << 24) | ((PK_COLS / 8) << 17);
            bool ok = mbar_wait(smem_u32(&sh->k_full), 0u, abort_flag, 2);
            int s = 0; uint32_t phs = 0;
            for (int i = 0; i < n && ok; i++) {
                const int b = i & 1;
                ok = mbar_wait(smem_u32(&sh->full[s]), phs, abort_flag, 3) && mbar_wait(smem_u32(&sh->d_empty[b]), ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag, 4);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t q = smem_desc_sw128(smem_u32(smem + s * S::STAGE));
#pragma unroll
                for (int m = 0; m < 3; m++)
#pragma unroll
                    for (int st = 0; st < 2 * NG; st++)
                        mma_f16_ts(tmem + b * PK_COLS, tmem_k + (m == 1) * 16 * NG + st * 8, q + (((m == 0) * S::KB + st / 4) * 16384 >> 4) + st % 4 * 2, idesc, m || st ? 1u : 0u);          // small products first
                mma_commit(smem_u32(&sh->empty[s]));
                mma_commit(smem_u32(&sh->d_full[b]));
                if (++s == S::DEPTH) { s = 0; phs ^= 1; }
            }
            mma_commit(smem_u32(&sh->drained));
            mbar_wait(smem_u32(&sh->drained), 0u, abort_flag, 5);
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, half = warp >> 2, own = quarter * 32 + lane, r = r0 + own;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        float sum = 0.0f;
        if (n) {
            if (half == 0) {
                const size_t row = p.c.row(kvh, min(r, R - 1));
                uint32_t sc[NG / 2];
#pragma unroll
                for (int j = 0; j < NG / 2; j++) sc[j] = __ldcg(reinterpret_cast<const uint32_t*>(p.c.scale + row * (2 * NG)) + j);
#pragma unroll 1
                for (int t = 0; t < 4; t += 2) {               // pieces of a key row, two at a time: 8 NG columns of tensor memory a part
                    uint32_t high[8 * NG], low[8 * NG];
#pragma unroll
                    for (int e = 0; e < 2 * NG; e++) {
                        const int j = e % NG;
                        const uint32_t w = __ldcg(reinterpret_cast<const uint32_t*>(p.c.k + row * (16 * NG)) + t * NG + e), k = j & 1 ? sc[j / 2] >> 16 : sc[j / 2] & 0xFFFFu;
                        __half2 f[4];
                        codes_of(w, f);
#pragma unroll
                        for (int u = 0; u < 4; u++) held_pieces(f[u], half2_of(k | k << 16), high[4 * e + u], low[4 * e + u]);
                    }
                    if constexpr (NG == 4) {
                        tmem_st32(tmem_k + lanes + t * 4 * NG, high);
                        tmem_st32(tmem_k + lanes + 16 * NG + t * 4 * NG, low);
                    } else {
                        tmem_st16(tmem_k + lanes + t * 4 * NG, high);
                        tmem_st16(tmem_k + lanes + 16 * NG + t * 4 * NG, low);
                    }
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh->k_full));
            }
            int s = 0; uint32_t phs = 0;
            for (int i = 0; i < n; i++) {
                const int b = i & 1, c0 = (first + i * n_parts) * PK_COLS;
                if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->full[s]), phs, abort_flag, 6) && mbar_wait(smem_u32(&sh->d_full[b]), (uint32_t)(i >> 1) & 1u, abort_flag, 7))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const float* f = reinterpret_cast<const float*>(smem + s * S::STAGE + S::IMAGE);
                const float2* st = reinterpret_cast<const float2*>(f + 128);
                // columns from which on the row is seen, and how many there are
                const int from = max(0, r - row0) * p.t.group - c0, upto = p.t.B * p.t.group - c0;
                const bool whole = __all_sync(0xffffffffu, from <= 0) && upto >= PK_COLS;
#pragma unroll 1
                for (int c = half * 64; c < half * 64 + 64; c += 32) {
                    uint32_t x[32];
                    tmem_ld32(tmem + lanes + b * PK_COLS + c, x);
                    tmem_wait_ld(x);
                    float part[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
                    for (int u = 0; u < 32; u += 2) {
                        const float2 ff = *reinterpret_cast<const float2*>(f + c + u);
                        const float4 ss = *reinterpret_cast<const float4*>(st + c + u);
                        const float y = ex2((__fmul_rn(__uint_as_float(x[u]), ff.x) - ss.x) - ss.y), z = ex2((__fmul_rn(__uint_as_float(x[u + 1]), ff.y) - ss.z) - ss.w);
                        part[u & 2] += whole || (c + u >= from && c + u < upto) ? y : 0.0f;
                        part[(u & 2) + 1] += whole || (c + u + 1 >= from && c + u + 1 < upto) ? z : 0.0f;
                    }
                    sum += (part[0] + part[1]) + (part[2] + part[3]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) { mbar_arrive(smem_u32(&sh->d_empty[b])); mbar_arrive(smem_u32(&sh->empty[s])); }
                if (++s == S::DEPTH) { s = 0; phs ^= 1; }
            }
        }
        if (half) sh->half[own] = sum;
        asm volatile("bar.sync 2, %0;" :: "n"(PW_SUM_WARPS * 32) : "memory");
        if (!half && r < R) parts[((size_t)own_part * p.c.n_kv + kvh) * p.c.max_rows + r] = sum + sh->half[own];
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == PW_MMA_WARP) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    }
    if (tid == 0 && sh->abort_flag) {
        *p.err = IBCU_KV4_WAIT_ERR;
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
    }
}

template <int NG>
int launch_prompt(ibcu_ctx* ctx, const PkParams& p, int rows, float* parts, int n_parts) {
    static SmemOptIn opt, opt_w;
    constexpr size_t smem = PkSmem<NG>::TOTAL + sizeof(PkShared), smem_w = PwSmem<NG>::TOTAL + sizeof(PwShared);
    static_assert(smem <= 227 * 1024 && smem_w <= 227 * 1024, "a block's shared memory");
    if (int rc = ibcu_allow_smem(ctx, opt, kv4_prompt_kernel<NG>, smem)) return rc;
    if (int rc = ibcu_launch(ctx, kv4_prompt_kernel<NG>, dim3(p.c.n_kv * p.tiles), dim3(PK_THREADS), smem, 1, true, p)) return rc;
    if (!p.stat) return IBCU_OK;
    if (int rc = ibcu_allow_smem(ctx, opt_w, kv4_prompt_weight_kernel<NG>, smem_w)) return rc;
    return ibcu_launch(ctx, kv4_prompt_weight_kernel<NG>, dim3(p.c.n_kv * n_parts * ((rows + 127) / 128)), dim3(PW_THREADS), smem_w, 1, true, p, parts, n_parts);
}

}  // namespace

// Blocks of the weights an SM: 2048 positions of 32 heads over 8, attention and weights, us with two, three and four: of 128 values 211, 218 and 221, of 64 values 188, 167 and 160.
int kv4_prompt_parts(ibcu_ctx* ctx, const Kv4& c, int tiles, int rows) {
    return std::min(std::min(tiles, 16), std::max(1, ((c.hd == 64 ? 4 : 2) * ctx->sm_count) / (((rows + 127) / 128) * c.n_kv)));
}
int kv4_prompt(ibcu_ctx* ctx, const Kv4& c, const Kv4Columns& t, const Kv4Place& at, const unsigned char* image, const float* qc, float* out, float2* stat, int rows, float* parts, int n_parts) {
    PkParams p;
    memset(&p, 0, sizeof p);
    p.c = c; p.t = t; p.at = at; p.image = image; p.qc = qc; p.out = out; p.stat = stat; p.tiles = t.ntiles / 8; p.err = ctx->kern_err;
    return c.hd == 128 ? launch_prompt<4>(ctx, p, rows, parts, n_parts) : launch_prompt<2>(ctx, p, rows, parts, n_parts);
}
