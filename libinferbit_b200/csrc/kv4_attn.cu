// Attention over the 4-bit KV cache on mma.sync (fp16 operands, FP32 sums), keeping FP32's accuracy.
//
// Scores of a KV head: [columns x values] times [values x rows]. A nibble n under the exponent of 1024 is the fp16 1024 + n (1024 + 16 n for
// the upper nibble of a byte); less 1032 (1152) it is the signed code, or 16 times it, exact. A group's sum is scaled by the row's key scale
// in FP32. Queries are two fp16 pieces of 11 bits each (2^-22 of the largest value is left out).
//     score = sum over groups j of ks[row][j] * sum_i (n_i - 8) q_i
// Outputs: [columns x rows] times [rows x values], the value codes unpacked from two rows at a time, and
//     out = sum over rows of P' (n - 8),  P' = 2^14 p vs[row][j]
// with P' split into two pieces too. (Without the subtraction unpacking is a mask alone, n as the subnormal n * 2^-24, and the bias of 8 can be
// taken off the sums. But those then are of codes that are all positive, hundreds of times their result after thousands of rows, and the
// instruction's additions round towards zero: outputs after 32767 rows were 1.5e-4 off, and 1.5e-6 with the keys alone unpacked so, against 3e-7.)
// The maximum that p refers to is that of score + L(row), 2^L a bound on the row's value scales: then P' never passes 2^14 (2^16 with the
// slack below), whatever the scales are, and a column's numbers do not depend on rows that it does not see.
//
// A block has a tile of 8 or 16 columns of one KV head and a chunk of rows; its four warps take 32 rows each in turn, every
// warp through a ring of its own that bulk copies fill (rows of a head lie one behind the other), so that no warp waits for another until the end. With
// up to 8 columns the M = 16 rows of an instruction are 8 columns twice, high and low pieces; with more they are 16 columns
// and every product is done twice.
#include "kv4.cuh"
#include "tc_common.cuh"
#include <algorithm>

namespace {

constexpr int KA_WARPS = 4, KA_ROWS = 32;            // warps of a block; rows of a ring stage
constexpr float KA_LOW = -3.0e38f;                   // where running maxima start (finite: nothing minus infinity)
constexpr float KA_SLACK = 1.9f;                     // by how much a maximum may be outgrown before the sums are rescaled

struct KaParams {
    Kv4 c; Kv4Columns t; Kv4Place at;
    const uint2* qf; const float* qc;
    float* out; float2* stat;                        // stat [unit][16] or NULL: a column's softmax weight is 2^((score - x) - y)
    float* pacc; float2* pml;                        // chunk results [unit][chunk][16][hd], [unit][chunk][16] (maximum, sum)
    int want, grid_chunks;
    int* err;
};

// `rows` rows in at most `want` chunks of whole stages; chunks of more than a stage a warp are whole rounds of the warps
__host__ __device__ __forceinline__ void ka_plan(int rows, int want, int& chunk, int& n) {
    const int stages = (rows + KA_ROWS - 1) / KA_ROWS;
    int per = (stages + want - 1) / want;
    if (per > KA_WARPS) per = (per + KA_WARPS - 1) / KA_WARPS * KA_WARPS;
    chunk = per * KA_ROWS;
    n = (stages + per - 1) / per;
}

__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) { const __half2 h = __floats2half2_rn(lo, hi); return *reinterpret_cast<const uint32_t*>(&h); }

// N 32-bit words from shared memory with the widest loads that their address allows (a multiple of 4 N)
template <int N>
__device__ __forceinline__ void lds_words(uint32_t* d, const unsigned char* s) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) { const uint4 v = *reinterpret_cast<const uint4*>(s + 4 * i); d[i] = v.x; d[i + 1] = v.y; d[i + 2] = v.z; d[i + 3] = v.w; }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) { const uint2 v = *reinterpret_cast<const uint2*>(s + 4 * i); d[i] = v.x; d[i + 1] = v.y; }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) d[i] = *reinterpret_cast<const uint32_t*>(s + 4 * i);
    }
}
// NG 16-bit units, two a word
template <int NG>
__device__ __forceinline__ void lds_units(uint32_t* d, const unsigned char* s) {
    if constexpr (NG % 2 == 0) lds_words<NG / 2>(d, s);
    else {
#pragma unroll
        for (int i = 0; i < NG; i++) {
            const uint32_t u = *reinterpret_cast<const uint16_t*>(s + 2 * i);
            if (i & 1) d[i / 2] |= u << 16; else d[i / 2] = u;
        }
    }
}
// The eight codes of a word less their bias, as four pairs: codes 0 and 4, 1 and 5 (16-fold), 2 and 6, 3 and 7 (16-fold)
__device__ __forceinline__ void unpack(uint32_t w, uint32_t* f) {
    auto less = [](uint32_t a, uint32_t b) { const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b)); return *reinterpret_cast<const uint32_t*>(&d); };
    constexpr uint32_t BASE = 0x64006400u, EIGHT = 0x64086408u, EIGHT16 = 0x64806480u;       // 1024, 1024 + 8, 1024 + 16 * 8
    f[0] = less((w & 0x000F000Fu) | BASE, EIGHT); f[1] = less((w & 0x00F000F0u) | BASE, EIGHT16);
    w >>= 8;
    f[2] = less((w & 0x000F000Fu) | BASE, EIGHT); f[3] = less((w & 0x00F000F0u) | BASE, EIGHT16);
}

template <int NG> struct KaStage {                   // a ring stage: 32 rows of keys, of values and of scales
    static constexpr int KEYS = 0, VALUES = KA_ROWS * 16 * NG, SCALES = 2 * VALUES, BYTES = SCALES + KA_ROWS * 4 * NG;
};
template <int NG, bool LARGE> struct KaSmem {
    static constexpr int DEPTH = NG > 4 ? 2 : 3;
    static constexpr int FRAGS = 0, QC = (LARGE ? 2 : 1) * NG * 1024, SCALES = QC + 128;
    static constexpr int RING = SCALES + KA_WARPS * (2 * NG + 1) * 128;
    static constexpr int TOTAL = RING + KA_WARPS * DEPTH * KaStage<NG>::BYTES;
    static_assert(KA_WARPS * (LARGE ? 16 : 8) * 32 * NG * 4 <= KA_WARPS * DEPTH * KaStage<NG>::BYTES, "the warps' results meet in the rings");
};

// A stage's scales in FP32, once per row instead of once per lane that uses them: sc [2 NG + 1][32], rows in the order t * 8 + 2 i + h
// for row 8 i + 4 h + t, so that a lane's eight rows lie side by side; the last line is L.
template <int NG, bool VALUES>
__device__ __forceinline__ void spread_scales(float* sc, const unsigned char* rows, int lane) {
    uint32_t w[NG];
    lds_words<NG>(w, rows + lane * 4 * NG);
    float* d = sc + (lane & 3) * 8 + (lane >> 3) * 2 + ((lane >> 2) & 1);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < (VALUES ? 2 * NG : NG); j++) {
        const uint32_t u = j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu;
        if (j >= NG) top = max(top, u & 0x7FFFu);
        d[j * 32] = __half2float(__ushort_as_half((unsigned short)u));
    }
    if (VALUES) d[2 * NG * 32] = (float)((int)(top >> 10) - 14);       // scales stay below 2^(exponent - 14)
}

// Scores of 32 rows: s[i][h][n] for row 8 i + 4 h + t and column g (n = 0), g + 8 (n = 1), in the column's own units
template <int NG, bool LARGE>
__device__ __forceinline__ void score_rows(float (&s)[4][2][LARGE ? 2 : 1], const uint32_t (&kw)[4][NG], const uint2* qf, const float* sc, int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int n = 0; n < (LARGE ? 2 : 1); n++) s[i][h][n] = 0.0f;
#pragma unroll
    for (int j = 0; j < NG; j++) {
        uint2 a[LARGE ? 2 : 1][2][2];
#pragma unroll
        for (int p = 0; p < (LARGE ? 2 : 1); p++)
#pragma unroll
            for (int st = 0; st < 2; st++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) a[p][st][hf] = qf[(((p * NG + j) * 2 + st) * 2 + hf) * 32 + lane];
        const float4 k0 = *reinterpret_cast<const float4*>(sc + j * 32 + t * 8), k1 = *reinterpret_cast<const float4*>(sc + j * 32 + t * 8 + 4);
        const float ks[4][2] = { { k0.x, k0.y }, { k0.z, k0.w }, { k1.x, k1.y }, { k1.z, k1.w } };
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t f[4];
            unpack(kw[i][j], f);
            float c[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
            for (int p = 0; p < (LARGE ? 2 : 1); p++) {
                mma_f16(c, a[p][0][0].x, a[p][0][1].x, a[p][0][0].y, a[p][0][1].y, f[0], f[1]);
                mma_f16(c, a[p][1][0].x, a[p][1][1].x, a[p][1][0].y, a[p][1][1].y, f[2], f[3]);
            }
            if constexpr (LARGE) {
#pragma unroll
                for (int n = 0; n < 2; n++) { s[i][0][n] = fmaf(ks[i][0], c[2 * n], s[i][0][n]); s[i][1][n] = fmaf(ks[i][1], c[2 * n + 1], s[i][1][n]); }
            } else {
                s[i][0][0] = fmaf(ks[i][0], c[0] + c[2], s[i][0][0]);
                s[i][1][0] = fmaf(ks[i][1], c[1] + c[3], s[i][1][0]);
            }
        }
    }
}

template <int NG, bool LARGE>
__global__ void __launch_bounds__(32 * KA_WARPS, NG > 4 ? 1 : (LARGE ? 2 : 3)) kv4_attn_kernel(const KaParams p) {
    using S = KaSmem<NG, LARGE>;
    using St = KaStage<NG>;
    constexpr int NC = LARGE ? 2 : 1, COLS = 8 * NC, HD = 32 * NG;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ unsigned long long full[KA_WARPS][S::DEPTH];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int tile = p.t.ntiles - 1 - blockIdx.x % p.t.ntiles, kvh = blockIdx.x / p.t.ntiles, sp = blockIdx.y;   // tiles that see most rows first
    const int unit = kvh * p.t.ntiles + tile, c0 = tile * COLS;
    if (tid == 0) {
        abort_flag = 0;
        for (int w = 0; w < KA_WARPS; w++) for (int d = 0; d < S::DEPTH; d++) mbar_init(smem_u32(&full[w][d]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // Launches ahead of the preparing one have ended when this one starts, since that one lets it start behind its own wait: what they wrote (a
    // device position, rows of earlier calls) may be read before this launch's own wait.
    int row0, pos0;
    if (!kv4_place(p.at, p.t.B, p.c.max_rows, p.err, row0, pos0)) return;
    int chunk, n_chunks;
    ka_plan(row0 + p.t.B, p.want, chunk, n_chunks);
    if (sp >= n_chunks) return;
    const int lim0 = row0 + c0 / p.t.group;                                                        // the last row that the tile's first column sees
    const int t0 = sp * chunk, t1 = min(t0 + chunk, row0 + min(p.t.B - 1, (c0 + COLS - 1) / p.t.group) + 1);
    const int stages = t1 > t0 ? (t1 - t0 + KA_ROWS - 1) / KA_ROWS : 0, mine = stages > warp ? (stages - warp + KA_WARPS - 1) / KA_WARPS : 0;
    unsigned char* ring = smem + S::RING + warp * S::DEPTH * St::BYTES;
    const size_t plane = p.c.row(kvh, 0);
    auto issue = [&](int n) {                                                                      // one lane: the n-th stage of this warp; whole groups of 8 rows, which the planes have
        const int r = t0 + (warp + n * KA_WARPS) * KA_ROWS, rows = min(KA_ROWS, (t1 - r + 7) & ~7), d = n % S::DEPTH;
        const uint32_t bar = smem_u32(&full[warp][d]), to = smem_u32(ring + d * St::BYTES);
        mbar_expect_tx(bar, (uint32_t)rows * 36 * NG);
        bulk_load(to + St::KEYS, p.c.k + (plane + r) * (16 * NG), (uint32_t)rows * 16 * NG, bar);
        bulk_load(to + St::VALUES, p.c.v + (plane + r) * (16 * NG), (uint32_t)rows * 16 * NG, bar);
        bulk_load(to + St::SCALES, p.c.scale + (plane + r) * (2 * NG), (uint32_t)rows * 4 * NG, bar);
    };
    int issued = 0;
    if (lane == 0)
        for (; issued < min(mine, (int)S::DEPTH) && t0 + (warp + issued * KA_WARPS) * KA_ROWS + KA_ROWS <= row0; issued++) issue(issued);
    pdl_wait();
    pdl_launch_dependents();
    if (lane == 0) {
        asm volatile("fence.proxy.async.global;" ::: "memory");                                    // rows that the preparing launch wrote
        for (; issued < min(mine, (int)S::DEPTH); issued++) issue(issued);
    }
    uint2* qf = reinterpret_cast<uint2*>(smem + S::FRAGS);
    float* qc = reinterpret_cast<float*>(smem + S::QC);
    {
        const uint4* src = reinterpret_cast<const uint4*>(p.qf + unit * kv4_frag_uint2(NG, LARGE));
        for (int e = tid; e < NC * NG * 64; e += 32 * KA_WARPS) reinterpret_cast<uint4*>(qf)[e] = __ldcg(src + e);
        if (tid < COLS) qc[tid] = __ldcg(p.qc + (size_t)unit * 16 + tid);
    }
    __syncthreads();
    float* sc = reinterpret_cast<float*>(smem + S::SCALES) + warp * (2 * NG + 1) * 32;
    float f[NC], m[NC], l[NC], acc[NG][4][4];
    int lim[NC];
#pragma unroll
    for (int n = 0; n < NC; n++) {
        f[n] = qc[g + 8 * n]; m[n] = KA_LOW; l[n] = 0.0f;
        lim[n] = row0 + (c0 + g + 8 * n) / p.t.group;
    }
#pragma unroll
    for (int j = 0; j < NG; j++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int u = 0; u < 4; u++) acc[j][i][u] = 0.0f;

    uint32_t phase = 0;
    int d = 0;
    bool wide = false;
    for (int it = 0; it < mine; it++) {
        const int r0 = t0 + (warp + it * KA_WARPS) * KA_ROWS;
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&full[warp][d]), phase, &abort_flag, IBCU_KV4_WAIT_ERR))) break;
        const unsigned char* stage = ring + d * St::BYTES;
        spread_scales<NG, true>(sc, stage + St::SCALES, lane);
        uint32_t kw[4][NG], vw[4][2][(NG + 1) / 2];
#pragma unroll
        for (int i = 0; i < 4; i++) lds_words<NG>(kw[i], stage + St::KEYS + (8 * i + (g >> 1) + 4 * (g & 1)) * 16 * NG + t * 4 * NG);
        __syncwarp();
        float s[4][2][NC];
        score_rows<NG, LARGE>(s, kw, qf, sc, lane);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) lds_units<NG>(vw[i][h], stage + St::VALUES + (8 * i + 4 * h + t) * 16 * NG + g * 2 * NG);
        __syncwarp();
        if (lane == 0 && it + S::DEPTH < mine) issue(it + S::DEPTH);                               // everything of the stage is in registers
        if (++d == S::DEPTH) { d = 0; phase ^= 1; }

        auto weigh = [&](auto masked) {
            constexpr bool MASK = decltype(masked)::value;
            const float4 l0 = *reinterpret_cast<const float4*>(sc + 2 * NG * 32 + t * 8), l1 = *reinterpret_cast<const float4*>(sc + 2 * NG * 32 + t * 8 + 4);
            const float L[4][2] = { { l0.x, l0.y }, { l0.z, l0.w }, { l1.x, l1.y }, { l1.z, l1.w } };
            auto seen = [&](int i, int h, int n) { return !MASK || r0 + 8 * i + 4 * h + t <= lim[n]; };
            float top[NC];
            bool grow = false;
#pragma unroll
            for (int n = 0; n < NC; n++) {
                top[n] = KA_LOW;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        s[i][h][n] *= f[n];
                        if (seen(i, h, n)) top[n] = fmaxf(top[n], s[i][h][n] + L[i][h]);
                    }
                top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], 1));
                top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], 2));
                grow = grow || top[n] > m[n] + KA_SLACK;
            }
            if (__any_sync(0xffffffffu, grow)) {
                wide = false;
#pragma unroll
                for (int n = 0; n < NC; n++) {
                    const float now = fmaxf(m[n], top[n]), corr = ex2(m[n] - now);
                    m[n] = now;
                    wide = wide || fabsf(now) > 524288.0f;
                    l[n] *= corr;
#pragma unroll
                    for (int j = 0; j < NG; j++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            if (LARGE) { acc[j][i][2 * n] *= corr; acc[j][i][2 * n + 1] *= corr; }
                            else { acc[j][i][0] *= corr; acc[j][i][1] *= corr; acc[j][i][2] *= corr; acc[j][i][3] *= corr; }
                        }
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int h = 0; h < 2; h++) s[i][h][n] -= m[n];
            // Beyond 2^19 (log2 units; such a softmax has one row) the maximum itself is rounded by more than the slack allows for.
            if (__any_sync(0xffffffffu, wide)) {
#pragma unroll
                for (int n = 0; n < NC; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int h = 0; h < 2; h++) s[i][h][n] = s[i][h][n] > 1.0f - L[i][h] ? 1.0f - L[i][h] : s[i][h][n];
            }
#pragma unroll
            for (int n = 0; n < NC; n++) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float e = seen(i, h, n) ? ex2(s[i][h][n] + 14.0f) : 0.0f;
                        s[i][h][n] = e;
                        l[n] += e;
                    }
            }
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const float4 v0 = *reinterpret_cast<const float4*>(sc + (NG + j) * 32 + t * 8), v1 = *reinterpret_cast<const float4*>(sc + (NG + j) * 32 + t * 8 + 4);
                const float vs[4][2] = { { v0.x, v0.y }, { v0.z, v0.w }, { v1.x, v1.y }, { v1.z, v1.w } };
#pragma unroll
                for (int u = 0; u < 2; u++) {                                                      // 16 rows: pieces 2 u and 2 u + 1
                    uint32_t hi[2][NC], lo[2][NC];
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int n = 0; n < NC; n++) {
                            float a = s[2 * u + i][0][n] * vs[2 * u + i][0], b = s[2 * u + i][1][n] * vs[2 * u + i][1];
                            if (!seen(2 * u + i, 0, n)) a = 0.0f;                                  // the row's scale may be NaN
                            if (!seen(2 * u + i, 1, n)) b = 0.0f;
                            hi[i][n] = pack_half(a, b);
                            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi[i][n]));
                            lo[i][n] = pack_half(a - back.x, b - back.y);
                        }
                    uint32_t x0 = __byte_perm(vw[2 * u][0][j / 2], vw[2 * u][1][j / 2], j & 1 ? 0x7632 : 0x5410);
                    uint32_t x1 = __byte_perm(vw[2 * u + 1][0][j / 2], vw[2 * u + 1][1][j / 2], j & 1 ? 0x7632 : 0x5410);
                    uint32_t b0[4], b1[4];
                    unpack(x0, b0);
                    unpack(x1, b1);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if constexpr (LARGE) {
                            mma_f16(acc[j][i], hi[0][0], hi[0][1], hi[1][0], hi[1][1], b0[i], b1[i]);
                            mma_f16(acc[j][i], lo[0][0], lo[0][1], lo[1][0], lo[1][1], b0[i], b1[i]);
                        } else {
                            mma_f16(acc[j][i], hi[0][0], lo[0][0], hi[1][0], lo[1][0], b0[i], b1[i]);
                        }
                    }
                }
            }
        };
        if (r0 + KA_ROWS - 1 <= lim0) weigh(std::false_type());
        else weigh(std::true_type());
        __syncwarp();                                                                              // the scales may be overwritten
    }

    // the four warps' results meet in the rings: [warp][column][value], and maxima and sums
    __shared__ float2 ml[KA_WARPS][16];
#pragma unroll
    for (int n = 0; n < NC; n++) {
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
        if (t == 0) ml[warp][g + 8 * n] = make_float2(m[n], l[n]);
    }
    __syncthreads();
    float* meet = reinterpret_cast<float*>(smem + S::RING);
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int j = 0; j < NG; j++) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const float a = LARGE ? acc[j][i][2 * n + u] : acc[j][i][u] + acc[j][i][u + 2];
                    o[4 * u + i] = i & 1 ? a * 0.0625f : a;
                }
            float4* to = reinterpret_cast<float4*>(meet + ((size_t)warp * COLS + g + 8 * n) * HD + 32 * j + 8 * t);
            to[0] = make_float4(o[0], o[1], o[2], o[3]);
            to[1] = make_float4(o[4], o[5], o[6], o[7]);
        }
    __syncthreads();
    if (tid == 0 && abort_flag) {
        *p.err = abort_flag;
        for (int i = 0; i < 1000; i++) __nanosleep(1000);      // copies still on their way into this block's shared memory land before it goes
    }
    for (int e = tid; e < COLS * HD / 4; e += 32 * KA_WARPS) {
        const int col = e / (HD / 4), d4 = e % (HD / 4), c = c0 + col, b = c / p.t.group;
        if (b >= p.t.B) break;
        float M = ml[0][col].x, wsum = 0.0f;
#pragma unroll
        for (int w = 1; w < KA_WARPS; w++) M = fmaxf(M, ml[w][col].x);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < KA_WARPS; w++) {
            const float k = ex2(ml[w][col].x - M);
            const float4 v = *reinterpret_cast<const float4*>(meet + ((size_t)w * COLS + col) * HD + 4 * d4);
            wsum = fmaf(ml[w][col].y, k, wsum);
            o.x = fmaf(v.x, k, o.x); o.y = fmaf(v.y, k, o.y); o.z = fmaf(v.z, k, o.z); o.w = fmaf(v.w, k, o.w);
        }
        if (n_chunks == 1) {
            float* to = p.out + ((size_t)b * p.t.n_heads + (size_t)kvh * p.t.group + c % p.t.group) * HD + 4 * d4;
            const float inv = 1.0f / wsum;
            to[0] = o.x * inv; to[1] = o.y * inv; to[2] = o.z * inv; to[3] = o.w * inv;
            if (d4 == 0 && p.stat) p.stat[(size_t)unit * 16 + col] = make_float2(M, log2f(wsum) - 14.0f);
        } else {
            const size_t at = ((size_t)unit * p.grid_chunks + sp) * 16 + col;
            *reinterpret_cast<float4*>(p.pacc + at * HD + 4 * d4) = o;
            if (d4 == 0) p.pml[at] = make_float2(M, wsum);
        }
    }
}

// grid (columns of a tile, units): the chunks of a column joined
__global__ void __launch_bounds__(128) kv4_join_kernel(const KaParams p) {
    extern __shared__ __align__(16) float4 part[];            // [threads]
    pdl_launch_dependents();
    pdl_wait();
    int row0, pos0, chunk, n;
    if (!kv4_place(p.at, p.t.B, p.c.max_rows, p.err, row0, pos0)) return;
    ka_plan(row0 + p.t.B, p.want, chunk, n);
    const int unit = blockIdx.y, kvh = unit / p.t.ntiles, tile = unit % p.t.ntiles, col = blockIdx.x, cc = tile * p.t.cols() + col, b = cc / p.t.group;
    if (n == 1 || b >= p.t.B) return;
    const int q4 = p.c.hd / 4, lanes = min(q4, 64), ways = 128 / lanes, way = threadIdx.x / lanes, tid = threadIdx.x;
    const size_t base = (size_t)unit * p.grid_chunks * 16 + col;
    float M = KA_LOW;
    for (int s = tid & 31; s < n; s += 32) M = fmaxf(M, __ldcg(&p.pml[base + (size_t)s * 16].x));
    M = warp_max(M);
    float sum = 0.0f;
    for (int s = tid & 31; s < n; s += 32) { const float2 v = __ldcg(&p.pml[base + (size_t)s * 16]); sum = fmaf(v.y, ex2(v.x - M), sum); }
    sum = warp_sum(sum);
    const float inv = 1.0f / sum;
    if (way < ways) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        const int d4 = tid % lanes;
#pragma unroll 4
        for (int s = way; s < n; s += ways) {
            const float k = ex2(__ldcg(&p.pml[base + (size_t)s * 16].x) - M);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p.pacc + (base + (size_t)s * 16) * p.c.hd) + d4);
            o.x = fmaf(v.x, k, o.x); o.y = fmaf(v.y, k, o.y); o.z = fmaf(v.z, k, o.z); o.w = fmaf(v.w, k, o.w);
        }
        part[tid] = o;
    }
    __syncthreads();
    if (tid < q4) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < ways; w++) { const float4 v = part[w * lanes + tid]; o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w; }
        float* to = p.out + ((size_t)b * p.t.n_heads + (size_t)kvh * p.t.group + cc % p.t.group) * p.c.hd + 4 * tid;
        to[0] = o.x * inv; to[1] = o.y * inv; to[2] = o.z * inv; to[3] = o.w * inv;
    }
    if (tid == 0 && p.stat) p.stat[(size_t)unit * 16 + col] = make_float2(M, log2f(sum) - 14.0f);
}

// Attention that the rows draw. grid (128 rows, KV heads, parts of the tiles): a warp holds the keys of 32 rows and walks the columns that see them; the
// scores are computed again, which costs less than writing them down once there are several columns. The parts of a row are added in order.
template <int NG, bool LARGE>
__global__ void __launch_bounds__(128) kv4_weight_kernel(const KaParams p, float decay, float* __restrict__ parts) {
    constexpr int NC = LARGE ? 2 : 1, COLS = 8 * NC;
    __shared__ __align__(16) uint2 qf[NC * NG * 128];
    __shared__ float qc[16];
    __shared__ float2 st[16];
    __shared__ __align__(16) float scales[4][NG * 32];
    pdl_launch_dependents();
    pdl_wait();
    int row0, pos0;
    if (!kv4_place(p.at, p.t.B, p.c.max_rows, p.err, row0, pos0)) return;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, kvh = blockIdx.y, R = row0 + p.t.B;
    const int r0 = blockIdx.x * 128 + warp * 32;
    if ((int)blockIdx.x * 128 >= R) return;
    float* sc = scales[warp];
    uint32_t kw[4][NG];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = min(r0 + 8 * i + (g >> 1) + 4 * (g & 1), R - 1);
        const uint32_t* src = reinterpret_cast<const uint32_t*>(p.c.k + p.c.row(kvh, r) * (16 * NG)) + t * NG;
#pragma unroll
        for (int j = 0; j < NG; j++) kw[i][j] = __ldcg(src + j);
    }
    {
        const __half* src = p.c.scale + p.c.row(kvh, min(r0 + lane, R - 1)) * (2 * NG);
        float* d = sc + (lane & 3) * 8 + (lane >> 3) * 2 + ((lane >> 2) & 1);
        for (int j = 0; j < NG; j++) d[j * 32] = __half2float(__ushort_as_half(__ldcg(reinterpret_cast<const unsigned short*>(src) + j)));
    }
    float w[4][2] = {};
    const int first = max(0, (int)blockIdx.x * 128 - row0) * p.t.group / COLS;                    // the first tile that sees a row of the block
    for (int tile = first + blockIdx.z; tile < p.t.ntiles; tile += gridDim.z) {
        const int unit = kvh * p.t.ntiles + tile, c0 = tile * COLS;
        __syncthreads();
        const uint4* src = reinterpret_cast<const uint4*>(p.qf + unit * kv4_frag_uint2(NG, LARGE));
        for (int e = tid; e < NC * NG * 64; e += 128) reinterpret_cast<uint4*>(qf)[e] = __ldcg(src + e);
        if (tid < COLS) qc[tid] = __ldcg(p.qc + (size_t)unit * 16 + tid);
        if (tid < COLS) st[tid] = __ldcg(p.stat + (size_t)unit * 16 + tid);
        __syncthreads();
        float s[4][2][NC];
        score_rows<NG, LARGE>(s, kw, qf, sc, lane);
#pragma unroll
        for (int n = 0; n < NC; n++) {
            const int c = c0 + g + 8 * n, b = c / p.t.group, lim = b < p.t.B ? row0 + b : -1;
            const float f = qc[g + 8 * n];
            const float2 off = st[g + 8 * n];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) if (r0 + 8 * i + 4 * h + t <= lim) w[i][h] += ex2((__fmul_rn(s[i][h][n], f) - off.x) - off.y);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float x = w[i][h];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            const int r = r0 + 8 * i + 4 * h + t;
            if (g == 0 && r < R) {
                const size_t at = p.c.row(kvh, r);
                if (parts) parts[((size_t)blockIdx.z * p.c.n_kv + kvh) * p.c.max_rows + r] = x;
                else p.c.weight[at] = (decay == 0.0f ? 0.0f : decay * __ldcg(p.c.weight + at)) + x;
            }
        }
}
__global__ void __launch_bounds__(256) kv4_weight_join_kernel(const KaParams p, float decay, const float* __restrict__ parts, int n) {
    pdl_launch_dependents();
    pdl_wait();
    int row0, pos0;
    if (!kv4_place(p.at, p.t.B, p.c.max_rows, p.err, row0, pos0)) return;
    const int r = blockIdx.x * 256 + threadIdx.x;
    if (r >= row0 + p.t.B) return;
    const size_t at = p.c.row(blockIdx.y, r);
    float x = 0.0f;
    for (int i = 0; i < n; i++) x += __ldcg(parts + (size_t)i * p.c.n_kv * p.c.max_rows + at);
    p.c.weight[at] = (decay == 0.0f ? 0.0f : decay * __ldcg(p.c.weight + at)) + x;
}

template <int NG, bool LARGE>
int launch_attention(ibcu_ctx* ctx, const KaParams& p, int units, int chunks, int rows, float decay, float* parts, int n_parts) {
    static SmemOptIn opt;
    if (int rc = ibcu_allow_smem(ctx, opt, kv4_attn_kernel<NG, LARGE>, KaSmem<NG, LARGE>::TOTAL)) return rc;
    int rc = ibcu_launch(ctx, kv4_attn_kernel<NG, LARGE>, dim3(units, chunks), dim3(32 * KA_WARPS), KaSmem<NG, LARGE>::TOTAL, 1, true, p);
    if (!rc && chunks > 1) rc = ibcu_launch(ctx, kv4_join_kernel, dim3(p.t.cols(), units), dim3(128), 128 * sizeof(float4), 1, true, p);
    if (rc || !p.stat) return rc;
    rc = ibcu_launch(ctx, kv4_weight_kernel<NG, LARGE>, dim3((rows + 127) / 128, p.c.n_kv, n_parts), dim3(128), 0, 1, true, p, decay, n_parts > 1 ? parts : (float*)nullptr);
    if (!rc && n_parts > 1) rc = ibcu_launch(ctx, kv4_weight_join_kernel, dim3((rows + 255) / 256, p.c.n_kv), dim3(256), 0, 1, true, p, decay, (const float*)parts, n_parts);
    return rc;
}
template <int NG>
int launch_attention(ibcu_ctx* ctx, const KaParams& p, int units, int chunks, int rows, float decay, float* parts, int n_parts) {
    return p.t.large ? launch_attention<NG, true>(ctx, p, units, chunks, rows, decay, parts, n_parts) : launch_attention<NG, false>(ctx, p, units, chunks, rows, decay, parts, n_parts);
}

}  // namespace

int kv4_attend(ibcu_ctx* ctx, const Kv4& c, float decay, const Kv4Place& at, const float* q, const float* k, const float* v, float* out, int n_heads, int B, double log2_theta, int rotate) {
    const int group = n_heads / c.n_kv, ng = c.hd / 32;
    const long columns = (long)B * group;
    const int large = columns > 8, ntiles = (int)((columns + (large ? 15 : 7)) / (large ? 16 : 8)), units = c.n_kv * ntiles;
    const int rows = at.at ? c.max_rows : at.row0 + B;
    const Kv4Columns t = { n_heads, group, B, large, ntiles };
    int want = std::max(1, (large ? 2 : 3) * ctx->sm_count / units), chunk, chunks;
    ka_plan(rows, want, chunk, chunks);
    if (at.at) chunks = std::min(want, (rows + KA_ROWS - 1) / KA_ROWS);                            // shorter contexts have more, shorter chunks
    const int row_blocks = (rows + 127) / 128;
    int n_parts = c.weight ? std::min(std::min(ntiles, 16), std::max(1, 6 * ctx->sm_count / (row_blocks * c.n_kv))) : 1;
    auto round_up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    const size_t b_qf = round_up(units * kv4_frag_uint2(ng, large) * sizeof(uint2)), b_qc = round_up((size_t)units * 16 * sizeof(float));
    const size_t b_stat = c.weight ? round_up((size_t)units * 16 * sizeof(float2)) : 0, b_ml = chunks > 1 ? round_up((size_t)units * chunks * 16 * sizeof(float2)) : 0;
    const size_t b_acc = chunks > 1 ? round_up((size_t)units * chunks * 16 * c.hd * sizeof(float)) : 0, b_parts = n_parts > 1 ? round_up((size_t)n_parts * c.n_kv * c.max_rows * sizeof(float)) : 0;
    if (int rc = ibcu_reserve(ctx, &ctx->scratch, &ctx->scratch_bytes, b_qf + b_qc + b_stat + b_ml + b_acc + b_parts)) return rc;
    char* s = (char*)ctx->scratch;
    auto take = [&](size_t n) { char* r = s; s += n; return r; };
    KaParams p;
    memset(&p, 0, sizeof p);
    p.c = c; p.t = t; p.at = at;
    uint2* qf = (uint2*)take(b_qf); float* qc = (float*)take(b_qc);
    p.qf = qf; p.qc = qc;
    p.stat = (float2*)take(b_stat); if (!c.weight) p.stat = nullptr;
    p.pml = (float2*)take(b_ml); p.pacc = (float*)take(b_acc);
    float* parts = (float*)take(b_parts);
    p.out = out; p.want = want; p.grid_chunks = chunks; p.err = ctx->kern_err;
    if (int rc = kv4_prepare(ctx, c, t, at, Kv4Prep{ q, k, v, qf, qc, log2_theta, rotate })) return rc;
    switch (ng) {
        case 1: return launch_attention<1>(ctx, p, units, chunks, rows, decay, parts, n_parts);
        case 2: return launch_attention<2>(ctx, p, units, chunks, rows, decay, parts, n_parts);
        case 3: return launch_attention<3>(ctx, p, units, chunks, rows, decay, parts, n_parts);
        case 4: return launch_attention<4>(ctx, p, units, chunks, rows, decay, parts, n_parts);
        case 6: return launch_attention<6>(ctx, p, units, chunks, rows, decay, parts, n_parts);
        default: return launch_attention<8>(ctx, p, units, chunks, rows, decay, parts, n_parts);
    }
}
