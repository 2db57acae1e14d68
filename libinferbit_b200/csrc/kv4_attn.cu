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
// instruction's additions round towards zero: outputs after 32767 rows were 1.5e-4 off, and 1.5e-6 with the keys alone unpacked so, against 3e-7.
// For the same reason 32 rows are summed by themselves and added to the sums rounded: in the instruction's own sums 16000 rows of one block were 2.8e-6 off.)
// The maximum that p refers to is that of score + L(row), 2^L a bound on the row's value scales: then P' never passes 2^14 (2^16 with the
// slack below), whatever the scales are, and a column's numbers do not depend on rows that it does not see.
//
// A warp has a tile of 8 or 16 columns of one KV head and takes 32 rows at a time through a ring of its own that bulk copies fill (rows of a
// head lie one behind the other), so that no warp waits for another before the end; the four warps of a block share the tile's rows and put their
// results together. Tiles of
//   4     keys and values as the M = 16 rows of an instruction, the columns' high and low pieces as its N = 8: a group of up to four query heads and one token.
//         728 instructions for 32 rows of 128 values, against 973 with tiles of eight;
//   8     the columns, as high and low pieces, are the M = 16 rows;
//   16    every product is done twice, once for each piece (LARGE), after a launch that prepares the queries and writes the call's rows. Blocks of the
//         others do both for themselves, in their one launch.
// A column's rows are cut into chunks where that fills the machine. The chunks' blocks stand in clusters, which put their results together in shared
// memory; up to eight chunks are one cluster, the results of more clusters are put together by a launch of its own. (32 heads of 128 values over
// 8 KV heads, one token after 512 rows: 6.4 us, against 8.6 with a second launch and 9.7 with the last block of a tile to finish doing it; after 4000: 9.0
// against 10.3 with clusters of four and a second launch.)
// What bounds it: instructions, of which a word of eight codes takes nine to unpack. After 32767 rows 18.4 us, 2.1 TB/s of cache, of which 11 us are the start, the ring's first
// copies and the joins; after 262143 rows 78 us, 3.9 TB/s.
#include "kv4.cuh"
#include "tc_common.cuh"
#include <algorithm>

namespace {

constexpr int KA_WARPS = 4, KA_ROWS = 32;            // warps of a block; rows of a ring stage
constexpr int KA_CLUSTER = 8;                        // blocks of a cluster at most
// Tiles up to which the scores are written down for the weights instead of computed again: 32 heads of 128 values over 8, two tiles after 1536 rows 15.8 us instead of 23.4, four
// 21.6 instead of 31.3; eight after 8000 rows, a thread a row, 76.8 against 70.3.
constexpr int KA_FEW_TILES = 4;
constexpr float KA_LOW = -3.0e38f;                   // where running maxima start (finite: nothing minus infinity)
constexpr float KA_SLACK = 1.9f;                     // by how much a maximum may be outgrown before the sums are rescaled

struct KaParams {
    Kv4 c; Kv4Columns t; Kv4Place at; Kv4Prep w;     // w.qf, w.qc: prepared fragments (LARGE)
    float* out; float2* stat;                        // stat [unit][16] or NULL: a column's softmax weight is 2^((score - x) - y)
    float* pacc; float2* pml;                        // results of clusters [unit][cluster][16][hd], [unit][cluster][16] (maximum, sum)
    float* scores; int score_rows;                   // few tiles, for the weights, or NULL: [unit][score_rows][column]
    int want, grid_chunks, cluster;                  // chunks at most; blocks a tile, whole clusters of them
    int* err;
};

// `rows` rows in at most `want` chunks of whole rounds of the warps; in one cluster's where that leaves four rounds at most
__host__ __device__ __forceinline__ void ka_plan(int rows, int want, int cluster, int& chunk, int& n) {
    const int stages = (rows + KA_ROWS - 1) / KA_ROWS;
    if (stages <= cluster * KA_WARPS * 4) want = want < cluster ? want : cluster;
    const int per = ((stages + want - 1) / want + KA_WARPS - 1) / KA_WARPS * KA_WARPS;
    chunk = per * KA_ROWS;
    n = (stages + per - 1) / per;
}

__device__ __forceinline__ void mma_f16(float* c, const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float* c, const uint4& a, uint32_t b0, uint32_t b1) {          // nothing to add to
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) { uint32_t d; asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a)); return d; }
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
// (w & mask) | base as the one instruction that it is (the compiler makes two of it, which were 128 of the 855 of a stage)
__device__ __forceinline__ uint32_t under(uint32_t w, uint32_t mask, uint32_t base) { uint32_t d; asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(mask), "r"(base)); return d; }
// The eight codes of a word less their bias, as four pairs: codes 0 and 4, 1 and 5 (16-fold), 2 and 6, 3 and 7 (16-fold)
__device__ __forceinline__ void unpack(uint32_t w, uint32_t* f) {
    auto less = [](uint32_t a, uint32_t b) { const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b)); return *reinterpret_cast<const uint32_t*>(&d); };
    constexpr uint32_t BASE = 0x64006400u, EIGHT = 0x64086408u, EIGHT16 = 0x64806480u;       // 1024, 1024 + 8, 1024 + 16 * 8
    f[0] = less(under(w, 0x000F000Fu, BASE), EIGHT); f[1] = less(under(w, 0x00F000F0u, BASE), EIGHT16);
    w >>= 8;
    f[2] = less(under(w, 0x000F000Fu, BASE), EIGHT); f[3] = less(under(w, 0x00F000F0u, BASE), EIGHT16);
}

template <int NG> struct KaStage {                   // a ring stage: 32 rows of keys, of values and of scales
    static constexpr int KEYS = 0, VALUES = KA_ROWS * 16 * NG, SCALES = 2 * VALUES, BYTES = SCALES + KA_ROWS * 4 * NG;
};
template <int NG, int COLS> struct KaSmem {
    static constexpr bool LARGE = COLS == 16;
    static constexpr int DEPTH = NG > 4 || COLS == 4 ? 2 : 3, FRAG_BYTES = (LARGE ? 2 : 1) * NG * 1024;
    static constexpr int FRAGS = 0, QC = FRAG_BYTES, SCALES = QC + 128;
    static constexpr int RING = SCALES + KA_WARPS * (2 * NG + 1) * 128;
    static constexpr int TOTAL = RING + KA_WARPS * DEPTH * KaStage<NG>::BYTES;       // few: angles of the positions follow
    static_assert(KA_WARPS * COLS * 32 * NG * 4 <= KA_WARPS * DEPTH * KaStage<NG>::BYTES, "the warps' results meet in the rings");
};

// A stage's scales in FP32, once per row instead of once per lane that uses them: sc [2 NG + 1][32], rows in the order t * 8 + 2 i + h
// for row 8 i + 4 h + t, so that a lane's eight rows lie side by side; the last line is L.
// (FOUR: row 8 i + (g >> 1) + 4 (g & 1) at g * 4 + i.)
template <int NG, bool FOUR>
__device__ __forceinline__ void spread_scales(float* sc, const unsigned char* rows, int lane) {
    uint32_t w[NG];
    lds_words<NG>(w, rows + lane * 4 * NG);
    float* d = sc + (FOUR ? (lane & 3) * 8 + ((lane >> 2) & 1) * 4 + (lane >> 3) : (lane & 3) * 8 + (lane >> 3) * 2 + ((lane >> 2) & 1));
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NG; j++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        d[2 * j * 32] = f.x;
        d[(2 * j + 1) * 32] = f.y;
        // groups NG.. are the values'
        if (2 * j >= NG) top = max(top, w[j] & 0x7FFFu);
        if (2 * j + 1 >= NG) top = max(top, w[j] >> 16 & 0x7FFFu);
    }
    d[2 * NG * 32] = (float)((int)(top >> 10) - 14);          // scales stay below 2^(exponent - 14)
}
// a lane's eight rows of a line of sc
__device__ __forceinline__ void lane_rows(float (&x)[4][2], const float* line, int t) {
    const float4 a = *reinterpret_cast<const float4*>(line + t * 8), b = *reinterpret_cast<const float4*>(line + t * 8 + 4);
    x[0][0] = a.x; x[0][1] = a.y; x[1][0] = a.z; x[1][1] = a.w; x[2][0] = b.x; x[2][1] = b.y; x[3][0] = b.z; x[3][1] = b.w;
}

// Scores of 32 rows for up to four columns. s[i]: row 8 i + (g >> 1) + 4 (g & 1), column t, in the column's own units.
template <int NG>
__device__ __forceinline__ void score_rows_four(float (&s)[4][1][1], const uint32_t (&kw)[4][NG], const uint2* qf, const float* sc, int lane) {
#pragma unroll
    for (int j = 0; j < NG; j++) {
        const uint2 b0 = qf[(j * 2) * 32 + lane], b1 = qf[(j * 2 + 1) * 32 + lane];
        const float4 line = *reinterpret_cast<const float4*>(sc + j * 32 + (lane >> 2) * 4);
        const float ks[4] = { line.x, line.y, line.z, line.w };
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            uint32_t u[4], w[4];
            unpack(kw[i][j], u);
            unpack(kw[i + 1][j], w);
            float c[4];
            mma_f16_first(c, make_uint4(u[0], w[0], u[1], w[1]), b0.x, b0.y);
            mma_f16(c, make_uint4(u[2], w[2], u[3], w[3]), b1.x, b1.y);
            s[i][0][0] = j ? fmaf(ks[i], c[0] + c[1], s[i][0][0]) : ks[i] * (c[0] + c[1]);
            s[i + 1][0][0] = j ? fmaf(ks[i + 1], c[2] + c[3], s[i + 1][0][0]) : ks[i + 1] * (c[2] + c[3]);
        }
    }
}

// For more columns: s[i][h][n] for row 8 i + 4 h + t and column g (n = 0), g + 8 (n = 1), in the column's own units. keys(i, j, f): the codes
// of group j of the lane's i-th row, unpacked.
template <int NG, bool LARGE, typename Keys>
__device__ __forceinline__ void score_rows(float (&s)[4][2][LARGE ? 2 : 1], Keys keys, const uint4* qf, const float* sc, int lane) {
#pragma unroll
    for (int j = 0; j < NG; j++) {
        const uint4 a0 = qf[(j * 2) * 32 + lane], a1 = qf[(j * 2 + 1) * 32 + lane];
        uint4 l0 = a0, l1 = a1;
        if (LARGE) { l0 = qf[((NG + j) * 2) * 32 + lane]; l1 = qf[((NG + j) * 2 + 1) * 32 + lane]; }
        float ks[4][2];
        lane_rows(ks, sc + j * 32, lane & 3);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t f[4];
            keys(i, j, f);
            float c[4];
            mma_f16_first(c, a0, f[0], f[1]);
            mma_f16(c, a1, f[2], f[3]);
            if (LARGE) { mma_f16(c, l0, f[0], f[1]); mma_f16(c, l1, f[2], f[3]); }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if constexpr (LARGE) {
                    s[i][h][0] = j ? fmaf(ks[i][h], c[h], s[i][h][0]) : ks[i][h] * c[h];
                    s[i][h][1] = j ? fmaf(ks[i][h], c[2 + h], s[i][h][1]) : ks[i][h] * c[2 + h];
                } else {
                    s[i][h][0] = j ? fmaf(ks[i][h], c[h] + c[2 + h], s[i][h][0]) : ks[i][h] * (c[h] + c[2 + h]);
                }
            }
        }
    }
}

// Results of clusters first, first + step, .. of a column added up at value 4 d4, against the maximum M. at: the column's first. A lane's weights are broadcast
// to the others: nothing in the loop waits for a load but the sums.
__device__ __forceinline__ float4 join_values(const KaParams& p, size_t at, int n, int first, int step, float M, int d4) {
    const int lane = threadIdx.x & 31, mine = (n - first + step - 1) / step;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < mine; s0 += 32) {
        const float w = s0 + lane < mine ? ex2(__ldcg(p.pml + at + (size_t)(first + (s0 + lane) * step) * 16).x - M) : 0.0f;
        const int end = min(32, mine - s0);
#pragma unroll 8
        for (int s = 0; s < end; s++) {
            const float k = __shfl_sync(0xffffffffu, w, s);
            const float4 v = d4 < p.c.hd / 4 ? __ldcg(reinterpret_cast<const float4*>(p.pacc + (at + (size_t)(first + (s0 + s) * step) * 16) * p.c.hd) + d4) : make_float4(0.f, 0.f, 0.f, 0.f);
            o.x = fmaf(v.x, k, o.x); o.y = fmaf(v.y, k, o.y); o.z = fmaf(v.z, k, o.z); o.w = fmaf(v.w, k, o.w);
        }
    }
    return o;
}
// maximum and sum over the clusters, by a warp
__device__ __forceinline__ float2 join_stat(const KaParams& p, size_t at, int n) {
    const int lane = threadIdx.x & 31;
    float2 own = lane < n ? __ldcg(p.pml + at + (size_t)lane * 16) : make_float2(KA_LOW, 0.0f);
    float M = own.x;
    for (int s = lane + 32; s < n; s += 32) M = fmaxf(M, __ldcg(p.pml + at + (size_t)s * 16).x);
    M = warp_max(M);
    float sum = own.y * ex2(own.x - M);
    for (int s = lane + 32; s < n; s += 32) { const float2 v = __ldcg(p.pml + at + (size_t)s * 16); sum = fmaf(v.y, ex2(v.x - M), sum); }
    return make_float2(M, warp_sum(sum));
}
__device__ __forceinline__ void join_store(const KaParams& p, int kvh, int cc, int d4, const float4& o, float inv) {
    float* to = p.out + ((size_t)(cc / p.t.group) * p.t.n_heads + (size_t)kvh * p.t.group + cc % p.t.group) * p.c.hd + 4 * d4;
    to[0] = o.x * inv; to[1] = o.y * inv; to[2] = o.z * inv; to[3] = o.w * inv;
}
// grid (columns of a tile, units), a block a column
__global__ void __launch_bounds__(128) kv4_join_kernel(const KaParams p) {
    __shared__ float4 part[4][64];
    pdl_launch_dependents();
    pdl_wait();
    int row0, pos0, chunk, n;
    if (!kv4_place(p.at, p.t.B, p.c.max_rows, p.err, row0, pos0)) return;
    ka_plan(row0 + p.t.B, p.want, p.cluster, chunk, n);
    n = (n + p.cluster - 1) / p.cluster;
    const int unit = blockIdx.y, kvh = unit / p.t.ntiles, cc = unit % p.t.ntiles * p.t.cols() + blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q4 = p.c.hd / 4;
    if (n == 1 || cc / p.t.group >= p.t.B) return;
    const size_t at = (size_t)unit * (p.grid_chunks / p.cluster) * 16 + blockIdx.x;
    const float2 st = join_stat(p, at, n);
    for (int d0 = 0; d0 < q4; d0 += 32) part[warp][d0 + lane] = join_values(p, at, n, warp, 4, st.x, d0 + lane);
    __syncthreads();
    if (threadIdx.x < q4) {
        float4 o = part[0][threadIdx.x];
        for (int w = 1; w < 4; w++) { const float4 v = part[w][threadIdx.x]; o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w; }
        join_store(p, kvh, cc, threadIdx.x, o, 1.0f / st.y);
    }
    if (threadIdx.x == 0 && p.stat) p.stat[(size_t)unit * 16 + blockIdx.x] = make_float2(st.x, log2f(st.y) - 14.0f);
}

template <int NG, int COLS>
__global__ void __launch_bounds__(32 * KA_WARPS, NG > 4 ? 1 : (COLS == 16 ? 2 : 3)) kv4_attn_kernel(const KaParams p) {
    using S = KaSmem<NG, COLS>;
    using St = KaStage<NG>;
    constexpr bool LARGE = COLS == 16, FOUR = COLS == 4;
    constexpr int NC = LARGE ? 2 : 1, HD = 32 * NG;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ unsigned long long full[KA_WARPS][S::DEPTH];
    __shared__ int abort_flag;
    __shared__ float2 ml[KA_WARPS][16], own[16];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    // tiles that see most rows first
    const int place = blockIdx.x / p.grid_chunks, kvh = place / p.t.ntiles, tile = p.t.ntiles - 1 - place % p.t.ntiles, sp = blockIdx.x % p.grid_chunks;
    const int rank = sp % p.cluster, peers_from = sp - rank;
    const int unit = kvh * p.t.ntiles + tile, c0 = tile * COLS;
    if (tid == 0) {
        abort_flag = 0;
        for (int w = 0; w < KA_WARPS; w++) for (int d = 0; d < S::DEPTH; d++) mbar_init(smem_u32(&full[w][d]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    double2* turn = reinterpret_cast<double2*>(smem + S::TOTAL);
    int row0 = p.at.row0, pos0 = p.at.pos0;
    if (!LARGE) {
        if (p.w.rotate && !p.at.at) kv4_angles(turn, p.t.B, pos0, HD, p.w.log2_theta);             // beside the end of the launch ahead
        pdl_wait();
        pdl_launch_dependents();
    }
    __syncthreads();
    // LARGE: launches ahead of the preparing one have ended when this one starts, since that one lets it start behind its own wait. What they wrote (a
    // device position, rows of earlier calls) may be read before this launch's own wait.
    if (!kv4_place(p.at, p.t.B, p.c.max_rows, p.err, row0, pos0)) return;
    if (!LARGE && p.w.rotate && p.at.at) kv4_angles(turn, p.t.B, pos0, HD, p.w.log2_theta);
    int chunk, n_chunks;
    ka_plan(row0 + p.t.B, p.want, p.cluster, chunk, n_chunks);
    if (peers_from >= n_chunks) return;                                                            // all of the cluster
    const int lim0 = row0 + c0 / p.t.group;                                                // the last row that the tile's first column sees
    const int t0 = sp * chunk, t1 = min(min(t0 + chunk, n_chunks * chunk), row0 + min(p.t.B - 1, (c0 + COLS - 1) / p.t.group) + 1);
    const int stages = t1 > t0 ? (t1 - t0 + KA_ROWS - 1) / KA_ROWS : 0, mine = stages > warp ? (stages - warp + KA_WARPS - 1) / KA_WARPS : 0;     // a warp takes every fourth stage
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
    const int old = p.w.k ? row0 : t1;                                                             // rows below were there before this call
    int issued = 0;
    if (lane == 0)
        for (; issued < min(mine, (int)S::DEPTH) && t0 + (warp + issued * KA_WARPS) * KA_ROWS + KA_ROWS <= old; issued++) issue(issued);
    uint4* qf = reinterpret_cast<uint4*>(smem + S::FRAGS);
    float* qc = reinterpret_cast<float*>(smem + S::QC);
    if constexpr (!LARGE) {
        __shared__ uint32_t amax[KA_WARPS][8];
        __syncthreads();
        if (p.w.k) {                                                                               // the call's rows of this chunk
            const int r0 = max(t0, row0), r1 = min(t1, row0 + p.t.B);
            for (int e = tid; e < (r1 - r0) * 2 * (HD / 8); e += 32 * KA_WARPS) {
                const int f = e / (HD / 8), r = r0 + f / 2, b = r - row0, i = e % (HD / 8) * 8;
                const bool key = f % 2 == 0;
                float x[8];
                kv4_load_eight(x, (key ? p.w.k : p.w.v) + ((size_t)b * p.c.n_kv + kvh) * HD + i);
                kv4_write_eight<NG>(p.c, x, key, kvh, r, i, p.w.rotate ? turn + b * (HD / 2) : nullptr);
            }
            asm volatile("fence.proxy.async.global;" ::: "memory");                                // the bulk copies read them
        }
        constexpr int JT = (NG + KA_WARPS - 1) / KA_WARPS;                                         // a warp has every fourth group of all columns
        const int column = FOUR ? g >> 1 : g, b = column / p.t.group;                              // FOUR: high pieces in even g, low ones in odd
        const bool on = b < p.t.B;
        const float* src = p.w.q + ((size_t)b * p.t.n_heads + (size_t)kvh * p.t.group + column % p.t.group) * HD + 8 * t;
        float x[JT][8];
        uint32_t m = 0;
#pragma unroll
        for (int jj = 0; jj < JT; jj++) {
            const int j = warp + jj * KA_WARPS;
            if (j >= NG) break;
            kv4_query<NG>(x[jj], src + 32 * j, on, p.w.rotate ? turn + b * (HD / 2) : nullptr, 32 * j + 8 * t);
#pragma unroll
            for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(x[jj][i]) & 0x7FFFFFFFu);
        }
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        if (t == 0) amax[warp][column] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < KA_WARPS; w++) m = max(m, amax[w][column]);
        const Kv4Up up = kv4_up(m, HD);
        if (warp == 0 && t == 0) qc[column] = up.back;
#pragma unroll
        for (int jj = 0; jj < JT; jj++) {
            const int j = warp + jj * KA_WARPS;
            if (j >= NG) break;
#pragma unroll
            for (int i = 0; i < 8; i++) x[jj][i] = x[jj][i] * up.a * up.b;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                uint32_t hi[2], lo[2];
                kv4_pieces(x[jj], s, hi, lo);
                if (FOUR) reinterpret_cast<uint2*>(qf)[(j * 2 + s) * 32 + lane] = g & 1 ? make_uint2(lo[0], lo[1]) : make_uint2(hi[0], hi[1]);
                else qf[(j * 2 + s) * 32 + lane] = make_uint4(hi[0], lo[0], hi[1], lo[1]);
            }
        }
    } else {
        pdl_wait();
        pdl_launch_dependents();
        if (lane == 0) asm volatile("fence.proxy.async.global;" ::: "memory");                     // rows that the preparing launch wrote
        const uint4* src = p.w.qf + unit * kv4_frags(NG);
        for (int e = tid; e < NG * 128; e += 32 * KA_WARPS) qf[e] = __ldcg(src + e);
        if (tid < 16) qc[tid] = __ldcg(p.w.qc + (size_t)unit * 16 + tid);
    }
    if (lane == 0) for (; issued < min(mine, (int)S::DEPTH); issued++) issue(issued);
    __syncthreads();
    float* sc = reinterpret_cast<float*>(smem + S::SCALES) + warp * (2 * NG + 1) * 32;
    constexpr int NA = FOUR ? 2 : 4;
    float f[NC], m[NC], l[NC], acc[NG][NA][4];
    int lim[NC];
#pragma unroll
    for (int n = 0; n < NC; n++) {
        const int column = FOUR ? t : g + 8 * n;
        f[n] = qc[column]; m[n] = KA_LOW; l[n] = 0.0f;
        lim[n] = row0 + (c0 + column) / p.t.group;
    }
#pragma unroll
    for (int j = 0; j < NG; j++)
#pragma unroll
        for (int i = 0; i < NA; i++)
#pragma unroll
            for (int u = 0; u < 4; u++) acc[j][i][u] = 0.0f;

    uint32_t phase = 0;
    int d = 0;
    bool wide = false;
    for (int it = 0; it < mine; it++) {
        const int r0 = t0 + (warp + it * KA_WARPS) * KA_ROWS;
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&full[warp][d]), phase, &abort_flag, IBCU_KV4_WAIT_ERR))) break;
        const unsigned char* stage = ring + d * St::BYTES;
        spread_scales<NG, FOUR>(sc, stage + St::SCALES, lane);
        uint32_t kw[4][NG], vw[4][2][(NG + 1) / 2];
#pragma unroll
        for (int i = 0; i < 4; i++) lds_words<NG>(kw[i], stage + St::KEYS + (8 * i + (g >> 1) + 4 * (g & 1)) * 16 * NG + t * 4 * NG);
        __syncwarp();
        float s[4][FOUR ? 1 : 2][NC];
        if constexpr (FOUR) score_rows_four<NG>(s, kw, reinterpret_cast<const uint2*>(qf), sc, lane);
        else score_rows<NG, LARGE>(s, [&](int i, int j, uint32_t* to) { unpack(kw[i][j], to); }, qf, sc, lane);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) lds_units<NG>(vw[i][h], stage + St::VALUES + (8 * i + 4 * h + t) * 16 * NG + g * 2 * NG);
        __syncwarp();
        if (lane == 0 && it + S::DEPTH < mine) issue(it + S::DEPTH);                               // everything of the stage is in registers
        if (++d == S::DEPTH) { d = 0; phase ^= 1; }

        auto weigh = [&](auto masked) {
            constexpr bool MASK = decltype(masked)::value;
            constexpr int NH = FOUR ? 1 : 2;                                                       // rows of a lane in eight
            float L[4][NH], top[NC];
            if constexpr (FOUR) { const float4 x = *reinterpret_cast<const float4*>(sc + 2 * NG * 32 + g * 4); L[0][0] = x.x; L[1][0] = x.y; L[2][0] = x.z; L[3][0] = x.w; }
            else lane_rows(L, sc + 2 * NG * 32, t);
            auto seen = [&](int i, int h, int n) { return !MASK || r0 + 8 * i + (FOUR ? (g >> 1) + 4 * (g & 1) : 4 * h + t) <= lim[n]; };
            constexpr int OVER0 = FOUR ? 4 : 1, OVER1 = FOUR ? 32 : 4;                              // lanes of a column
            bool grow = false;
#pragma unroll
            for (int n = 0; n < NC; n++) {
                top[n] = KA_LOW;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        s[i][h][n] *= f[n];
                        if (p.scores) p.scores[((size_t)unit * p.score_rows + r0 + 8 * i + (FOUR ? (g >> 1) + 4 * (g & 1) : 4 * h + t)) * COLS + (FOUR ? t : g + 8 * n)] = s[i][h][n];
                        if (seen(i, h, n)) top[n] = fmaxf(top[n], s[i][h][n] + L[i][h]);
                    }
                grow = grow || top[n] > m[n] + KA_SLACK;
            }
            if (__any_sync(0xffffffffu, grow)) {
                wide = false;
#pragma unroll
                for (int n = 0; n < NC; n++) {
#pragma unroll
                    for (int o = OVER0; o < OVER1; o *= 2) top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], o));
                    const float now = fmaxf(m[n], top[n]), corr = ex2(m[n] - now);
                    m[n] = now;
                    wide = wide || fabsf(now) > 524288.0f;
                    l[n] *= corr;
#pragma unroll
                    for (int j = 0; j < NG; j++) {
#pragma unroll
                        for (int i = 0; i < NA; i++) {
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
                    for (int h = 0; h < NH; h++) s[i][h][n] -= m[n];
            // Beyond 2^19 (log2 units; such a softmax has one row) the maximum itself is rounded by more than the slack allows for.
            if (__any_sync(0xffffffffu, wide)) {
#pragma unroll
                for (int n = 0; n < NC; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int h = 0; h < NH; h++) s[i][h][n] = s[i][h][n] > 1.0f - L[i][h] ? 1.0f - L[i][h] : s[i][h][n];
            }
#pragma unroll
            for (int n = 0; n < NC; n++) {
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        const float e = seen(i, h, n) ? ex2(s[i][h][n] + 14.0f) : 0.0f;
                        s[i][h][n] = e;
                        l[n] += e;
                    }
            }
            if constexpr (FOUR) {
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    const float4 line = *reinterpret_cast<const float4*>(sc + (NG + j) * 32 + g * 4);
                    const float vs[4] = { line.x, line.y, line.z, line.w };
                    uint32_t b[4];                                                                 // [rows 8 i ..][columns' pieces], transposed
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float a = s[i][0][0] * vs[i];
                        if (!seen(i, 0, 0)) a = 0.0f;                                              // the row's scale may be NaN
                        const float hi = __uint_as_float(__float_as_uint(a) & 0xFFFFE000u);        // eleven bits, cut off: the low piece has the same sign and what is left to 2^-22
                        b[i] = transpose_8x8(pack_half(hi, a - hi));
                    }
                    float part[2][4];                                                              // these rows', added to the sums rounded
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        uint32_t x[4], y[4];
                        unpack(__byte_perm(vw[2 * u][0][j / 2], vw[2 * u][1][j / 2], j & 1 ? 0x7632 : 0x5410), x);
                        unpack(__byte_perm(vw[2 * u + 1][0][j / 2], vw[2 * u + 1][1][j / 2], j & 1 ? 0x7632 : 0x5410), y);
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            if (u) mma_f16(part[q], make_uint4(x[q], x[q + 2], y[q], y[q + 2]), b[2 * u], b[2 * u + 1]);
                            else mma_f16_first(part[q], make_uint4(x[q], x[q + 2], y[q], y[q + 2]), b[2 * u], b[2 * u + 1]);
                        }
                    }
#pragma unroll
                    for (int q = 0; q < 2; q++)
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[j][q][e] += part[q][e];
                }
            } else {
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    float vs[4][2];
                    lane_rows(vs, sc + (NG + j) * 32, t);
                    uint32_t hi[2][2][NC], lo[2][2][NC], b0[2][4], b1[2][4];                       // 16 rows each: pieces 2 u and 2 u + 1
#pragma unroll
                    for (int u = 0; u < 2; u++) {
#pragma unroll
                        for (int i = 0; i < 2; i++)
#pragma unroll
                            for (int n = 0; n < NC; n++) {
                                float a = s[2 * u + i][0][n] * vs[2 * u + i][0], b = s[2 * u + i][1][n] * vs[2 * u + i][1];
                                if (!seen(2 * u + i, 0, n)) a = 0.0f;                              // the row's scale may be NaN
                                if (!seen(2 * u + i, 1, n)) b = 0.0f;
                                hi[u][i][n] = pack_half(a, b);
                                const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi[u][i][n]));
                                lo[u][i][n] = pack_half(a - back.x, b - back.y);
                            }
                        unpack(__byte_perm(vw[2 * u][0][j / 2], vw[2 * u][1][j / 2], j & 1 ? 0x7632 : 0x5410), b0[u]);
                        unpack(__byte_perm(vw[2 * u + 1][0][j / 2], vw[2 * u + 1][1][j / 2], j & 1 ? 0x7632 : 0x5410), b1[u]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float part[4];                                                             // these rows', added to the sums rounded
                        if constexpr (LARGE) {
                            mma_f16_first(part, make_uint4(lo[0][0][0], lo[0][0][1], lo[0][1][0], lo[0][1][1]), b0[0][i], b1[0][i]);
                            mma_f16(part, make_uint4(lo[1][0][0], lo[1][0][1], lo[1][1][0], lo[1][1][1]), b0[1][i], b1[1][i]);
                            mma_f16(part, make_uint4(hi[0][0][0], hi[0][0][1], hi[0][1][0], hi[0][1][1]), b0[0][i], b1[0][i]);
                            mma_f16(part, make_uint4(hi[1][0][0], hi[1][0][1], hi[1][1][0], hi[1][1][1]), b0[1][i], b1[1][i]);
                        } else {
                            mma_f16_first(part, make_uint4(hi[0][0][0], lo[0][0][0], hi[0][1][0], lo[0][1][0]), b0[0][i], b1[0][i]);
                            mma_f16(part, make_uint4(hi[1][0][0], lo[1][0][0], hi[1][1][0], lo[1][1][0]), b0[1][i], b1[1][i]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[j][i][e] += part[e];
                    }
                }
            }
        };
        if (r0 + KA_ROWS - 1 <= lim0) weigh(std::false_type());
        else weigh(std::true_type());
        __syncwarp();                                                                              // the scales may be overwritten
    }

#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
        for (int o = FOUR ? 4 : 1; o < (FOUR ? 32 : 4); o *= 2) l[n] += __shfl_xor_sync(0xffffffffu, l[n], o);
    auto give_up = [&]() {                                     // by one thread of the block, when its waits are over
        if (!*(volatile int*)&abort_flag) return;
        *p.err = IBCU_KV4_WAIT_ERR;
        for (int i = 0; i < 1000; i++) __nanosleep(1000);      // copies still on their way into this block's shared memory land before it goes
    };
    // the four warps' results meet in the rings: [warp][column][value], and maxima and sums
#pragma unroll
    for (int n = 0; n < NC; n++) if (FOUR ? g == 0 : t == 0) ml[warp][FOUR ? t : g + 8 * n] = make_float2(m[n], l[n]);
    __syncthreads();
    float* meet = reinterpret_cast<float*>(smem + S::RING);
#pragma unroll
    for (int j = 0; j < NG; j++) {
        if constexpr (FOUR)                                                                        // values 4g..4g+3 of group j of column t
            *reinterpret_cast<float4*>(meet + ((size_t)warp * COLS + t) * HD + 32 * j + 4 * g) = make_float4(
                acc[j][0][0] + acc[j][0][1], (acc[j][1][0] + acc[j][1][1]) * 0.0625f, acc[j][0][2] + acc[j][0][3], (acc[j][1][2] + acc[j][1][3]) * 0.0625f);
        else {
#pragma unroll
            for (int n = 0; n < NC; n++)
#pragma unroll
                for (int u = 0; u < 2; u++) {                                                      // values 8t+4u..8t+4u+3 of group j of column g + 8 n
                    auto value = [&](int i) { return LARGE ? acc[j][i][2 * n + u] : acc[j][i][u] + acc[j][i][u + 2]; };
                    *reinterpret_cast<float4*>(meet + ((size_t)warp * COLS + g + 8 * n) * HD + 32 * j + 8 * t + 4 * u) = make_float4(value(0), value(1) * 0.0625f, value(2), value(3) * 0.0625f);
                }
        }
    }
    __syncthreads();
    if (tid == 0) give_up();
    auto store = [&](int col, int d4, const float4& o, float M, float sum) {
        const int c = c0 + col;
        if (n_chunks <= p.cluster) {
            join_store(p, kvh, c, d4, o, 1.0f / sum);
            if (d4 == 0 && p.stat) p.stat[(size_t)unit * 16 + col] = make_float2(M, log2f(sum) - 14.0f);
        } else {
            const size_t at = ((size_t)unit * (p.grid_chunks / p.cluster) + sp / p.cluster) * 16 + col;
            *reinterpret_cast<float4*>(p.pacc + at * HD + 4 * d4) = o;
            if (d4 == 0) p.pml[at] = make_float2(M, sum);
        }
    };
    auto add = [](float4& o, float& sum, const float4& v, const float2& of, float M) {
        const float k = ex2(of.x - M);
        sum = fmaf(of.y, k, sum);
        o.x = fmaf(v.x, k, o.x); o.y = fmaf(v.y, k, o.y); o.z = fmaf(v.z, k, o.z); o.w = fmaf(v.w, k, o.w);
    };
    for (int e = tid; e < COLS * HD / 4; e += 32 * KA_WARPS) {
        const int col = e / (HD / 4), d4 = e % (HD / 4);
        if ((c0 + col) / p.t.group >= p.t.B) break;
        float M = ml[0][col].x, sum = 0.0f;
#pragma unroll
        for (int w = 1; w < KA_WARPS; w++) M = fmaxf(M, ml[w][col].x);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < KA_WARPS; w++) add(o, sum, *reinterpret_cast<const float4*>(meet + ((size_t)w * COLS + col) * HD + 4 * d4), ml[w][col], M);
        if (p.cluster == 1) store(col, d4, o, M, sum);
        else {
            *reinterpret_cast<float4*>(meet + (size_t)col * HD + 4 * d4) = o;                      // read by this thread alone until here
            if (d4 == 0) own[col] = make_float2(M, sum);
        }
    }
    if (p.cluster == 1) return;
    // and the blocks of a cluster in one another's shared memory, each with its part of the values
    cluster_arrive(); cluster_wait();
    const int peers = min(p.cluster, n_chunks - peers_from);
    for (int e = rank * 32 * KA_WARPS + tid; e < COLS * HD / 4; e += p.cluster * 32 * KA_WARPS) {
        const int col = e / (HD / 4), d4 = e % (HD / 4);
        if ((c0 + col) / p.t.group >= p.t.B) break;
        float2 of[KA_CLUSTER];
        float4 v[KA_CLUSTER];
#pragma unroll
        for (int r = 0; r < KA_CLUSTER; r++) {
            if (r >= peers) break;
            of[r] = peer_load_f2(smem_u32(&own[col]), r);
            v[r] = peer_load_f4(smem_u32(meet + (size_t)col * HD + 4 * d4), r);
        }
        float M = of[0].x, sum = 0.0f;
#pragma unroll
        for (int r = 1; r < KA_CLUSTER; r++) if (r < peers) M = fmaxf(M, of[r].x);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < KA_CLUSTER; r++) if (r < peers) add(o, sum, v[r], of[r], M);
        store(col, d4, o, M, sum);
    }
    cluster_arrive(); cluster_wait();                          // nobody reads this block's shared memory any more
}

// Attention that the rows draw, of few tiles: from the scores that the attention wrote down, a thread for a row's four columns of every tile, all loads on their way at once. (32
// heads of 128 values over 8, one token after 4000 rows: 8.9 us without weights, 10.8 with them, 16.8 with the kernel below, which computes the scores again.)
template <int COLS>
__global__ void __launch_bounds__(256) kv4_weight_few_kernel(const KaParams p, float decay) {
    constexpr int LANES = COLS / 4, TILES = COLS == 16 ? KA_FEW_TILES : 1;
    pdl_launch_dependents();
    pdl_wait();
    int row0, pos0;
    if (!kv4_place(p.at, p.t.B, p.c.max_rows, p.err, row0, pos0)) return;
    const int c4 = threadIdx.x % LANES * 4, kvh = blockIdx.y, R = row0 + p.t.B;
    for (int r0 = blockIdx.x * (256 / LANES); r0 < R; r0 += gridDim.x * (256 / LANES)) {
        const int r = r0 + threadIdx.x / LANES;
        const bool on = r < R;
        const size_t at = p.c.row(kvh, on ? r : 0);
        float4 x[TILES], off[TILES][2];
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const size_t unit = (size_t)kvh * p.t.ntiles + i;
            if (!on || i >= p.t.ntiles) continue;
            x[i] = __ldcg(reinterpret_cast<const float4*>(p.scores + (unit * p.score_rows + r) * COLS + c4));
            off[i][0] = __ldcg(reinterpret_cast<const float4*>(p.stat + unit * 16 + c4));
            off[i][1] = __ldcg(reinterpret_cast<const float4*>(p.stat + unit * 16 + c4) + 1);
        }
        const float old = !on || decay == 0.0f ? 0.0f : decay * __ldcg(p.c.weight + at);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            if (!on || i >= p.t.ntiles) continue;
            const float v[4] = { x[i].x, x[i].y, x[i].z, x[i].w }, m[4] = { off[i][0].x, off[i][0].z, off[i][1].x, off[i][1].z }, l[4] = { off[i][0].y, off[i][0].w, off[i][1].y, off[i][1].w };
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int b = (i * COLS + c4 + c) / p.t.group;
                if (b < p.t.B && r <= row0 + b) sum += ex2((v[c] - m[c]) - l[c]);
            }
        }
#pragma unroll
        for (int o = 1; o < LANES; o *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (on && c4 == 0) p.c.weight[at] = old + sum;
    }
}

// The same of many tiles. grid (128 rows, KV heads, parts of the tiles): a warp holds the unpacked keys of 32 rows and walks the columns that see them,
// whose fragments come through a ring; the scores are computed again. The parts of a row are added in order.
constexpr int KW_DEPTH = 3;
template <int NG> struct KwSmem {
    static constexpr int FRAG_BYTES = 2 * NG * 1024, QC = FRAG_BYTES, STAT = QC + 64, STAGE = STAT + 128 + 64;
    static constexpr int SCALES = KW_DEPTH * STAGE, TOTAL = SCALES + KA_WARPS * NG * 128;
};
template <int NG>
__global__ void __launch_bounds__(32 * KA_WARPS) kv4_weight_kernel(const KaParams p, float decay, float* __restrict__ parts) {
    using S = KwSmem<NG>;
    constexpr int NC = 2, COLS = 16;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ unsigned long long full[KW_DEPTH];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, kvh = blockIdx.y;
    if (tid == 0) {
        abort_flag = 0;
        for (int d = 0; d < KW_DEPTH; d++) mbar_init(smem_u32(&full[d]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();
    int row0, pos0;
    if (!kv4_place(p.at, p.t.B, p.c.max_rows, p.err, row0, pos0)) return;
    const int R = row0 + p.t.B, r0 = blockIdx.x * 128 + warp * 32;
    if ((int)blockIdx.x * 128 >= R) return;
    const int first = max(0, (int)blockIdx.x * 128 - row0) * p.t.group / COLS + blockIdx.z;       // tiles that see a row of the block, every gridDim.z-th
    const int n = first < p.t.ntiles ? (p.t.ntiles - first + gridDim.z - 1) / gridDim.z : 0;
    auto issue = [&](int i) {
        const int unit = kvh * p.t.ntiles + first + i * gridDim.z, d = i % KW_DEPTH;
        const uint32_t bar = smem_u32(&full[d]), to = smem_u32(smem + d * S::STAGE);
        mbar_expect_tx(bar, S::FRAG_BYTES + 64 + 128);
        bulk_load(to, p.w.qf + unit * kv4_frags(NG), S::FRAG_BYTES, bar);
        bulk_load(to + S::QC, p.w.qc + (size_t)unit * 16, 64, bar);
        bulk_load(to + S::STAT, p.stat + (size_t)unit * 16, 128, bar);
    };
    if (tid == 0) {
        asm volatile("fence.proxy.async.global;" ::: "memory");                                    // the launches ahead wrote them
        for (int i = 0; i < min(n, KW_DEPTH); i++) issue(i);
    }
    float* sc = reinterpret_cast<float*>(smem + S::SCALES) + warp * NG * 32;
    uint32_t kf[4][NG][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = min(r0 + 8 * i + (g >> 1) + 4 * (g & 1), R - 1);
        const uint32_t* src = reinterpret_cast<const uint32_t*>(p.c.k + p.c.row(kvh, r) * (16 * NG)) + t * NG;
#pragma unroll
        for (int j = 0; j < NG; j++) unpack(__ldcg(src + j), kf[i][j]);
    }
    {
        const __half* src = p.c.scale + p.c.row(kvh, min(r0 + lane, R - 1)) * (2 * NG);
        float* d = sc + (lane & 3) * 8 + (lane >> 3) * 2 + ((lane >> 2) & 1);
        for (int j = 0; j < NG; j++) d[j * 32] = __half2float(__ushort_as_half(__ldcg(reinterpret_cast<const unsigned short*>(src) + j)));
    }
    __syncwarp();
    float w[4][2] = {};
    int d = 0;
    uint32_t phase = 0;
    for (int i = 0; i < n; i++) {
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&full[d]), phase, &abort_flag, IBCU_KV4_WAIT_ERR))) { __syncthreads(); continue; }      // the barrier below is everyone's
        const unsigned char* stage = smem + d * S::STAGE;
        float s[4][2][NC];
        score_rows<NG, true>(s, [&](int k, int j, uint32_t* to) {
#pragma unroll
            for (int u = 0; u < 4; u++) to[u] = kf[k][j][u];
        }, reinterpret_cast<const uint4*>(stage), sc, lane);
        const int c0 = (first + i * gridDim.z) * COLS;
#pragma unroll
        for (int k = 0; k < NC; k++) {
            const int b = (c0 + g + 8 * k) / p.t.group, lim = b < p.t.B ? row0 + b : -1;
            const float f = reinterpret_cast<const float*>(stage + S::QC)[g + 8 * k];
            const float2 off = reinterpret_cast<const float2*>(stage + S::STAT)[g + 8 * k];
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int h = 0; h < 2; h++) if (r0 + 8 * q + 4 * h + t <= lim) w[q][h] += ex2((__fmul_rn(s[q][h][k], f) - off.x) - off.y);
        }
        __syncthreads();
        if (tid == 0 && i + KW_DEPTH < n) issue(i + KW_DEPTH);
        if (++d == KW_DEPTH) { d = 0; phase ^= 1; }
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
    if (tid == 0 && *(volatile int*)&abort_flag) {
        *p.err = IBCU_KV4_WAIT_ERR;
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
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

// what a call launches
struct KaCall { int cols, chunks, rows, n_parts; float decay; float* parts; };

template <int NG, int COLS>
int launch_attention(ibcu_ctx* ctx, const KaParams& p, const KaCall& k) {
    static SmemOptIn opt;
    constexpr bool LARGE = COLS == 16;
    const size_t smem = KaSmem<NG, COLS>::TOTAL + (!LARGE && p.w.rotate ? (size_t)p.t.B * 16 * NG * sizeof(double2) : 0);
    if (int rc = ibcu_allow_smem(ctx, opt, kv4_attn_kernel<NG, COLS>, smem)) return rc;
    int rc = ibcu_launch(ctx, kv4_attn_kernel<NG, COLS>, dim3(p.c.n_kv * p.t.ntiles * k.chunks), dim3(32 * KA_WARPS), smem, p.cluster, true, p);
    if (!rc && k.chunks > p.cluster) rc = ibcu_launch(ctx, kv4_join_kernel, dim3(std::min(p.t.cols(), p.t.B * p.t.group), p.c.n_kv * p.t.ntiles), dim3(128), 0, 1, true, p);
    if (rc || !p.stat) return rc;
    if (p.scores) return ibcu_launch(ctx, kv4_weight_few_kernel<COLS>, dim3((unsigned)std::min(((long)k.rows * (COLS / 4) + 255) / 256, (long)std::max(1, 4 * ctx->sm_count / p.c.n_kv)), p.c.n_kv), dim3(256), 0, 1, true, p, k.decay);
    if constexpr (LARGE) {
        static SmemOptIn opt_w;
        if ((rc = ibcu_allow_smem(ctx, opt_w, kv4_weight_kernel<NG>, KwSmem<NG>::TOTAL))) return rc;
        rc = ibcu_launch(ctx, kv4_weight_kernel<NG>, dim3((k.rows + 127) / 128, p.c.n_kv, k.n_parts), dim3(32 * KA_WARPS), KwSmem<NG>::TOTAL, 1, true, p, k.decay, k.n_parts > 1 ? k.parts : (float*)nullptr);
        if (!rc && k.n_parts > 1) rc = ibcu_launch(ctx, kv4_weight_join_kernel, dim3((k.rows + 255) / 256, p.c.n_kv), dim3(256), 0, 1, true, p, k.decay, (const float*)k.parts, k.n_parts);
    }
    return rc;
}
template <int NG>
int launch_attention(ibcu_ctx* ctx, const KaParams& p, const KaCall& k) {
    return k.cols == 16 ? launch_attention<NG, 16>(ctx, p, k) : k.cols == 8 ? launch_attention<NG, 8>(ctx, p, k) : launch_attention<NG, 4>(ctx, p, k);
}

}  // namespace

int kv4_attend(ibcu_ctx* ctx, const Kv4& c, float decay, const Kv4Place& at, const float* q, const float* k, const float* v, float* out, int n_heads, int B, double log2_theta, int rotate) {
    const int group = n_heads / c.n_kv, ng = c.hd / 32;
    const long columns = (long)B * group;
    const int large = columns > 8, ntiles = (int)((columns + (large ? 15 : 7)) / (large ? 16 : 8)), units = c.n_kv * ntiles;
    const int rows = at.at ? c.max_rows : at.row0 + B;
    const Kv4Columns t = { n_heads, group, B, large, ntiles };
    KaCall call;
    memset(&call, 0, sizeof call);
    call.rows = rows; call.decay = decay; call.cols = large ? 16 : columns > 4 ? 8 : 4;
    // A prompt: tcgen05 (kv4_prompt.cu) takes half of the time a row and less once its tiles of 128 columns have enough SMs, the tiles of 16 here fill the machine with fewer.
    // 32 heads over 8 after 8000 rows, us here and there: of 128 values 158 and 204 with 32 tiles of 128, 272 and 204 with 40; of 64 values 132 and 170 with 48, 193 and 168 with 56.
    if ((c.hd == 64 || c.hd == 128) && large && c.n_kv * (columns / 128) >= (c.hd == 64 ? ctx->sm_count * 3 / 8 : ctx->sm_count / 4)) {
        Kv4Columns tp = t;
        tp.ntiles = (int)((columns + 127) / 128) * 8;
        tp.large = 2;
        const size_t tiles = (size_t)c.n_kv * tp.ntiles / 8, b_image = tiles * ng * 16384, b_qc = tiles * 512, b_stat = c.weight ? tiles * 1024 : 0;
        const int n_parts = c.weight ? kv4_prompt_parts(ctx, c, tp.ntiles / 8, rows) : 0;
        if (int rc = ibcu_reserve(ctx, &ctx->scratch, &ctx->scratch_bytes, b_image + b_qc + b_stat + (size_t)n_parts * c.n_kv * c.max_rows * sizeof(float))) return rc;
        char* s = (char*)ctx->scratch;
        float* qc = (float*)(s + b_image); float2* stat = c.weight ? (float2*)(s + b_image + b_qc) : nullptr; float* parts = (float*)(s + b_image + b_qc + b_stat);
        if (int rc = kv4_prepare(ctx, c, tp, at, Kv4Prep{ q, k, v, (uint4*)s, qc, log2_theta, rotate })) return rc;
        if (int rc = kv4_prompt(ctx, c, tp, at, (const unsigned char*)s, qc, out, stat, rows, parts, n_parts)) return rc;
        if (!c.weight) return IBCU_OK;
        KaParams p;
        memset(&p, 0, sizeof p);
        p.c = c; p.t = tp; p.at = at; p.err = ctx->kern_err;
        return ibcu_launch(ctx, kv4_weight_join_kernel, dim3((rows + 255) / 256, c.n_kv), dim3(256), 0, 1, true, p, decay, (const float*)parts, n_parts);
    }
    const int stages = (rows + KA_ROWS - 1) / KA_ROWS;
    // Blocks an SM that chunks are cut for: what fits, but two where a stage is short beside a block's start (one token of 32 heads over 8 of 64 values after 32767
    // rows: 14.8 us, 17.3 with three; of 128 values 21.9 with two, 18.4 with three). One cluster of eight, and so no second launch, for contexts that leave each
    // of its warps four stages at most (after 4000 rows 9.0 against 10.3 us, after 8000 12.4 against 11.9). Beyond, clusters spare the second launch results to read, but find
    // their places only while the machine is not full: of eight where there is an SM for each block (one KV head 12.6 us, 14.3 by four), of four up to four fifths of it (32 heads over 4 after
    // 20000 rows 15.4 us, 17.5 without), of two for many chunks (32 over 8 after 131071 rows 43.5, 44.6 without and by four), none else (32 heads of their own after 32767
    // rows 42.9, 46.6 by two).
    const int fit = (large || ng > 4 ? 2 : 3) * ctx->sm_count;
    int want = std::max(1, (columns <= 4 && ng <= 2 ? 2 * ctx->sm_count : fit) / units), chunk;
    if (stages <= KA_CLUSTER * KA_WARPS * 4) want = std::min(want, KA_CLUSTER);
    if (want > 16) want &= ~1;
    // A place on the device may be anywhere in the cache: clusters of four where there are chunks enough to leave them room, so that a short context in a long cache meets in one (512
    // rows in 32768 8.6 us, 10.2 without; 30000 rows 20.0 and 19.7).
    if (at.at && want > KA_CLUSTER && fit * 4 / 5 / units >= 16) want = std::min(want, fit * 4 / 5 / units / 4 * 4);
    ka_plan(rows, want, KA_CLUSTER, chunk, call.chunks);
    if (at.at) call.chunks = std::min(want, (stages + KA_WARPS - 1) / KA_WARPS);                   // shorter contexts may have more, shorter chunks
    const long blocks = (long)units * call.chunks;
    const int most = call.chunks <= KA_CLUSTER || blocks <= ctx->sm_count ? KA_CLUSTER : blocks * 5 / 4 <= fit ? 4 : call.chunks > 16 ? 2 : 1;
    int cluster = 1;
    while (cluster < std::min(call.chunks, most)) cluster *= 2;
    call.chunks = (call.chunks + cluster - 1) / cluster * cluster;
    const int joined = call.chunks / cluster;
    const int row_blocks = (rows + 127) / 128;
    call.n_parts = c.weight && ntiles >= 16 ? std::min(std::min(ntiles, 16), std::max(1, 6 * ctx->sm_count / (row_blocks * c.n_kv))) : 1;
    auto round_up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    const size_t b_qf = large ? round_up(units * kv4_frags(ng) * sizeof(uint4)) : 0, b_qc = large ? round_up((size_t)units * 16 * sizeof(float)) : 0;
    const size_t b_scores = c.weight && ntiles <= KA_FEW_TILES ? round_up((size_t)units * stages * KA_ROWS * call.cols * sizeof(float)) : 0;
    const size_t b_stat = c.weight ? round_up((size_t)units * 16 * sizeof(float2)) : 0, b_ml = joined > 1 ? round_up((size_t)units * joined * 16 * sizeof(float2)) : 0;
    const size_t b_acc = joined > 1 ? round_up((size_t)units * joined * 16 * c.hd * sizeof(float)) : 0, b_parts = call.n_parts > 1 ? round_up((size_t)call.n_parts * c.n_kv * c.max_rows * sizeof(float)) : 0;
    if (int rc = ibcu_reserve(ctx, &ctx->scratch, &ctx->scratch_bytes, b_qf + b_qc + b_scores + b_stat + b_ml + b_acc + b_parts)) return rc;
    char* s = (char*)ctx->scratch;
    auto take = [&](size_t n) { char* r = s; s += n; return r; };
    KaParams p;
    memset(&p, 0, sizeof p);
    p.c = c; p.t = t; p.at = at;
    uint4* qf = (uint4*)take(b_qf); float* qc = (float*)take(b_qc);
    p.w = Kv4Prep{ q, k, v, qf, qc, log2_theta, rotate };
    p.scores = (float*)take(b_scores); if (!b_scores) p.scores = nullptr;
    p.score_rows = stages * KA_ROWS;
    p.stat = (float2*)take(b_stat); if (!c.weight) p.stat = nullptr;
    p.pml = (float2*)take(b_ml); p.pacc = (float*)take(b_acc);
    call.parts = (float*)take(b_parts);
    p.out = out; p.want = want; p.grid_chunks = call.chunks; p.cluster = cluster; p.err = ctx->kern_err;
    if (large) { if (int rc = kv4_prepare(ctx, c, t, at, p.w)) return rc; }
    switch (ng) {
        case 1: return launch_attention<1>(ctx, p, call);
        case 2: return launch_attention<2>(ctx, p, call);
        case 3: return launch_attention<3>(ctx, p, call);
        case 4: return launch_attention<4>(ctx, p, call);
        case 6: return launch_attention<6>(ctx, p, call);
        default: return launch_attention<8>(ctx, p, call);
    }
}
