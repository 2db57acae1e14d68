// INT8 weights x INT8 activations with one scale per output row and one per token: a prompt's projections as integer products, any
// number of tokens. Sums are exact 32-bit integers, so a result does not depend on how the work is cut.
#include "common.cuh"
#include "tc_common.cuh"
#include "tc_maps.cuh"
#include <algorithm>
#include <type_traits>

namespace {

// one block per token: scale = max|x| * (1 / 127), codes rint(x * (1 / scale)); columns N..ldq-1 of the codes are zero. VEC: rows of whole
// float4s, which the thread keeps between the maximum and the codes (up to QR_KEEP of them; further ones are read twice). Bound by memory: 511 rows of 14336
// took 12 us one value at a time.
constexpr int QR_KEEP = 8;
__device__ __forceinline__ uint32_t size_of(const float4& v) {
    return max(max(__float_as_uint(v.x) & 0x7FFFFFFFu, __float_as_uint(v.y) & 0x7FFFFFFFu), max(__float_as_uint(v.z) & 0x7FFFFFFFu, __float_as_uint(v.w) & 0x7FFFFFFFu));
}
// a token's scale and what turns its values into codes, from the bits of its largest magnitude
__device__ __forceinline__ float token_scale(uint32_t m, float& inv) {
    if (m < 0x0D800000u) { inv = 0.0f; return 0.0f; }         // below 2^-100: zeros
    if (m >= 0x7F800000u) { inv = 0.0f; return __uint_as_float(0x7FFFFFFFu); }           // NaN or Inf: all results of the token are NaN
    const float s = __fmul_rn(__uint_as_float(m), 1.0f / 127.0f);
    inv = __fdiv_rn(1.0f, s);
    return s;
}
// rint(v * inv) in the lowest byte: what is added lifts a value's integer part to the lowest bits, rounded to even
__device__ __forceinline__ uint32_t code_bits(float v, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.0f)); }
__device__ __forceinline__ int8_t code_of(float v, float inv) { return inv > 0.0f ? (int8_t)code_bits(v, inv) : (int8_t)0; }
__device__ __forceinline__ uint32_t codes_of(const float4& v, float inv) {
    const uint32_t lo = __byte_perm(code_bits(v.x, inv), code_bits(v.y, inv), 0x0040), hi = __byte_perm(code_bits(v.z, inv), code_bits(v.w, inv), 0x0040);
    return inv > 0.0f ? __byte_perm(lo, hi, 0x5410) : 0u;
}

// Rows of `n` bytes that begin anywhere, `from` apart, into rows `to` apart (a multiple of 16): TMA wants rows that start on 16 bytes.
struct AlignJob { const uint8_t* src; uint8_t* dst; long from, to, rows; int n; };
__device__ void align_rows(const AlignJob& j, long block, long blocks) {
    const int per = (int)(j.to / 16);
    for (long e = block * blockDim.x + threadIdx.x; e < j.rows * per; e += blocks * blockDim.x) {
        const long r = e / per;
        const int c = (int)(e % per) * 16;
        const uint8_t* a = j.src + r * j.from + c;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (c + 16 < j.n) {                                   // aligned words and a shift; the last word is not past the row's end
            const uint32_t* w = reinterpret_cast<const uint32_t*>((uintptr_t)a & ~(uintptr_t)3);
            const uint32_t sh = (uint32_t)((uintptr_t)a & 3) * 8;
            uint32_t x[5];
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = __ldcg(w + i);
            x[4] = sh ? __ldcg(w + 4) : 0u;
            v = make_uint4(__funnelshift_r(x[0], x[1], sh), __funnelshift_r(x[1], x[2], sh), __funnelshift_r(x[2], x[3], sh), __funnelshift_r(x[3], x[4], sh));
        } else {
            uint8_t b[16];
            for (int i = 0; i < 16; i++) b[i] = c + i < j.n ? __ldcg(a + i) : (uint8_t)0;
            memcpy(&v, b, 16);
        }
        *reinterpret_cast<uint4*>(j.dst + r * j.to + c) = v;
    }
}
// What a call has to copy beside quantising its tokens: blocks behind the tokens' share the jobs.
struct AlignJobs { AlignJob j[5]; int n, blocks; };

// OWN: the codes are this library's scratch, which only the product behind this launch reads, after its own wait. A caller's codes with their scales are an INT8 tensor
// as well as activations, and products read weights ahead of their wait: that launch starts nobody early, which
// costs the two calls of a prompt what they overlapped: with 4096 output rows, one token of 4096 7.1 us (6.4), 64 tokens 12 (10.3), 511 of 14336 35.8 (34.7).
template <bool VEC, bool OWN>
__global__ void __launch_bounds__(512) quantize_rows_kernel(const float* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scale, int N, int ldq, int B, const AlignJobs jobs) {
    __shared__ uint32_t red[16];
    if (OWN) pdl_launch_dependents();
    pdl_wait();
    if ((int)blockIdx.x >= B) {
        for (int i = 0; i < jobs.n; i++) align_rows(jobs.j[i], blockIdx.x - B, jobs.blocks);
        return;
    }
    const size_t b = blockIdx.x;
    const float* xb = x + b * N;
    int8_t* qb = q + b * ldq;
    const int tid = threadIdx.x, nth = blockDim.x, n4 = N / 4;
    const float4* x4 = reinterpret_cast<const float4*>(xb);
    float4 kept[QR_KEEP];
    uint32_t m = 0;
    if (VEC) {
#pragma unroll
        for (int u = 0; u < QR_KEEP; u++) kept[u] = tid + u * nth < n4 ? __ldcg(x4 + tid + u * nth) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < QR_KEEP; u++) m = max(m, size_of(kept[u]));
        for (int i = tid + QR_KEEP * nth; i < n4; i += nth) m = max(m, size_of(__ldcg(x4 + i)));
    } else {
        for (int i = tid; i < N; i += nth) m = max(m, __float_as_uint(__ldcg(xb + i)) & 0x7FFFFFFFu);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((tid & 31) == 0) red[tid >> 5] = m;
    __syncthreads();
    for (int w = 0; w < nth / 32; w++) m = max(m, red[w]);
    float inv;
    const float s = token_scale(m, inv);
    if (VEC) {
        auto put = [&](int i, const float4& v) { reinterpret_cast<uint32_t*>(qb)[i] = codes_of(v, inv); };
#pragma unroll
        for (int u = 0; u < QR_KEEP; u++) if (tid + u * nth < n4) put(tid + u * nth, kept[u]);
        for (int i = tid + QR_KEEP * nth; i < n4; i += nth) put(i, __ldcg(x4 + i));
        for (int i = N + tid; i < ldq; i += nth) qb[i] = 0;
    } else {
        for (int i = tid; i < ldq; i += nth) qb[i] = i < N ? code_of(__ldcg(xb + i), inv) : (int8_t)0;
    }
    if (tid == 0) scale[b] = s;
}

// ── the product on the fifth-generation tensor cores ──
// tcgen05.mma kind::i8: weights are the A operand, 128 output rows, tokens the B operand, up to 256; a lane of tensor memory is an output row,
// so that a warp's store of one token's results is 128 bytes in a row. Per block of 128 columns TMA brings both operands; 32-bit
// accumulators are two buffers of tensor memory, one being read out while the other is filled. Blocks walk the tiles, the tiles of
// tokens of the same rows next to one another, so that weights are read from memory once. Eight warps write results out: with four, two tensors of
// 14336 x 4096 at 2048 tokens took 263 us, 174 of them without the stores.
// Few tiles are cut along the columns, over a cluster of S blocks: block r takes the r-th part, and the sums of the r-th TL tokens meet in
// its shared memory. They are whole numbers: S changes nothing in the result.
constexpr int W8_MAX_STAGES = 12, W8_OUT_WARPS = 8, W8_TMA_WARP = W8_OUT_WARPS, W8_MMA_WARP = W8_OUT_WARPS + 1, W8_THREADS = (W8_OUT_WARPS + 2) * 32;

struct alignas(64) W8Maps { CUtensorMap w[4], x; };
struct W8Params {
    ibcu_linear_t t[4];
    int n_tensors, tile_start[5];                    // tiles of 128 rows of tensor i: [tile_start[i], tile_start[i + 1])
    int B, NT, token_tiles, nkb, S, stages, tmem_cols, early_weights;   // NT: tokens a tile; nkb: blocks of 128 columns; early_weights: no launch of this call writes them
    int edge;                                        // 131072 columns: see w8_sum
    const float* sx;
    int* err;
};
struct W8Shared {
    unsigned long long full[W8_MAX_STAGES], empty[W8_MAX_STAGES], acc_full[2], acc_empty[2], drained;
    uint32_t tmem_base;
    int abort_flag;
    float sx[2][256];
};

// A sum as a float. 131072 products of -128 and -128 are 2^31, which wraps to -2^31; that no other codes come to (the lowest is -128 * 127 * 131072).
__device__ __forceinline__ float w8_unwrap(float sum) { return sum == -2147483648.0f ? 2147483648.0f : sum; }
__device__ __forceinline__ float w8_sum(uint32_t sum, bool edge) { const float f = (float)(int)sum; return edge ? w8_unwrap(f) : f; }

// A tile's results from tensor memory, by eight warps: this thread's output row, 32 tokens at a time or the last 16. Each warp's store of a token is 128 bytes.
__device__ __forceinline__ void write_tile(const ibcu_linear_t& W, uint32_t tmem, int row, int tok0, int tokens, int NT, float sw, const float* sx, bool edge) {
    const int warp = threadIdx.x >> 5;
    const bool have = row < W.M;
    const size_t ld = (size_t)W.out_stride;
    const uint32_t from = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    for (int c = (warp >> 2) * 32; c < NT; c += W8_OUT_WARPS * 8) {          // 32 tokens at a time, or the last 16
        uint32_t acc[32];
        if (NT - c >= 32) { tmem_ld32(from + c, acc); tmem_wait_ld(acc); }
        else tmem_ld16(from + c, acc);
        float sum[32];
#pragma unroll
        for (int u = 0; u < 32; u++) sum[u] = (float)(int)acc[u];
        if (edge) {
#pragma unroll
            for (int u = 0; u < 32; u++) sum[u] = w8_unwrap(sum[u]);
        }
        const int n = have ? min(32, tokens - c) : 0;
        float* o = W.out + (size_t)(tok0 + c) * ld + row;
        auto finish = [&](auto whole, auto add) {
#pragma unroll
            for (int u0 = 0; u0 < 32; u0 += 8) {
                float old[8];
#pragma unroll
                for (int u = 0; u < 8; u++) old[u] = decltype(add)::value && (decltype(whole)::value || u0 + u < n) ? __ldcg(o + (size_t)u * ld) : 0.0f;
                const float4 s0 = *reinterpret_cast<const float4*>(sx + c + u0), s1 = *reinterpret_cast<const float4*>(sx + c + u0 + 4);
                const float f[8] = { s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w };
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const float y = sum[u0 + u] * (sw * f[u]);
                    if (decltype(whole)::value || u0 + u < n) o[(size_t)u * ld] = decltype(add)::value ? old[u] + y : y;
                }
                o += 8 * ld;
                if (!decltype(whole)::value && u0 + 8 >= n) break;
            }
        };
        if (W.epilogue == IBCU_EPI_ADD) { if (n == 32) finish(std::true_type(), std::true_type()); else if (n > 0) finish(std::false_type(), std::true_type()); }
        else if (n == 32) finish(std::true_type(), std::false_type());
        else if (n > 0) finish(std::false_type(), std::false_type());
        __syncwarp();
    }
}

// tokens of a tile whose sums meet in one block of S, in fours
__host__ __device__ __forceinline__ int w8_share(int NT, int S) { return (NT / 4 + S - 1) / S * 4; }

__global__ void __launch_bounds__(W8_THREADS, 1) w8a8_tc_kernel(const __grid_constant__ W8Maps maps, const W8Params p) {
    extern __shared__ __align__(1024) unsigned char w8_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int S = p.S, rank = (int)blockIdx.x % S, first = (int)blockIdx.x / S, step = (int)gridDim.x / S;
    const int tiles = p.tile_start[p.n_tensors] * p.token_tiles;
    const int k0 = (int)((long)p.nkb * rank / S), nk = (int)((long)p.nkb * (rank + 1) / S) - k0;
    const int stage_bytes = 16384 + p.NT * 128;
    W8Shared* sh = reinterpret_cast<W8Shared*>(w8_smem + (size_t)p.stages * stage_bytes);
    volatile int* abort_flag = &sh->abort_flag;
    if (tid == 0) {
        for (int s = 0; s < W8_MAX_STAGES; s++) { mbar_init(smem_u32(&sh->full[s]), 1); mbar_init(smem_u32(&sh->empty[s]), 1); }
        for (int s = 0; s < 2; s++) { mbar_init(smem_u32(&sh->acc_full[s]), 1); mbar_init(smem_u32(&sh->acc_empty[s]), W8_OUT_WARPS); }
        mbar_init(smem_u32(&sh->drained), 1);
        sh->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    auto place = [&](int tile, int& ti, int& row0, int& tok0) {
        const int rt = tile / p.token_tiles;
        tok0 = tile % p.token_tiles * p.NT;
        ti = 0;
#pragma unroll
        for (int i = 1; i < 4; i++) if (i < p.n_tensors && rt >= p.tile_start[i]) ti = i;
        row0 = (rt - p.tile_start[ti]) * 128;
    };

    // Blocks at work at the same time start at different blocks of columns: those that share rows or tokens would otherwise read the same
    // lines at the same moment and queue for them. (Integer sums: the order is free.)
    auto turn_of = [&](int tile) { return (tile / p.token_tiles + tile % p.token_tiles * 4) % nk; };
    auto column = [&](int turn, int i) { const int k = i + turn; return (k0 + (k < nk ? k : k - nk)) * 128; };

    if (warp == W8_MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&sh->tmem_base)), "r"((uint32_t)p.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        pdl_launch_dependents();                     // not before this block holds its tensor memory: see linear_tc.cu
    }
    if (warp == W8_TMA_WARP) {
        // the first stages' weights are on their way before the tokens' codes are there
        const bool one = elect_one();
        int ti, row0, tok0;
        const int ahead = p.early_weights && first < tiles ? min(p.stages, nk) : 0;
        if (one && ahead) {
            place(first, ti, row0, tok0);
            const int turn = turn_of(first);
            for (int s = 0; s < ahead; s++) {
                mbar_expect_tx(smem_u32(&sh->full[s]), (uint32_t)stage_bytes);
                tma_load_2d(smem_u32(w8_smem + (size_t)s * stage_bytes), &maps.w[ti], column(turn, s), row0, smem_u32(&sh->full[s]));
            }
        }
        __syncwarp();
        pdl_wait();
        if (one) {
            asm volatile("fence.proxy.async.global;" ::: "memory");
            int s = 0; uint32_t ph = 1;
            bool ok = true;
            long n = 0;
            for (int tile = first; tile < tiles && ok; tile += step) {
                place(tile, ti, row0, tok0);
                const int turn = turn_of(tile);
                for (int i = 0; i < nk; i++, n++) {
                    const uint32_t at = smem_u32(w8_smem + (size_t)s * stage_bytes), bar = smem_u32(&sh->full[s]);
                    if (n >= ahead) {
                        ok = mbar_wait(smem_u32(&sh->empty[s]), ph, abort_flag, 1);
                        if (!ok) break;
                        mbar_expect_tx(bar, (uint32_t)stage_bytes);
                        tma_load_2d(at, &maps.w[ti], column(turn, i), row0, bar);
                    }
                    tma_load_2d(at + 16384, &maps.x, column(turn, i), tok0, bar);
                    if (++s == p.stages) { s = 0; ph ^= 1; }
                }
            }
        }
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (warp != W8_TMA_WARP) asm volatile("bar.sync 1, %0;" :: "n"(W8_THREADS - 32) : "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = warp == W8_TMA_WARP ? 0u : sh->tmem_base;

    if (warp == W8_MMA_WARP) {
        pdl_wait();
        if (elect_one()) {
            // s32 accumulators, both operands signed bytes, 128 rows
            const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.NT >> 3) << 17) | (8u << 24);
            int s = 0, j = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int tile = first; tile < tiles && ok; tile += step, j++) {
                ok = mbar_wait(smem_u32(&sh->acc_empty[j & 1]), (uint32_t)((j >> 1) & 1) ^ 1u, abort_flag, 2);
                const uint32_t d = tmem + (uint32_t)((j & 1) * p.NT);
                for (int i = 0; i < nk && ok; i++) {
                    ok = mbar_wait(smem_u32(&sh->full[s]), ph, abort_flag, 3);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = smem_u32(w8_smem + (size_t)s * stage_bytes);
                    const uint64_t ad = smem_desc_sw128(at), bd = smem_desc_sw128(at + 16384);
#pragma unroll
                    for (int m = 0; m < 4; m++) mma_i8_ss(d, ad + m * 2, bd + m * 2, idesc, (i | m) ? 1u : 0u);
                    mma_commit(smem_u32(&sh->empty[s]));
                    if (++s == p.stages) { s = 0; ph ^= 1; }
                }
                if (ok) mma_commit(smem_u32(&sh->acc_full[j & 1]));
            }
            mma_commit(smem_u32(&sh->drained));
            mbar_wait(smem_u32(&sh->drained), 0u, abort_flag, 4);              // nothing of this block is left in the tensor pipe
        }
        __syncwarp();
    } else if (warp < W8_OUT_WARPS) {
        pdl_wait();
        int j = 0;
        for (int tile = first; tile < tiles; tile += step, j++) {
            int ti, row0, tok0;
            place(tile, ti, row0, tok0);
            const ibcu_linear_t& W = p.t[ti];
            const int row = row0 + (tid & 127), tokens = min(p.NT, p.B - tok0);
            const bool have = row < W.M;
            const float sw = !have ? 0.0f : W.scales_fp32 ? reinterpret_cast<const float*>(W.scales)[row] : __half2float(reinterpret_cast<const __half*>(W.scales)[row]);
            float* sx = sh->sx[j & 1];
            if (tid < p.NT) sx[tid] = tid < tokens ? __ldcg(p.sx + tok0 + tid) : 0.0f;
            asm volatile("bar.sync 2, %0;" :: "n"(W8_OUT_WARPS * 32) : "memory");
            const bool there = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->acc_full[j & 1]), (uint32_t)((j >> 1) & 1), abort_flag, 5));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (S > 1) break;                        // one tile a cluster; its parts meet below
            if (!there) continue;                    // gave up: the barrier above is still everyone's
            write_tile(W, tmem + (uint32_t)((j & 1) * p.NT), row, tok0, tokens, p.NT, sw, sx, p.edge);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh->acc_empty[j & 1]));
        }
    }
    if (S > 1) {
        __syncwarp();
        cluster_arrive(); cluster_wait();            // every block of the cluster has done its products: the rings are free
        const int TL = w8_share(p.NT, S);            // tokens a block
        const uint32_t meet = smem_u32(w8_smem);     // [source block][4 tokens][row][token]
        const int r = tid & 127;
        if (warp < W8_OUT_WARPS && !*abort_flag) {
            const uint32_t from = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            for (int c = (warp >> 2) * 16; c < p.NT; c += W8_OUT_WARPS * 4) {
                uint32_t acc[16];
                tmem_ld16(from + c, acc);
#pragma unroll
                for (int u = 0; u < 16; u += 4)
                    peer_store_u32x4(meet + (uint32_t)((((rank * TL + (c + u) % TL) / 4) * 128 + r) * 16), (uint32_t)((c + u) / TL), acc + u);
            }
        }
        __syncwarp();
        cluster_arrive(); cluster_wait();
        if (warp < W8_OUT_WARPS && !*abort_flag) {
            int ti, row0, tok0;
            place(first, ti, row0, tok0);
            const ibcu_linear_t& W = p.t[ti];
            const int row = row0 + r, mine = min(TL, min(p.NT, p.B - tok0) - rank * TL);
            const uint4* got = reinterpret_cast<const uint4*>(w8_smem);
            if (row < W.M) {
                const float sw = W.scales_fp32 ? reinterpret_cast<const float*>(W.scales)[row] : __half2float(reinterpret_cast<const __half*>(W.scales)[row]);
                for (int t = (tid >> 7) * 4; t < mine; t += 8) {
                    uint4 sum = got[(t / 4) * 128 + r];
                    for (int k = 1; k < S; k++) { const uint4 v = got[((k * TL + t) / 4) * 128 + r]; sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w; }
                    const uint32_t four[4] = { sum.x, sum.y, sum.z, sum.w };
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        if (t + u < mine) {
                            float* to = W.out + (size_t)(tok0 + rank * TL + t + u) * W.out_stride + row;
                            const float y = w8_sum(four[u], p.edge) * (sw * sh->sx[0][rank * TL + t + u]);
                            *to = W.epilogue == IBCU_EPI_ADD ? __ldcg(to) + y : y;
                        }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == W8_MMA_WARP) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"((uint32_t)p.tmem_cols) : "memory");
    }
    if (tid == 0 && sh->abort_flag) {
        *p.err = 420 + sh->abort_flag;
        for (int i = 0; i < 1000; i++) __nanosleep(1000);      // copies still on their way into this block's shared memory land before it goes
    }
}

// The same product by pairs of blocks (cta_group::2): 256 output rows by up to 256 tokens, each block with 128 of the rows and half of the tokens' codes in its
// shared memory, results of its rows in its tensor memory. A block of columns is 32 KB a block instead of 48 for as many products, which the copies keep
// ahead of (48 took 707 cycles of the copies for 524 of products). The first block issues the products; both blocks' copies report to its
// barriers, and its commits to both.
__global__ void __launch_bounds__(W8_THREADS, 1) w8a8_pair_kernel(const __grid_constant__ W8Maps maps, const W8Params p) {
    extern __shared__ __align__(1024) unsigned char w8_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = blockIdx.x & 1, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const int tiles = p.tile_start[p.n_tensors] * p.token_tiles, nk = p.nkb, half = p.NT / 2;
    const int stage_bytes = 16384 + half * 128;
    W8Shared* sh = reinterpret_cast<W8Shared*>(w8_smem + (size_t)p.stages * stage_bytes);
    volatile int* abort_flag = &sh->abort_flag;
    if (tid == 0) {
        for (int s = 0; s < W8_MAX_STAGES; s++) { mbar_init(smem_u32(&sh->full[s]), 1); mbar_init(smem_u32(&sh->empty[s]), 1); }
        for (int s = 0; s < 2; s++) { mbar_init(smem_u32(&sh->acc_full[s]), 1); mbar_init(smem_u32(&sh->acc_empty[s]), 2 * W8_OUT_WARPS); }
        mbar_init(smem_u32(&sh->drained), 1);
        sh->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    cluster_arrive(); cluster_wait();                // the other block runs and its barriers are there
    auto place = [&](int tile, int& ti, int& row0, int& tok0) {
        const int rt = tile / p.token_tiles;
        tok0 = tile % p.token_tiles * p.NT;
        ti = 0;
#pragma unroll
        for (int i = 1; i < 4; i++) if (i < p.n_tensors && rt >= p.tile_start[i]) ti = i;
        row0 = (rt - p.tile_start[ti]) * 256 + rank * 128;
    };
    auto turn_of = [&](int tile) { return (tile / p.token_tiles + tile % p.token_tiles * 4) % nk; };          // see w8a8_tc_kernel
    auto column = [&](int turn, int i) { const int k = i + turn; return (k < nk ? k : k - nk) * 128; };
    if (warp == W8_MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&sh->tmem_base)), "r"((uint32_t)p.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        pdl_launch_dependents();                     // not before this block holds its tensor memory: see linear_tc.cu
    }
    if (warp == W8_TMA_WARP) {
        const bool one = elect_one();
        int ti, row0, tok0;
        const int ahead = p.early_weights && first < tiles ? min(p.stages, nk) : 0;
        if (one && ahead) {
            place(first, ti, row0, tok0);
            const int turn = turn_of(first);
            for (int s = 0; s < ahead; s++) {
                if (rank == 0) mbar_expect_tx(smem_u32(&sh->full[s]), 2u * (uint32_t)stage_bytes);
                tma_load_2d_pair(smem_u32(w8_smem + (size_t)s * stage_bytes), &maps.w[ti], column(turn, s), row0, peer_address(smem_u32(&sh->full[s]), 0));
            }
        }
        __syncwarp();
        pdl_wait();
        if (one) {
            asm volatile("fence.proxy.async.global;" ::: "memory");
            int s = 0; uint32_t ph = 1;
            bool ok = true;
            long n = 0;
            for (int tile = first; tile < tiles && ok; tile += step) {
                place(tile, ti, row0, tok0);
                const int turn = turn_of(tile);
                for (int i = 0; i < nk; i++, n++) {
                    const uint32_t at = smem_u32(w8_smem + (size_t)s * stage_bytes), bar = peer_address(smem_u32(&sh->full[s]), 0);
                    if (n >= ahead) {
                        ok = mbar_wait(smem_u32(&sh->empty[s]), ph, abort_flag, 1);
                        if (!ok) break;
                        if (rank == 0) mbar_expect_tx(smem_u32(&sh->full[s]), 2u * (uint32_t)stage_bytes);
                        tma_load_2d_pair(at, &maps.w[ti], column(turn, i), row0, bar);
                    }
                    tma_load_2d_pair(at + 16384, &maps.x, column(turn, i), tok0 + rank * half, bar);
                    if (++s == p.stages) { s = 0; ph ^= 1; }
                }
            }
        }
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (warp != W8_TMA_WARP) asm volatile("bar.sync 1, %0;" :: "n"(W8_THREADS - 32) : "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = warp == W8_TMA_WARP ? 0u : sh->tmem_base;
    if (warp == W8_MMA_WARP) {
        pdl_wait();
        if (rank == 0 && elect_one()) {
            // s32 accumulators, both operands signed bytes, 256 rows
            const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.NT >> 3) << 17) | (16u << 24);
            int s = 0, j = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int tile = first; tile < tiles && ok; tile += step, j++) {
                ok = mbar_wait(smem_u32(&sh->acc_empty[j & 1]), (uint32_t)((j >> 1) & 1) ^ 1u, abort_flag, 2);
                const uint32_t d = tmem + (uint32_t)((j & 1) * p.NT);
                for (int i = 0; i < nk && ok; i++) {
                    ok = mbar_wait(smem_u32(&sh->full[s]), ph, abort_flag, 3);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = smem_u32(w8_smem + (size_t)s * stage_bytes);
                    const uint64_t ad = smem_desc_sw128(at), bd = smem_desc_sw128(at + 16384);
#pragma unroll
                    for (int m = 0; m < 4; m++) mma_i8_pair(d, ad + m * 2, bd + m * 2, idesc, (i | m) ? 1u : 0u);
                    mma_commit_pair(smem_u32(&sh->empty[s]));
                    if (++s == p.stages) { s = 0; ph ^= 1; }
                }
                if (ok) mma_commit_pair(smem_u32(&sh->acc_full[j & 1]));
            }
            mma_commit_pair(smem_u32(&sh->drained));
            mbar_wait(smem_u32(&sh->drained), 0u, abort_flag, 4);              // nothing is left in the tensor pipe
        }
        __syncwarp();
    } else if (warp < W8_OUT_WARPS) {
        pdl_wait();
        int j = 0;
        for (int tile = first; tile < tiles; tile += step, j++) {
            int ti, row0, tok0;
            place(tile, ti, row0, tok0);
            const ibcu_linear_t& W = p.t[ti];
            const int row = row0 + (tid & 127), tokens = min(p.NT, p.B - tok0);
            const float sw = row >= W.M ? 0.0f : W.scales_fp32 ? reinterpret_cast<const float*>(W.scales)[row] : __half2float(reinterpret_cast<const __half*>(W.scales)[row]);
            float* sx = sh->sx[j & 1];
            if (tid < p.NT) sx[tid] = tid < tokens ? __ldcg(p.sx + tok0 + tid) : 0.0f;
            asm volatile("bar.sync 2, %0;" :: "n"(W8_OUT_WARPS * 32) : "memory");
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sh->acc_full[j & 1]), (uint32_t)((j >> 1) & 1), abort_flag, 5))) continue;          // gave up: the barrier above is still everyone's
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            write_tile(W, tmem + (uint32_t)((j & 1) * p.NT), row, tok0, tokens, p.NT, sw, sx, p.edge);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_peer(peer_address(smem_u32(&sh->acc_empty[j & 1]), 0));
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (tid == 0 && sh->abort_flag) {
        *p.err = 440 + sh->abort_flag;
        for (int i = 0; i < 1000; i++) __nanosleep(1000);      // copies still on their way into this block's shared memory land before it goes
    }
    __syncthreads();
    cluster_arrive(); cluster_wait();                // neither block's barriers or tensor memory are needed any more
    if (warp == W8_MMA_WARP) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"((uint32_t)p.tmem_cols) : "memory");
    }
}

// ── few tokens ──
// Up to four tokens are bound by the weights' bytes and, for one matrix, by latency: one launch, a warp a row, whose bytes are all on
// their way before the launch ahead has ended; meanwhile every block quantises the tokens for itself (or copies their codes), then four products a dp4a. 4096 x 4096
// at one token, replayed: 5.2 us from FP32 and 4.4 from codes, of which the weights' 16 MB are 2.6.
constexpr int WF_WARPS = 8, WF_AHEAD = 8, WF_TOKENS = 4;
struct WfParams { ibcu_linear_t t[4]; int n, row_start[5], N, B; const float* x; const int8_t* xq; const float* sx; };

template <int B>
__global__ void __launch_bounds__(WF_WARPS * 32) w8a8_few_kernel(const WfParams p) {
    extern __shared__ __align__(16) int8_t codes[];           // [B][N]
    __shared__ uint32_t red[WF_WARPS];
    __shared__ float scale[B];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n16 = p.N / 16, rows = p.row_start[p.n], step = gridDim.x * WF_WARPS;
    auto tensor_of = [&](int row) { int ti = 0; for (int i = 1; i < p.n; i++) if (row >= p.row_start[i]) ti = i; return ti; };
    int row = blockIdx.x * WF_WARPS + warp;
    uint4 w[WF_AHEAD];
    auto fetch = [&](int first) {                             // WF_AHEAD pieces of the row a lane
        const int ti = tensor_of(row);
        const uint4* src = reinterpret_cast<const uint4*>((const int8_t*)p.t[ti].w + (size_t)(row - p.row_start[ti]) * p.N);
#pragma unroll
        for (int u = 0; u < WF_AHEAD; u++) {
            const int i = first + lane + 32 * u;
            w[u] = i < n16 ? ld_stream_u4(src + i) : make_uint4(0, 0, 0, 0);
        }
    };
    if (row < rows) fetch(0);
    pdl_launch_dependents();
    pdl_wait();
    if (p.x) {
        const int n4 = p.N / 4;
        for (int b = 0; b < B; b++) {
            const float4* x4 = reinterpret_cast<const float4*>(p.x + (size_t)b * p.N);
            float4 kept[4];
            uint32_t m = 0;
#pragma unroll
            for (int u = 0; u < 4; u++) kept[u] = tid + u * 256 < n4 ? __ldcg(x4 + tid + u * 256) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < 4; u++) m = max(m, size_of(kept[u]));
            for (int i = tid + 1024; i < n4; i += 256) m = max(m, size_of(__ldcg(x4 + i)));
            m = __reduce_max_sync(0xffffffffu, m);
            if (lane == 0) red[warp] = m;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WF_WARPS; i++) m = max(m, red[i]);
            float inv;
            const float s = token_scale(m, inv);
            uint32_t* to = reinterpret_cast<uint32_t*>(codes + (size_t)b * p.N);
#pragma unroll
            for (int u = 0; u < 4; u++) if (tid + u * 256 < n4) to[tid + u * 256] = codes_of(kept[u], inv);
            for (int i = tid + 1024; i < n4; i += 256) to[i] = codes_of(__ldcg(x4 + i), inv);
            if (tid == 0) scale[b] = s;
            __syncthreads();
        }
    } else {
        for (int i = tid; i < B * n16; i += 256) reinterpret_cast<uint4*>(codes)[i] = __ldcg(reinterpret_cast<const uint4*>(p.xq) + i);
        if (tid < B) scale[tid] = __ldcg(p.sx + tid);
        __syncthreads();
    }
    for (; row < rows; row += step) {
        int sum[B] = {};
        for (int first = 0; first < n16; first += 32 * WF_AHEAD) {
            if (first || row != (int)(blockIdx.x * WF_WARPS + warp)) fetch(first);
#pragma unroll
            for (int u = 0; u < WF_AHEAD; u++) {
                const int i = first + lane + 32 * u;
                if (i >= n16) break;
#pragma unroll
                for (int b = 0; b < B; b++) {
                    const uint4 x = *reinterpret_cast<const uint4*>(codes + (size_t)b * p.N + 16 * i);
                    sum[b] = __dp4a((int)w[u].x, (int)x.x, sum[b]); sum[b] = __dp4a((int)w[u].y, (int)x.y, sum[b]);
                    sum[b] = __dp4a((int)w[u].z, (int)x.z, sum[b]); sum[b] = __dp4a((int)w[u].w, (int)x.w, sum[b]);
                }
            }
        }
        const ibcu_linear_t& t = p.t[tensor_of(row)];
        const int r = row - p.row_start[tensor_of(row)];
        int mine = 0;
#pragma unroll
        for (int b = 0; b < B; b++) { const int v = __reduce_add_sync(0xffffffffu, sum[b]); if (lane == b) mine = v; }
        if (lane < B) {
            const float sw = t.scales_fp32 ? reinterpret_cast<const float*>(t.scales)[r] : __half2float(reinterpret_cast<const __half*>(t.scales)[r]);
            float* o = t.out + (size_t)lane * t.out_stride + r;
            const float y = (float)mine * (sw * scale[lane]);
            *o = t.epilogue == IBCU_EPI_ADD ? __ldcg(o) + y : y;
        }
    }
}

int check_call(ibcu_ctx* ctx, const ibcu_linear_t* ts, int n, int N, int B, const char* call) {
    IBCU_REQUIRE(ctx, ts && n >= 1 && n <= 4, "%s: %d tensors (1 to 4)", call, n);
    IBCU_REQUIRE(ctx, N >= 1 && N <= 131072 && B >= 1 && B <= (1 << 20), "%s: N=%d (up to 131072) B=%d (up to %d)", call, N, B, 1 << 20);
    for (int i = 0; i < n; i++) {
        IBCU_REQUIRE(ctx, ts[i].w && ts[i].scales && ts[i].out, "%s: null pointer", call);
        IBCU_REQUIRE(ctx, ts[i].M >= 1 && ts[i].M <= 0x7FFFFF00 && ts[i].out_stride >= ts[i].M, "%s: M=%d (up to 2^31 - 256) out_stride=%d", call, ts[i].M, ts[i].out_stride);
        IBCU_REQUIRE(ctx, ts[i].epilogue == IBCU_EPI_STORE || ts[i].epilogue == IBCU_EPI_ADD, "%s: epilogue=%d", call, ts[i].epilogue);
    }
    return IBCU_OK;
}

template <bool OWN>
int quantize(ibcu_ctx* ctx, const float* x, int8_t* q, float* scale, int N, int ldq, int B, const AlignJobs& jobs) {
    const bool vec = N % 4 == 0 && ldq % 4 == 0 && ((uintptr_t)x & 15) == 0 && ((uintptr_t)q & 3) == 0;
    return ibcu_launch(ctx, vec ? quantize_rows_kernel<true, OWN> : quantize_rows_kernel<false, OWN>, dim3(B + (jobs.n ? jobs.blocks : 0)), dim3(N > 8192 || (B < ctx->sm_count && N >= 2048) ? 512 : 256), 0, 1, true,
                       x, q, scale, N, ldq, B, jobs);
}

// Few tokens: IBCU_DECLINED where the call is not one for that kernel. x: FP32 tokens, or their codes and scales. A token costs it the reading of its codes
// for every row and, from FP32, its quantisation by every block, the tensor cores a launch more and a longer start. us there and here, replayed: 4096 x 4096
// one token 7.2 and 5.2, two 7.3 and 7.0, three 7.5 and 8.9; 4096 x 8192 one 8.8 and 9.1; 2048 x 2048 four 6.8 and 5.6; with codes 4096 x 4096 four 6.3 and 6.1,
// 4096 x 8192 two 7.7 and 6.8, three 7.6 and 8.5. Beyond two rows a warp its loads no longer run ahead: 12000 x 512 one token 4.6 and 5.6.
int product_few(ibcu_ctx* ctx, const ibcu_linear_t* ts, int n, const float* x, const int8_t* xq, const float* sx, int N, int B) {
    double rows = 0.0;
    for (int i = 0; i < n; i++) rows += ts[i].M;
    if (B > WF_TOKENS || N % 16 || (long)B * N > 65536 || ((uintptr_t)(x ? (const void*)x : xq) & 15) || rows > 2.0 * WF_WARPS * 4 * ctx->sm_count ||
        (double)B * N * (x ? rows + 3300.0 : rows) > (x ? 55e6 : 75e6)) return IBCU_DECLINED;
    WfParams p;
    memset(&p, 0, sizeof p);
    for (int i = 0; i < n; i++) {
        if ((uintptr_t)ts[i].w & 15) return IBCU_DECLINED;
        p.t[i] = ts[i];
        p.row_start[i + 1] = p.row_start[i] + ts[i].M;
    }
    p.n = n; p.N = N; p.B = B; p.x = x; p.xq = xq; p.sx = sx;
    auto kern = B == 1 ? w8a8_few_kernel<1> : B == 2 ? w8a8_few_kernel<2> : B == 3 ? w8a8_few_kernel<3> : w8a8_few_kernel<4>;
    static SmemOptIn opt[WF_TOKENS];
    const size_t smem = (size_t)B * N;
    if (int rc = ibcu_allow_smem(ctx, opt[B - 1], kern, smem)) return rc;
    const int fit = std::max(1, std::min(4, (int)(220 * 1024 / (smem + 1024))));
    return ibcu_launch(ctx, kern, dim3(std::min((p.row_start[n] + WF_WARPS - 1) / WF_WARPS, fit * ctx->sm_count)), dim3(WF_WARPS * 32), smem, 1, true, p);
}

// How a call is cut: tokens in tiles of equal size (up to 256), and columns over S blocks where the tiles leave SMs idle.
struct W8Cut { int NT, token_tiles, S, pairs; };
W8Cut w8_cut(int sm_count, long row_tiles, long pair_tiles, int nkb, int B) {
    W8Cut best = { 0, 0, 1, 0 };
    double least = 1e30;
    for (int n = (B + 255) / 256; n <= (B + 255) / 256 + 3; n++) {
        const int NT = ((B + n - 1) / n + 15) / 16 * 16, tt = (B + NT - 1) / NT;
        for (int S = 1; S <= 8; S *= 2) {
            // (clusters of four and eight find their places in one group of SMs each: 33 and 12 of them at once)
            if (S > 1 && (row_tiles * tt > (S == 2 ? sm_count / 2 : S == 4 ? sm_count * 9 / 40 : sm_count / 12) || nkb < 2 * S)) break;
            const double waves = (double)((row_tiles * tt * S + sm_count - 1) / sm_count);
            // Cycles: a block of columns is as long as its bytes are on their way, 70 of them a cycle (the products of 256 tokens take 524 of the 702); then
            // the results, or S blocks' sums that meet. Over 13 shapes of 8 to 511 tokens within 7 % of the best of all cuts, 2 % on the mean.
            const double t = waves * ((double)((nkb + S - 1) / S) * (16384 + 128 * NT) / 70.0 + (S > 1 ? 1800 + 24 * NT : 900 + 4 * NT));
            if (t < least) { least = t; best = { NT, tt, S, 0 }; }
        }
        // pairs of blocks: half the tokens' codes a block, until the products are what a block of columns takes
        const int NP = (NT + 31) / 32 * 32, tp = (B + NP - 1) / NP;
        const double waves = (double)((pair_tiles * tp + sm_count / 2 - 1) / (sm_count / 2));
        const double t = waves * (nkb * std::max((16384 + 64 * NP) / 70.0, 2.1 * NP) + 1200 + 4 * NP);
        if (t < least) { least = t; best = { NP, tp, 1, 1 }; }
    }
    return best;
}

// x: FP32 tokens, whose codes and scales go into xq (rows ldq apart) and sx first; NULL: they are there
int product(ibcu_ctx* ctx, const ibcu_linear_t* ts, int n, const float* x, int8_t* xq, float* sx, int N, int ldq, int B, const char* call) {
    const size_t pitch = (N + 15) & ~15;
    IBCU_REQUIRE(ctx, tensor_map_encoder(), "%s: the driver has no tensor maps", call);
    // operands whose rows do not start on 16 bytes: copies whose rows do
    size_t need = 0, at[5] = {};
    bool copy[5] = {};
    for (int i = 0; i < n; i++)
        if ((copy[i] = N % 16 || ((uintptr_t)ts[i].w & 15))) { at[i] = need; need += ((size_t)ts[i].M * pitch + 255) & ~(size_t)255; }
    if ((copy[4] = ldq % 16 || ((uintptr_t)xq & 15))) { at[4] = need; need += ((size_t)B * pitch + 255) & ~(size_t)255; }
    AlignJobs jobs;
    memset(&jobs, 0, sizeof jobs);
    if (need) {
        if (int rc = ibcu_reserve(ctx, &ctx->scratch, &ctx->scratch_bytes, need)) return rc;
        long pieces = 0;
        for (int i = 0; i < 5; i++) {
            if (!copy[i]) continue;
            const long rows = i < 4 ? ts[i].M : B;
            jobs.j[jobs.n++] = { (const uint8_t*)(i < 4 ? ts[i].w : xq), (uint8_t*)ctx->scratch + at[i], i < 4 ? N : ldq, (long)pitch, rows, N };
            pieces = std::max(pieces, rows * (long)(pitch / 16));
        }
        jobs.blocks = (int)std::min((pieces + 255) / 256, 8L * ctx->sm_count);
    }
    if (x || need) { if (int rc = quantize<true>(ctx, x, xq, sx, N, ldq, x ? B : 0, jobs)) return rc; }
    W8Maps maps;
    W8Params p;
    memset(&p, 0, sizeof p);
    bool ok = true;
    p.early_weights = 1;
    for (int i = 0; i < n; i++) {
        p.t[i] = ts[i];
        p.tile_start[i + 1] = p.tile_start[i] + (ts[i].M + 127) / 128;
        if (copy[i]) p.early_weights = 0;
        ok = ok && tensor_map_bytes(&maps.w[i], copy[i] ? (uint8_t*)ctx->scratch + at[i] : (const uint8_t*)ts[i].w, ts[i].M, N, copy[i] ? (long)pitch : N, 128);
    }
    for (int i = n; i < 4; i++) maps.w[i] = maps.w[0];
    p.n_tensors = n; p.B = B; p.nkb = (N + 127) / 128; p.edge = N == 131072; p.sx = sx; p.err = ctx->kern_err;
    const long row_tiles = p.tile_start[n];
    long pair_tiles = 0;
    for (int i = 0; i < n; i++) pair_tiles += (ts[i].M + 255) / 256;
    const W8Cut cut = w8_cut(ctx->sm_count, row_tiles, pair_tiles, p.nkb, B);
    const bool pairs = cut.pairs;
    p.NT = cut.NT; p.token_tiles = cut.token_tiles; p.S = cut.S;
    ok = ok && tensor_map_bytes(&maps.x, copy[4] ? (uint8_t*)ctx->scratch + at[4] : (const uint8_t*)xq, B, N, copy[4] ? (long)pitch : ldq, pairs ? p.NT / 2 : p.NT);
    IBCU_REQUIRE(ctx, ok, "%s: no tensor map for N=%d", call, N);
    if (pairs) for (int i = 0; i < n; i++) p.tile_start[i + 1] = p.tile_start[i] + (ts[i].M + 255) / 256;
    const int stage = 16384 + (pairs ? p.NT / 2 : p.NT) * 128, room = 227 * 1024 - (int)sizeof(W8Shared) - 1024;
    p.stages = std::min(std::min(W8_MAX_STAGES, room / stage), std::max(2, (p.nkb + p.S - 1) / p.S * 2));
    size_t rings = (size_t)p.stages * stage;
    const size_t meet = p.S > 1 ? (size_t)p.S * w8_share(p.NT, p.S) * 512 : 0;
    if (rings < meet) { p.stages = (int)((meet + stage - 1) / stage); rings = (size_t)p.stages * stage; }
    for (p.tmem_cols = 32; p.tmem_cols < 2 * p.NT; p.tmem_cols *= 2) {}
    const long tiles = (pairs ? pair_tiles : row_tiles) * p.token_tiles;
    const int grid = p.S > 1 ? (int)tiles * p.S : (int)std::min(tiles, (long)ctx->sm_count);
    const size_t smem = rings + sizeof(W8Shared);
    if (pairs) {
        static SmemOptIn opt_pair;
        if (int rc = ibcu_allow_smem(ctx, opt_pair, w8a8_pair_kernel, smem)) return rc;
        return ibcu_launch(ctx, w8a8_pair_kernel, dim3(2 * (int)std::min(tiles, (long)ctx->sm_count / 2)), dim3(W8_THREADS), smem, 2, true, maps, p);
    }
    static SmemOptIn opt;
    if (int rc = ibcu_allow_smem(ctx, opt, w8a8_tc_kernel, smem)) return rc;
    return ibcu_launch(ctx, w8a8_tc_kernel, dim3(grid), dim3(W8_THREADS), smem, p.S, true, maps, p);
}

}  // namespace

extern "C" int ibcu_quantize_rows_int8(ibcu_ctx* ctx, const float* x, int8_t* q, float* scale, int N, int B) {
    IBCU_CHECK_CTX(ctx);
    IBCU_REQUIRE(ctx, x && q && scale, "ibcu_quantize_rows_int8: null pointer");
    // a block's index into a row steps by 512 beyond its end
    IBCU_REQUIRE(ctx, N >= 1 && N <= (1 << 30) && B >= 1, "ibcu_quantize_rows_int8: N=%d (up to 2^30) B=%d", N, B);
    AlignJobs none;
    memset(&none, 0, sizeof none);
    return quantize<false>(ctx, x, q, scale, N, N, B, none);
}

extern "C" int ibcu_linear_w8a8(ibcu_ctx* ctx, const ibcu_linear_t* tensors, int n_tensors, const int8_t* xq, const float* sx, int N, int B) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_call(ctx, tensors, n_tensors, N, B, "ibcu_linear_w8a8")) return rc;
    IBCU_REQUIRE(ctx, xq && sx, "ibcu_linear_w8a8: null pointer");
    const int rc = product_few(ctx, tensors, n_tensors, nullptr, xq, sx, N, B);
    if (rc != IBCU_DECLINED) return rc;
    return product(ctx, tensors, n_tensors, nullptr, const_cast<int8_t*>(xq), const_cast<float*>(sx), N, N, B, "ibcu_linear_w8a8");
}

extern "C" int ibcu_linear_w8a8_fp32(ibcu_ctx* ctx, const ibcu_linear_t* tensors, int n_tensors, const float* x, int N, int B) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_call(ctx, tensors, n_tensors, N, B, "ibcu_linear_w8a8_fp32")) return rc;
    IBCU_REQUIRE(ctx, x, "ibcu_linear_w8a8_fp32: null pointer");
    int rc = product_few(ctx, tensors, n_tensors, x, nullptr, nullptr, N, B);
    if (rc != IBCU_DECLINED) return rc;
    const int ldq = (N + 15) & ~15;
    const size_t qb = ((size_t)B * ldq + 255) & ~(size_t)255;
    if ((rc = ibcu_reserve(ctx, &ctx->xpack, &ctx->xpack_bytes, qb + (size_t)B * sizeof(float)))) return rc;
    return product(ctx, tensors, n_tensors, x, (int8_t*)ctx->xpack, (float*)((char*)ctx->xpack + qb), N, ldq, B, "ibcu_linear_w8a8_fp32");
}
