// KV cache held in 4 bits: the write of new rows, their read-back, attention over the cache with the attention weight that every row
// draws, and the eviction of rows by that weight.
//
// A row of a KV head is hd values in groups of 32; a group has one fp16 scale s = max|x| * (1 / 7) and codes rint(x / s) + 8 in 1..15, so
// that value = (code - 8) * s. Planes are per KV head, rows of a head one behind the other: k and v [head][max_rows][hd / 2] bytes,
// scale [head][max_rows][2 hd / 32] (the key's groups, then the value's). Inside a row the values lie in the order in which
// the lanes of a matrix instruction take them: a key row is four pieces, piece t with values 8t..8t+7 of group 0, then of group 1, and
// so on; a value row is eight pieces, piece g with values 4g..4g+3 of every group. Two values a byte, the first in the low nibble.
#include "common.cuh"
#include <algorithm>
#include <cmath>

namespace {

struct Kv4 {
    uint8_t* k; uint8_t* v; __half* scale; float* weight;
    int n_kv, hd, max_rows;
    __host__ __device__ size_t row(int h, int r) const { return (size_t)h * max_rows + r; }
};

__device__ __forceinline__ int key_place(int i, int ng) { return ((i & 31) / 8 * ng + i / 32) * 8 + (i & 7); }      // where value i of a row lies
__device__ __forceinline__ int value_place(int i, int ng) { return ((i & 31) / 4 * ng + i / 32) * 4 + (i & 3); }
__device__ __forceinline__ float held(const uint8_t* row, int place, float s) { return (float)((row[place >> 1] >> ((place & 1) * 4) & 15) - 8) * s; }

// The adjacent pair (x0, x1) at angle pos * theta^(-2m / hd): in 64 bits, because far positions times a rounded frequency are off by
// whole steps of a 4-bit code, rounded once at the end.
__device__ __forceinline__ void turn_pair(float& x0, float& x1, int m, int hd, int pos, double log2_theta) {
    double s, c;
    sincos((double)pos * exp2(-2.0 * m / hd * log2_theta), &s, &c);
    const double a = x0, b = x1;
    x0 = (float)(a * c - b * s);
    x1 = (float)(a * s + b * c);
}

// A group's scale and the factor that turns its values into codes; amax_bits: the largest magnitude's bits (NaN and Inf above all)
__device__ __forceinline__ __half group_scale(uint32_t amax_bits, float& inv) {
    if (amax_bits >= 0x7F800000u) { inv = 0.0f; return __ushort_as_half(0x7FFF); }          // NaN: the row says so wherever it is seen
    const float s = __fmul_rn(__uint_as_float(amax_bits), 1.0f / 7.0f);
    const __half h = __float2half_rn(fminf(s, 65504.0f));
    inv = __half2float(h) > 0.0f ? __fdiv_rn(1.0f, __half2float(h)) : 0.0f;
    return h;
}
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
    const float q = inv > 0.0f ? fminf(fmaxf(rintf(__fmul_rn(x, inv)), -7.0f), 7.0f) : 0.0f;
    return (uint32_t)((int)q + 8);
}

// grid (positions, KV heads, 2): the key (z = 0, rotated) or value row of one position; a thread has four values of a row
__global__ void __launch_bounds__(64) kv4_write_kernel(Kv4 c, const float* __restrict__ k, const float* __restrict__ v, int row0, int pos0, double log2_theta, int rotate) {
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x, h = blockIdx.y, i = threadIdx.x * 4, ng = c.hd / 32;
    const bool key = blockIdx.z == 0;
    if (i >= c.hd) return;                                    // whole groups of eight lanes stay
    const float* src = (key ? k : v) + ((size_t)b * c.n_kv + h) * c.hd + i;
    float x[4] = { src[0], src[1], src[2], src[3] };
    if (key && rotate) {
        turn_pair(x[0], x[1], i / 2, c.hd, pos0 + b, log2_theta);
        turn_pair(x[2], x[3], i / 2 + 1, c.hd, pos0 + b, log2_theta);
    }
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < 4; u++) m = max(m, __float_as_uint(x[u]) & 0x7FFFFFFFu);
    const unsigned lanes = 0xFFu << (threadIdx.x & 24);       // the eight lanes of a group
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(lanes, m, o));
    float inv;
    const __half s = group_scale(m, inv);
    uint32_t w = 0;
#pragma unroll
    for (int u = 0; u < 4; u++) w |= code_of(x[u], inv) << (4 * u);
    const size_t row = c.row(h, row0 + b);
    const int place = key ? key_place(i, ng) : value_place(i, ng);       // four values stay together in both orders
    *reinterpret_cast<uint16_t*>((key ? c.k : c.v) + row * (c.hd / 2) + place / 2) = (uint16_t)w;
    if ((i & 31) == 0) c.scale[row * 2 * ng + (key ? 0 : ng) + i / 32] = s;
    if (key && i == 0 && c.weight) c.weight[row] = 0.0f;
}

// grid (rows, KV heads): the values that the cache holds
__global__ void __launch_bounds__(128) kv4_read_kernel(Kv4 c, float* __restrict__ k, float* __restrict__ v, int row0) {
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x, h = blockIdx.y, ng = c.hd / 32;
    const size_t row = c.row(h, row0 + b);
    for (int i = threadIdx.x; i < c.hd; i += blockDim.x) {
        const size_t o = ((size_t)b * c.n_kv + h) * c.hd + i;
        k[o] = held(c.k + row * (c.hd / 2), key_place(i, ng), __half2float(c.scale[row * 2 * ng + i / 32]));
        v[o] = held(c.v + row * (c.hd / 2), value_place(i, ng), __half2float(c.scale[row * 2 * ng + ng + i / 32]));
    }
}

__global__ void __launch_bounds__(128) turn_queries_kernel(const float* __restrict__ q, float* __restrict__ out, int hd, int n_heads, int pos0, double log2_theta, int rotate) {
    pdl_launch_dependents();
    pdl_wait();
    const size_t base = ((size_t)blockIdx.x * n_heads + blockIdx.y) * hd;
    for (int m = threadIdx.x; m < hd / 2; m += blockDim.x) {
        float a = q[base + 2 * m], b = q[base + 2 * m + 1];
        if (rotate) turn_pair(a, b, m, hd, pos0 + blockIdx.x, log2_theta);
        out[base + 2 * m] = a; out[base + 2 * m + 1] = b;
    }
}

// grid (positions, query heads), 8 warps: a warp takes every eighth row, a lane one value of each group, with a running maximum and sum
__global__ void __launch_bounds__(256) kv4_attn_kernel(Kv4 c, const float* __restrict__ q, float* __restrict__ out, float2* __restrict__ stat, int n_heads, int row0) {
    __shared__ float sm[8], sl[8], sa[8][256];
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.x, h = blockIdx.y, kvh = h / (n_heads / c.n_kv), lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ng = c.hd / 32;
    const size_t at = ((size_t)b * n_heads + h) * c.hd;
    const float scale = 1.0f / sqrtf((float)c.hd);
    float qv[8], acc[8], m = -INFINITY, l = 0.0f;
    for (int j = 0; j < 8; j++) { qv[j] = j < ng ? q[at + 32 * j + lane] : 0.0f; acc[j] = 0.0f; }
    for (int r = warp; r <= row0 + b; r += 8) {
        const size_t row = c.row(kvh, r);
        float s = 0.0f;
        for (int j = 0; j < 8; j++)
            if (j < ng) s = fmaf(qv[j], held(c.k + row * (c.hd / 2), key_place(32 * j + lane, ng), __half2float(c.scale[row * 2 * ng + j])), s);
        s = warp_sum(s) * scale;
        const float mn = fmaxf(m, s), corr = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(s - mn);
        l = l * corr + p;
        for (int j = 0; j < 8; j++)
            if (j < ng) acc[j] = acc[j] * corr + p * held(c.v + row * (c.hd / 2), value_place(32 * j + lane, ng), __half2float(c.scale[row * 2 * ng + ng + j]));
        m = mn;
    }
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
    for (int j = 0; j < 8; j++) sa[warp][32 * j + lane] = acc[j];
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
    for (int w = 0; w < 8; w++) M = fmaxf(M, sm[w]);
    for (int w = 0; w < 8; w++) L += sl[w] == 0.0f ? 0.0f : sl[w] * expf(sm[w] - M);
    for (int d = threadIdx.x; d < c.hd; d += 256) {
        float a = 0.0f;
        for (int w = 0; w < 8; w++) a += sl[w] == 0.0f ? 0.0f : sa[w][d] * expf(sm[w] - M);
        out[at + d] = a / L;
    }
    if (threadIdx.x == 0 && stat) stat[(size_t)b * n_heads + h] = make_float2(M, L);
}

// grid (rows, KV heads), a warp: weight of a row = decay * weight + its share of every query's attention
__global__ void __launch_bounds__(32) kv4_weight_kernel(Kv4 c, const float* __restrict__ q, const float2* __restrict__ stat, int n_heads, int row0, int B, float decay) {
    pdl_launch_dependents();
    pdl_wait();
    const int r = blockIdx.x, kvh = blockIdx.y, group = n_heads / c.n_kv, lane = threadIdx.x, ng = c.hd / 32;
    const size_t row = c.row(kvh, r);
    const float scale = 1.0f / sqrtf((float)c.hd);
    float kv[8], w = 0.0f;
    for (int j = 0; j < 8; j++) kv[j] = j < ng ? held(c.k + row * (c.hd / 2), key_place(32 * j + lane, ng), __half2float(c.scale[row * 2 * ng + j])) : 0.0f;
    for (int b = max(0, r - row0); b < B; b++)
        for (int g = 0; g < group; g++) {
            const int h = kvh * group + g;
            const float* qh = q + ((size_t)b * n_heads + h) * c.hd;
            float s = 0.0f;
            for (int j = 0; j < 8; j++) if (j < ng) s = fmaf(kv[j], qh[32 * j + lane], s);
            s = warp_sum(s) * scale;
            const float2 st = stat[(size_t)b * n_heads + h];
            w += expf(s - st.x) / st.y;
        }
    if (lane == 0) c.weight[row] = (decay == 0.0f ? 0.0f : decay * c.weight[row]) + w;
}

// weights as whole numbers in the order of the choice: larger weight first, NaN last, the two zeros equal
__device__ __forceinline__ uint32_t weight_order(float w) {
    const uint32_t u = __float_as_uint(w);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
    if ((u << 1) == 0u) return 0x80000000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// one block per KV head: the `want` rows of [lo, hi) with the largest weights, equal ones from the lowest row, beside all rows outside it,
// in ascending order into kept[]. The bound is found bit by bit.
__global__ void __launch_bounds__(1024) kv4_choose_kernel(Kv4 c, int32_t* __restrict__ kept, int rows, int keep, int lo, int hi, int want) {
    __shared__ int count, base_gt, base_eq;
    __shared__ int wsum[32], wsum2[32];
    pdl_launch_dependents();
    pdl_wait();
    const int h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* w = c.weight + c.row(h, 0);
    uint32_t bound = 0;                                       // the largest order that at least `want` rows reach
    for (int bit = 31; bit >= 0 && want > 0; bit--) {
        const uint32_t t = bound | 1u << bit;
        __syncthreads();
        if (tid == 0) count = 0;
        __syncthreads();
        int n = 0;
        for (int r = lo + tid; r < hi; r += 1024) n += weight_order(w[r]) >= t;
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0) atomicAdd(&count, n);
        __syncthreads();
        if (count >= want) bound = t;
    }
    __syncthreads();
    if (tid == 0) count = 0;
    __syncthreads();
    int n = 0;
    for (int r = lo + tid; r < hi; r += 1024) n += weight_order(w[r]) > bound;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) atomicAdd(&count, n);
    __syncthreads();
    const int ties = want - count;                            // rows at the bound that stay, from the lowest
    if (tid == 0) { base_gt = 0; base_eq = 0; }
    for (int r0 = 0; r0 < rows; r0 += 1024) {
        __syncthreads();
        const int r = r0 + tid;
        const bool inside = r >= lo && r < hi;
        const uint32_t o = inside ? weight_order(w[r]) : 0u;
        const bool eq = inside && o == bound && want > 0, sure = r < rows && (!inside || (want > 0 && o > bound));
        const unsigned me = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) wsum[warp] = __popc(me);
        __syncthreads();
        int eq_before = base_eq + __popc(me & ((1u << lane) - 1));
        for (int i = 0; i < warp; i++) eq_before += wsum[i];
        const bool stay = sure || (eq && eq_before < ties);
        const unsigned ms = __ballot_sync(0xffffffffu, stay);
        if (lane == 0) wsum2[warp] = __popc(ms);
        __syncthreads();
        int at = base_gt + __popc(ms & ((1u << lane) - 1));
        for (int i = 0; i < warp; i++) at += wsum2[i];
        if (stay && at < keep) kept[(size_t)h * keep + at] = r;
        __syncthreads();
        if (tid == 0) for (int i = 0; i < 32; i++) { base_eq += wsum[i]; base_gt += wsum2[i]; }
    }
}

// grid (pieces, KV heads): a block moves 16 bytes (4 of the weights) of every kept row. Rows only move towards the front, so a pass that has
// all its rows in registers before it stores the first may write over the rows it came from.
__global__ void __launch_bounds__(1024) kv4_move_kernel(Kv4 src, Kv4 dst, const int32_t* __restrict__ kept, int keep) {
    pdl_launch_dependents();
    pdl_wait();
    const int h = blockIdx.y, kp = src.hd / 32, sp = src.hd / 32;                     // pieces of 16 bytes in a code row; words of 4 bytes in a row of scales
    const int32_t* idx = kept + (size_t)h * keep;
    const int p = blockIdx.x;
    for (int i0 = 0; i0 < keep; i0 += 1024) {
        const int i = i0 + threadIdx.x;
        uint4 x = make_uint4(0, 0, 0, 0);
        size_t from = 0, to = 0;
        if (i < keep) {
            from = src.row(h, idx[i]); to = dst.row(h, i);
            if (p < kp) x = reinterpret_cast<const uint4*>(src.k)[from * kp + p];
            else if (p < 2 * kp) x = reinterpret_cast<const uint4*>(src.v)[from * kp + p - kp];
            else if (p < 2 * kp + sp) x.x = reinterpret_cast<const uint32_t*>(src.scale)[from * sp + p - 2 * kp];
            else if (src.weight && dst.weight) x.x = __float_as_uint(src.weight[from]);
        }
        __syncthreads();
        if (i < keep) {
            if (p < kp) reinterpret_cast<uint4*>(dst.k)[to * kp + p] = x;
            else if (p < 2 * kp) reinterpret_cast<uint4*>(dst.v)[to * kp + p - kp] = x;
            else if (p < 2 * kp + sp) reinterpret_cast<uint32_t*>(dst.scale)[to * sp + p - 2 * kp] = x.x;
            else if (src.weight && dst.weight) dst.weight[to] = __uint_as_float(x.x);
        }
        __syncthreads();
    }
}

Kv4 planes(const ibcu_kv4_t* t) { return Kv4{ t->k, t->v, (__half*)t->scale, t->weight, t->n_kv_heads, t->head_dim, t->max_rows }; }

int check_cache(ibcu_ctx* ctx, const ibcu_kv4_t* t, const char* call) {
    IBCU_REQUIRE(ctx, t && t->k && t->v && t->scale, "%s: null pointer", call);
    const int hd = t->head_dim;
    IBCU_REQUIRE(ctx, hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 192 || hd == 256, "%s: head_dim=%d (32, 64, 96, 128, 192 or 256)", call, hd);
    IBCU_REQUIRE(ctx, t->n_kv_heads >= 1 && t->n_kv_heads <= 1024 && t->max_rows >= 8 && t->max_rows % 8 == 0, "%s: n_kv_heads=%d max_rows=%d (rows in multiples of 8)", call, t->n_kv_heads, t->max_rows);
    IBCU_REQUIRE(ctx, (((uintptr_t)t->k | (uintptr_t)t->v | (uintptr_t)t->scale) & 15) == 0 && ((uintptr_t)t->weight & 3) == 0, "%s: k, v and scale must be 16-byte aligned", call);
    IBCU_REQUIRE(ctx, !t->weight || (t->decay >= 0.0f && t->decay <= 1.0f), "%s: decay=%g outside 0..1", call, (double)t->decay);
    return IBCU_OK;
}
int check_rows(ibcu_ctx* ctx, const ibcu_kv4_t* t, int row0, int n, const char* call) {
    IBCU_REQUIRE(ctx, row0 >= 0 && n >= 1 && (long)row0 + n <= t->max_rows, "%s: rows %d..%ld outside the cache of %d", call, row0, (long)row0 + n, t->max_rows);
    return IBCU_OK;
}
int check_rotation(ibcu_ctx* ctx, int pos0, int B, float theta, const char* call) {
    IBCU_REQUIRE(ctx, pos0 >= 0 && (long)pos0 + B <= 0x7FFFFFFFL && theta >= 0.0f && theta <= 3.0e38f, "%s: pos0=%d theta=%g", call, pos0, (double)theta);
    return IBCU_OK;
}
double log2_of(float theta) { return theta > 0.0f ? log2((double)theta) : 0.0; }

int attend(ibcu_ctx* ctx, const Kv4& c, float decay, const float* q, float* out, int n_heads, int row0, int B, float2* stat) {
    int rc = ibcu_launch(ctx, kv4_attn_kernel, dim3(B, n_heads), dim3(256), 0, 1, true, c, q, out, stat, n_heads, row0);
    if (!rc && c.weight) rc = ibcu_launch(ctx, kv4_weight_kernel, dim3(row0 + B, c.n_kv), dim3(32), 0, 1, true, c, q, (const float2*)stat, n_heads, row0, B, decay);
    return rc;
}

}  // namespace

extern "C" int ibcu_kv4_write(ibcu_ctx* ctx, const ibcu_kv4_t* cache, const float* k, const float* v, int row0, int pos0, int B, float theta) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_cache(ctx, cache, "ibcu_kv4_write")) return rc;
    IBCU_REQUIRE(ctx, k && v, "ibcu_kv4_write: null pointer");
    if (int rc = check_rows(ctx, cache, row0, B, "ibcu_kv4_write")) return rc;
    if (int rc = check_rotation(ctx, pos0, B, theta, "ibcu_kv4_write")) return rc;
    return ibcu_launch(ctx, kv4_write_kernel, dim3(B, cache->n_kv_heads, 2), dim3(64), 0, 1, true, planes(cache), k, v, row0, pos0, log2_of(theta), theta > 0.0f ? 1 : 0);
}

extern "C" int ibcu_kv4_read(ibcu_ctx* ctx, const ibcu_kv4_t* cache, float* k, float* v, int row0, int n) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_cache(ctx, cache, "ibcu_kv4_read")) return rc;
    IBCU_REQUIRE(ctx, k && v, "ibcu_kv4_read: null pointer");
    if (int rc = check_rows(ctx, cache, row0, n, "ibcu_kv4_read")) return rc;
    return ibcu_launch(ctx, kv4_read_kernel, dim3(n, cache->n_kv_heads), dim3(128), 0, 1, true, planes(cache), k, v, row0);
}

static int check_heads(ibcu_ctx* ctx, const ibcu_kv4_t* cache, int n_heads, int B, const char* call) {
    IBCU_REQUIRE(ctx, n_heads >= 1 && n_heads <= 65535 && n_heads % cache->n_kv_heads == 0, "%s: %d heads over %d", call, n_heads, cache->n_kv_heads);
    return IBCU_OK;
}

extern "C" int ibcu_attention_kv4(ibcu_ctx* ctx, const ibcu_kv4_t* cache, const float* q, float* out, int n_heads, int row0, int B) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_cache(ctx, cache, "ibcu_attention_kv4")) return rc;
    IBCU_REQUIRE(ctx, q && out, "ibcu_attention_kv4: null pointer");
    if (int rc = check_rows(ctx, cache, row0, B, "ibcu_attention_kv4")) return rc;
    if (int rc = check_heads(ctx, cache, n_heads, B, "ibcu_attention_kv4")) return rc;
    int rc = ibcu_reserve(ctx, &ctx->scratch, &ctx->scratch_bytes, (size_t)B * n_heads * sizeof(float2));
    if (rc) return rc;
    return attend(ctx, planes(cache), cache->decay, q, out, n_heads, row0, B, (float2*)ctx->scratch);
}

extern "C" int ibcu_attention_decode_kv4(ibcu_ctx* ctx, const ibcu_kv4_t* cache, const float* q, const float* k, const float* v, float* out,
                                         int n_heads, int row0, int pos0, int B, float theta) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_cache(ctx, cache, "ibcu_attention_decode_kv4")) return rc;
    IBCU_REQUIRE(ctx, q && k && v && out, "ibcu_attention_decode_kv4: null pointer");
    if (int rc = check_rows(ctx, cache, row0, B, "ibcu_attention_decode_kv4")) return rc;
    if (int rc = check_heads(ctx, cache, n_heads, B, "ibcu_attention_decode_kv4")) return rc;
    if (int rc = check_rotation(ctx, pos0, B, theta, "ibcu_attention_decode_kv4")) return rc;
    const size_t st = ((size_t)B * n_heads * sizeof(float2) + 255) & ~(size_t)255;
    int rc = ibcu_reserve(ctx, &ctx->scratch, &ctx->scratch_bytes, st + (size_t)B * n_heads * cache->head_dim * sizeof(float));
    if (rc) return rc;
    float* qr = (float*)((char*)ctx->scratch + st);
    rc = ibcu_kv4_write(ctx, cache, k, v, row0, pos0, B, theta);
    if (!rc) rc = ibcu_launch(ctx, turn_queries_kernel, dim3(B, n_heads), dim3(128), 0, 1, true, q, qr, cache->head_dim, n_heads, pos0, log2_of(theta), theta > 0.0f ? 1 : 0);
    if (!rc) rc = attend(ctx, planes(cache), cache->decay, qr, out, n_heads, row0, B, (float2*)ctx->scratch);
    return rc;
}

extern "C" int ibcu_kv4_evict(ibcu_ctx* ctx, const ibcu_kv4_t* src, const ibcu_kv4_t* dst, int rows, int keep, int sink, int recent, int32_t* kept) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_cache(ctx, src, "ibcu_kv4_evict")) return rc;
    if (int rc = check_cache(ctx, dst, "ibcu_kv4_evict")) return rc;
    IBCU_REQUIRE(ctx, src->weight, "ibcu_kv4_evict: the cache keeps no weights to go by");
    IBCU_REQUIRE(ctx, src->n_kv_heads == dst->n_kv_heads && src->head_dim == dst->head_dim, "ibcu_kv4_evict: caches of different heads");
    IBCU_REQUIRE(ctx, rows >= 1 && rows <= src->max_rows && keep >= 1 && keep <= rows && keep <= dst->max_rows && sink >= 0 && recent >= 0 && (long)sink + recent <= keep,
                 "ibcu_kv4_evict: %d of %d rows (at most %d), first %d and last %d", keep, rows, dst->max_rows, sink, recent);
    const int nkv = src->n_kv_heads;
    if (!kept) {
        int rc = ibcu_reserve(ctx, &ctx->scratch, &ctx->scratch_bytes, (size_t)nkv * keep * sizeof(int32_t));
        if (rc) return rc;
        kept = (int32_t*)ctx->scratch;
    }
    int rc = ibcu_launch(ctx, kv4_choose_kernel, dim3(nkv), dim3(1024), 0, 1, true, planes(src), kept, rows, keep, sink, rows - recent, keep - sink - recent);
    if (!rc) rc = ibcu_launch(ctx, kv4_move_kernel, dim3(3 * (src->head_dim / 32) + 1, nkv), dim3(1024), 0, 1, true, planes(src), planes(dst), (const int32_t*)kept, keep);
    return rc;
}
