// What the kernels of the 4-bit KV cache share: the cache's planes, the order of a row, and how a call's query heads are laid out for the
// matrix instructions. See kv4.cu for the cache and kv4_attn.cu for the attention.
#pragma once
#include "common.cuh"

struct Kv4 {
    uint8_t* k; uint8_t* v; __half* scale; float* weight;
    int n_kv, hd, max_rows;
    __host__ __device__ size_t row(int h, int r) const { return (size_t)h * max_rows + r; }
};

// The columns of a KV head are its query heads at every position, column = position * group + head of the group. They go through the
// kernels in one tile (up to 8 columns) or in tiles of 16. The queries of a tile of 16 are the A operand's fragments, two fp16 pieces of every
// value: [unit = KV head * tiles + tile][part][group of 32][step][lane] uint4, a part for the high pieces and one for the low ones, with columns 0-7 in the
// fragments' even registers and 8-15 in the odd ones. Beside them qc [unit][16]: the factor that turns a column's sums into exponents of 2.
// Prompts (kv4_prompt.cu) go in tiles of 128 columns, eight of 16 side by side, as operand images instead: [KV head * tiles + tile][part][64 values][column]
// rows of 128 bytes in the 128-byte swizzle, a row's 16-byte pieces in the order of a key row's words (piece t * (hd / 32) + j: values 32 j + 8 t..), the eight values of a
// piece as 0, 4, 1, 5, 2, 6, 3, 7.
struct Kv4Columns {
    int n_heads, group, B, large, ntiles;                      // large: tiles of 16; 2: as images, ntiles a multiple of 8
    __host__ __device__ int cols() const { return large ? 16 : 8; }
};
__host__ __device__ constexpr size_t kv4_frags(int ng) { return (size_t)ng * 128; }            // uint4s of a unit

// where rows and positions of a call are: arguments, or {row0, pos0} in device memory
struct Kv4Place { int row0, pos0; const int* at; };
// Reads them where they are on the device. False, and the context's error word set, if the rows would not fit or the positions pass 31 bits, as the calls with arguments refuse them.
__device__ __forceinline__ bool kv4_place(const Kv4Place& p, int B, int max_rows, int* err, int& row0, int& pos0) {
    row0 = p.row0; pos0 = p.pos0;
    if (!p.at) return true;
    row0 = __ldcg(p.at); pos0 = __ldcg(p.at + 1);
    if (row0 >= 0 && pos0 >= 0 && row0 <= max_rows - B && pos0 <= 0x7FFFFFFF - B) return true;
    *err = IBCU_KV4_PLACE_ERR;
    return false;
}

// ── rows ──
__device__ __forceinline__ int kv4_key_place(int i, int ng) { return ((i & 31) / 8 * ng + i / 32) * 8 + (i & 7); }      // where value i of a row lies
__device__ __forceinline__ int kv4_value_place(int i, int ng) { return ((i & 31) / 4 * ng + i / 32) * 4 + (i & 3); }

// Angles of positions pos0, pos0 + 1, ..: turn[position][pair % 4][pair / 4] (threads with neighbouring eights of values read neighbours) = cosine and sine of position * theta^(-2 pair / hd), in 64 bits, because far positions
// times a rounded frequency are off by whole steps of a 4-bit code. By all threads of a block; about a microsecond.
__device__ __forceinline__ void kv4_angles(double2* turn, int positions, int pos0, int hd, double log2_theta) {
    const int half = hd / 2;
    for (int e = threadIdx.x; e < positions * half; e += blockDim.x) {
        double s, c;
        sincos(((double)pos0 + e / half) * exp2((double)(e % half) * (-2.0 / hd * log2_theta)), &s, &c);
        turn[e / half * half + (e & 3) * (half / 4) + e % half / 4] = make_double2(c, s);
    }
}
// an adjacent pair, turned in 64 bits and rounded once
__device__ __forceinline__ void kv4_turn(float& x0, float& x1, const double2 cs) {
    const double a = x0, z = x1;
    x0 = (float)(a * cs.x - z * cs.y);
    x1 = (float)(a * cs.y + z * cs.x);
}
// A group's scale and the factor that turns its values into codes; amax_bits: the largest magnitude's bits (NaN and Inf above all)
__device__ __forceinline__ __half kv4_scale(uint32_t amax_bits, float& inv) {
    if (amax_bits >= 0x7F800000u) { inv = 0.0f; return __ushort_as_half(0x7FFF); }          // NaN: the row says so wherever it is seen
    const float s = __fmul_rn(__uint_as_float(amax_bits), 1.0f / 7.0f);
    const __half h = __float2half_rn(fminf(s, 8192.0f));                                    // seven of them, the largest value, are an fp16 too
    inv = __half2float(h) > 0.0f ? __frcp_rn(__half2float(h)) : 0.0f;
    return h;
}
// Eight codes. What is added lifts a value's integer part to the lowest bits, rounded to even as rint does.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], float inv) {
    uint32_t w = 0;
#pragma unroll
    for (int u = 0; u < 8; u++) w |= (__float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(x[u], inv), -7.0f), 7.0f), 12582920.0f)) & 15u) << (4 * u);
    return inv > 0.0f ? w : 0x88888888u;
}
// eight values of a row, at any address
__device__ __forceinline__ void kv4_load_eight(float (&x)[8], const float* src) {
    if (((uintptr_t)src & 15) == 0) {                          // else every lane's sector is fetched eight times
        const float4 a = __ldcg(reinterpret_cast<const float4*>(src)), b = __ldcg(reinterpret_cast<const float4*>(src) + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __ldcg(src + i);
    }
}
// Values i..i+7 of a key or value row of head h into the cache. Four neighbouring lanes have a group, whose largest magnitude they
// share. turn: the position's angles, or NULL.
template <int NG>
__device__ __forceinline__ void kv4_write_eight(const Kv4& c, float (&x)[8], bool key, int h, int r, int i, const double2* turn) {
    const int lane = threadIdx.x & 31;
    if (key && turn) {
#pragma unroll
        for (int u = 0; u < 4; u++) kv4_turn(x[2 * u], x[2 * u + 1], turn[u * 4 * NG + i / 8]);
    }
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < 8; u++) m = max(m, __float_as_uint(x[u]) & 0x7FFFFFFFu);
    const unsigned lanes = 0xFu << (lane & 28);
    m = max(m, __shfl_xor_sync(lanes, m, 1));
    m = max(m, __shfl_xor_sync(lanes, m, 2));
    float inv;
    const __half s = kv4_scale(m, inv);
    const uint32_t w = kv4_codes(x, inv);
    const size_t row = c.row(h, r);
    uint8_t* to = (key ? c.k : c.v) + row * (16 * NG);
    if (key) *reinterpret_cast<uint32_t*>(to + kv4_key_place(i, NG) / 2) = w;               // a word of the key's order, two pieces of the value's
    else {
        *reinterpret_cast<uint16_t*>(to + kv4_value_place(i, NG) / 2) = (uint16_t)w;
        *reinterpret_cast<uint16_t*>(to + kv4_value_place(i + 4, NG) / 2) = (uint16_t)(w >> 16);
    }
    if ((i & 31) == 0) c.scale[row * 2 * NG + (key ? 0 : NG) + i / 32] = s;
    if (key && i == 0 && c.weight) c.weight[row] = 0.0f;
}

// ── queries ──
// values i..i+7 of one query (src: the first of them), turned by its position's angles (turn, or NULL)
template <int NG>
__device__ __forceinline__ void kv4_query(float (&x)[8], const float* src, bool on, const double2* turn, int i) {
#pragma unroll
    for (int u = 0; u < 8; u++) x[u] = 0.0f;
    if (!on) return;
    kv4_load_eight(x, src);
    if (turn) {
#pragma unroll
        for (int u = 0; u < 4; u++) kv4_turn(x[2 * u], x[2 * u + 1], turn[u * 4 * NG + i / 8]);
    }
}
// The largest magnitude of a query goes to [2^13, 2^14). A power of 2 up to 2^120, in two factors: what that leaves small are queries below
// 2^-106, whose scores are zeros beside one another anyway. back: takes it off the sums again; log2(e) makes exponents of 2 of them.
struct Kv4Up { float a, b, back; };
__device__ __forceinline__ Kv4Up kv4_up(uint32_t amax_bits, int hd) {
    const int e = min(120, max(-114, 13 - ((int)(amax_bits >> 23) - 127)));
    return { __int_as_float(((e >> 1) + 127) << 23), __int_as_float((e - (e >> 1) + 127) << 23),
             (float)fmin((double)__int_as_float((min(126, -e) + 127) << 23) * (1.4426950408889634 / sqrt((double)hd)), 3.0e38) };
}
// Fragments of step s: high and low pieces of codes 2 s and 2 s + 4 of the lane's eight, and of 2 s + 1 and 2 s + 5, which reach the product 16-fold
__device__ __forceinline__ void kv4_pieces(const float (&x)[8], int s, uint32_t (&hi)[2], uint32_t (&lo)[2]) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const float f = u ? 0.0625f : 1.0f, a = x[2 * s + u] * f, z = x[2 * s + u + 4] * f;
        const __half2 h = __floats2half2_rn(a, z), l = __floats2half2_rn(a - __low2float(h), z - __high2float(h));
        hi[u] = *reinterpret_cast<const uint32_t*>(&h);
        lo[u] = *reinterpret_cast<const uint32_t*>(&l);
    }
}

// Prepares a call's queries (q != NULL) and writes its rows (k != NULL), one launch. Defined in kv4.cu.
struct Kv4Prep { const float *q, *k, *v; uint4* qf; float* qc; double log2_theta; int rotate; };
int kv4_prepare(ibcu_ctx* ctx, const Kv4& c, const Kv4Columns& t, const Kv4Place& at, const Kv4Prep& w);
// A prompt's attention over images that are prepared: kv4_prompt.cu, for head_dim 64 and 128. stat, parts: for the weights, or NULL.
int kv4_prompt_parts(ibcu_ctx* ctx, const Kv4& c, int tiles, int rows);
int kv4_prompt(ibcu_ctx* ctx, const Kv4& c, const Kv4Columns& t, const Kv4Place& at, const unsigned char* image, const float* qc, float* out, float2* stat, int rows, float* parts, int n_parts);
// The attention of a call, with what it has to prepare. q, k, v as above (k NULL: the rows are there). Defined in kv4_attn.cu.
int kv4_attend(ibcu_ctx* ctx, const Kv4& c, float decay, const Kv4Place& at, const float* q, const float* k, const float* v, float* out, int n_heads, int B, double log2_theta, int rotate);
