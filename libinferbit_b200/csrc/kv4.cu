// KV cache held in 4 bits: the write of new rows, their read-back, attention over the cache with the attention weight that every row
// draws, and the eviction of rows by that weight.
//
// A row of a KV head is hd values in groups of 32; a group has one fp16 scale s = max|x| * (1 / 7) and codes rint(x / s) + 8 in 1..15, so
// that value = (code - 8) * s. Planes are per KV head, rows of a head one behind the other: k and v [head][max_rows][hd / 2] bytes,
// scale [head][max_rows][2 hd / 32] (the key's groups, then the value's). Inside a row the values lie in the order in which
// the lanes of a matrix instruction take them: a key row is four pieces, piece t with values 8t..8t+7 of group 0, then of group 1, and
// so on; a value row is eight pieces, piece g with values 4g..4g+3 of every group. Two values a byte, the first in the low nibble.
#include "kv4.cuh"
#include "tc_common.cuh"
#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

__device__ __forceinline__ float scale_at(const __half* p) { return __half2float(__ushort_as_half(__ldcg(reinterpret_cast<const unsigned short*>(p)))); }

// One launch ahead of the attention of more than eight columns, and that of ibcu_kv4_write: blocks below qblocks turn a tile of 16 columns of every
// qparts-th KV head into fragments or their part of an image, the others write the rows of a position. Heads share a position's angles. Bound by
// instructions: 29 for 32 values of rows, 17 of queries, and the turning. The rows of 2048 positions of 8 heads of 128 values 6.9 us (5.8 unturned, 2.9 for the
// bytes); 11.6 with four values a thread, lengths not known at compile time and a position's angles in the order of its pairs.
struct PrepParams { Kv4 c; Kv4Columns t; Kv4Place at; Kv4Prep w; int qblocks, qparts, wparts; int* err; };

template <int NG>
__global__ void __launch_bounds__(128) kv4_prep_kernel(const PrepParams p) {
    constexpr int HD = 32 * NG, HALF = HD / 2, JT = (NG + 3) / 4;
    extern __shared__ __align__(16) double2 turn[];           // [positions of the block][HALF]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool queries = (int)blockIdx.x < p.qblocks;
    // a block of a few rows is short: no division that it can do without
    int tile = 0, c0 = 0, b0 = blockIdx.x - p.qblocks, b1, part = 0;
    if (queries) {
        tile = blockIdx.x % p.t.ntiles;
        c0 = tile * 16;
        b0 = c0 / p.t.group;
        b1 = min(p.t.B - 1, (c0 + 15) / p.t.group);
    } else {
        if (p.wparts > 1) { part = b0 % p.wparts; b0 /= p.wparts; }
        b1 = b0;
    }
    int row0 = p.at.row0, pos0 = p.at.pos0;
    if (p.at.at) {
        pdl_wait();
        if (!kv4_place(p.at, p.t.B, p.c.max_rows, p.err, row0, pos0)) return;
    }
    if (p.w.rotate) kv4_angles(turn, b1 - b0 + 1, pos0 + b0, HD, p.w.log2_theta);
    if (!p.at.at) pdl_wait();
    pdl_launch_dependents();                                  // not earlier: the attention reads rows of earlier calls ahead of its own wait
    __syncthreads();
    if ((NG == 2 || NG == 4) && queries && p.t.large == 2) {
        // a warp has four columns, eight lanes each, whose pieces are whole sectors of the image
        const int col = warp * 4 + (lane >> 3), pl = lane & 7, b = (c0 + col) / p.t.group, head = (c0 + col) % p.t.group, at = tile % 8 * 16 + col;
        const bool on = b < p.t.B;
        const double2* angles = p.w.rotate ? turn + (b - b0) * HALF : nullptr;
#pragma unroll 2
        for (int kvh = blockIdx.x / p.t.ntiles; kvh < p.c.n_kv; kvh += p.qparts) {
            const size_t unit = (size_t)kvh * p.t.ntiles + tile;
            const float* src = p.w.q + ((size_t)b * p.t.n_heads + (size_t)kvh * p.t.group + head) * HD;
            constexpr int PL = NG < 4 ? 1 : NG / 2;           // pieces of a lane
            float x[PL][8];
            uint32_t m = 0;
#pragma unroll
            for (int u = 0; u < PL; u++) {
                const int piece = pl + 8 * u, i = piece % NG * 32 + piece / NG * 8;
                kv4_query<NG>(x[u], src + i, on, angles, i);
#pragma unroll
                for (int n = 0; n < 8; n++) m = max(m, __float_as_uint(x[u][n]) & 0x7FFFFFFFu);
            }
#pragma unroll
            for (int o = 1; o < 8; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const Kv4Up up = kv4_up(m, HD);
            if (pl == 0) p.w.qc[unit * 16 + col] = up.back;
            unsigned char* image = reinterpret_cast<unsigned char*>(p.w.qf) + unit / 8 * (NG * 16384) + at * 128 + ((pl ^ (at & 7)) << 4);
#pragma unroll
            for (int u = 0; u < PL; u++) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float a = x[u][i] * up.a * up.b, z = x[u][i + 4] * up.a * up.b;
                    const __half2 h = __floats2half2_rn(a, z), l = __floats2half2_rn(a - __low2float(h), z - __high2float(h));
                    hi[i] = *reinterpret_cast<const uint32_t*>(&h);
                    lo[i] = *reinterpret_cast<const uint32_t*>(&l);
                }
                *reinterpret_cast<uint4*>(image + u * 16384) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(image + (NG / 2 + u) * 16384) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        return;
    }
    if (queries) {
        // lane = column g and column g + 8, piece t: values 8t..8t+7 of every group; a warp has every fourth group
        __shared__ uint32_t amax[2][4][16];
        const int g = lane >> 2, t = lane & 3;
        int b[2], head[2];
#pragma unroll
        for (int n = 0; n < 2; n++) { const int col = c0 + g + 8 * n; b[n] = col / p.t.group; head[n] = col % p.t.group; }
        int turns = 0;
        for (int kvh = blockIdx.x / p.t.ntiles; kvh < p.c.n_kv; kvh += p.qparts, turns ^= 1) {
            const size_t unit = (size_t)kvh * p.t.ntiles + tile;
            float x[2][JT][8];
            uint32_t m[2] = { 0, 0 };
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const bool on = b[n] < p.t.B;
                const float* src = p.w.q + ((size_t)b[n] * p.t.n_heads + (size_t)kvh * p.t.group + head[n]) * HD + 8 * t;
                const double2* angles = p.w.rotate ? turn + (b[n] - b0) * HALF : nullptr;
#pragma unroll
                for (int jj = 0; jj < JT; jj++) {
                    const int j = warp + 4 * jj;
                    if (j >= NG) break;
                    kv4_query<NG>(x[n][jj], src + 32 * j, on, angles, 32 * j + 8 * t);
#pragma unroll
                    for (int i = 0; i < 8; i++) m[n] = max(m[n], __float_as_uint(x[n][jj][i]) & 0x7FFFFFFFu);
                }
                m[n] = max(m[n], __shfl_xor_sync(0xffffffffu, m[n], 1));
                m[n] = max(m[n], __shfl_xor_sync(0xffffffffu, m[n], 2));
                if (t == 0) amax[turns][warp][g + 8 * n] = m[n];
            }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < 2; n++) {
#pragma unroll
                for (int w = 0; w < 4; w++) m[n] = max(m[n], amax[turns][w][g + 8 * n]);
                const Kv4Up up = kv4_up(m[n], HD);
                if (warp == 0 && t == 0) p.w.qc[unit * 16 + g + 8 * n] = up.back;
#pragma unroll
                for (int jj = 0; jj < JT; jj++)
#pragma unroll
                    for (int i = 0; i < 8; i++) x[n][jj][i] = x[n][jj][i] * up.a * up.b;
            }
#pragma unroll
            for (int jj = 0; jj < JT; jj++) {
                const int j = warp + 4 * jj;
                if (j >= NG) break;
                uint4* qf = p.w.qf + unit * kv4_frags(NG) + lane;
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    uint32_t hi[2][2], lo[2][2];
#pragma unroll
                    for (int n = 0; n < 2; n++) kv4_pieces(x[n][jj], s, hi[n], lo[n]);
                    qf[(j * 2 + s) * 32] = make_uint4(hi[0][0], hi[1][0], hi[0][1], hi[1][1]);
                    qf[((NG + j) * 2 + s) * 32] = make_uint4(lo[0][0], lo[1][0], lo[0][1], lo[1][1]);
                }
            }
        }
        return;
    }
    // heads wparts apart; a thread has eight values of a row, twice ahead of their use
    constexpr int OCTS = HD / 8;
    const int keys = (p.wparts > 1 ? 1 : p.c.n_kv) * OCTS;     // wparts: 1, or the KV heads
    for (int e0 = tid; e0 < 2 * keys; e0 += 256) {
        float x[2][8];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int e = e0 + u * 128, f = e < keys ? e : e - keys;
            if (e < 2 * keys) kv4_load_eight(x[u], (e < keys ? p.w.k : p.w.v) + ((size_t)b0 * p.c.n_kv + part + f / OCTS * p.wparts) * HD + f % OCTS * 8);
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int e = e0 + u * 128, f = e < keys ? e : e - keys;
            if (e < 2 * keys) kv4_write_eight<NG>(p.c, x[u], e < keys, part + f / OCTS * p.wparts, row0 + b0, f % OCTS * 8, p.w.rotate ? turn : nullptr);
        }
    }
}

// The values that the cache holds: a thread has a word of eight codes of a key row and the word at the same place of the value row, a block as many whole positions as it
// has threads for. 2048 rows of 8 heads of 128 values 5.4 us, of which the bytes are 2.9; 8192 rows 15.5 of 11.7.
template <int NG>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4 c, float* __restrict__ k, float* __restrict__ v, int row0, int n) {
    constexpr int WORDS = 4 * NG;
    pdl_launch_dependents();
    pdl_wait();
    const int per_row = c.n_kv * WORDS, at_once = max(1, 256 / per_row), own = at_once > 1 ? threadIdx.x / per_row : 0;
    const bool vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
    if (own >= at_once) return;
    auto put = [&](float* to, uint32_t codes, float s) {      // the four lowest codes: under the exponent of 2^23 a code n is the float 2^23 + n
        float x[4];
#pragma unroll
        for (int u = 0; u < 4; u++) x[u] = (__uint_as_float((codes >> (4 * u) & 15u) | 0x4B000000u) - 8388616.0f) * s;
        if (vec) *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
        else { to[0] = x[0]; to[1] = x[1]; to[2] = x[2]; to[3] = x[3]; }
    };
    for (long b = (long)blockIdx.x * at_once + own; b < n; b += (long)gridDim.x * at_once)
        for (int i = threadIdx.x - own * per_row; i < per_row; i += 256) {
            const int h = i / WORDS, w = i % WORDS;
            const size_t row = c.row(h, row0 + (int)b), out = ((size_t)b * c.n_kv + h) * (32 * NG);
            const uint32_t kw = __ldcg(reinterpret_cast<const uint32_t*>(c.k) + row * WORDS + w), vw = __ldcg(reinterpret_cast<const uint32_t*>(c.v) + row * WORDS + w);
            const __half* sc = c.scale + row * 2 * NG;
            const int j = w % NG, t = w / NG, u0 = 2 * w, u1 = 2 * w + 1;              // the key's group and piece; the value row's units of four codes
            const float ks = scale_at(sc + j), v0 = scale_at(sc + NG + u0 % NG), v1 = scale_at(sc + NG + u1 % NG);
            put(k + out + 32 * j + 8 * t, kw, ks);
            put(k + out + 32 * j + 8 * t + 4, kw >> 16, ks);
            put(v + out + 32 * (u0 % NG) + 4 * (u0 / NG), vw, v0);
            put(v + out + 32 * (u1 % NG) + 4 * (u1 / NG), vw >> 16, v1);
        }
}

// weights as whole numbers in the order of the choice: larger weight first, NaN last, the two zeros equal
__device__ __forceinline__ uint32_t weight_order(float w) {
    const uint32_t u = __float_as_uint(w);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
    if ((u << 1) == 0u) return 0x80000000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The choice: the `want` rows of [lo, hi) with the largest weights, equal ones from the lowest row, beside all rows outside it, in ascending
// order into kept[]. A cluster of CS blocks per KV head, block r with the r-th part of the rows, a thread with `per` neighbouring ones, in registers up to KEYS (0: read again every time).
// The bound is found eight bits at a time: every block counts its rows by those bits, and adds up the blocks' counts for itself; one barrier of
// the cluster a round, since each round has counters of its own. MOVE: the block then copies its kept rows into another cache.
// Bound by latency: a round is a meeting, the blocks' counts and a scan, 1.5 us, and there are three of them mostly (rows with equal bits that all stay end it):
// 9.7 us for 4096 rows of 8 heads to 1024, 19 for 65529 to 8192. (32 rounds of one bit by one block a head, every weight read again each time: 330.) Keys in
// registers: 131071 rows 23 us, 50 with the weights read every time; one a thread where that is enough: 4096 rows 9.7 us, 10.9 with room for eight.
constexpr int CH_THREADS = 1024, CH_CLUSTER = 8;
// Kept rows of a block times their values up to which the choosing launch copies them: 4096 rows of 8 heads of 128 values to 1024 take 9.7 us, 10.4 with a launch of its own; 65529 to
// 40000 42.7 and 37.4; 65529 rows of one head to 20000 25.1 and 16.7.
constexpr long CH_MOVE = 65536;
// rows list[i0..i1-1] (list NULL: i0..i1-1) of a head to rows i0..i1-1 of another cache, by a block; two pieces a thread on their way at a time
__device__ __forceinline__ void move_rows(const Kv4& src, const Kv4& dst, int h, const int32_t* list, long i0, long i1) {
    const int ng = src.hd / 32, tid = threadIdx.x, piece = tid % ng, at_once = CH_THREADS / ng;
    if (tid >= at_once * ng) return;
    for (i0 += tid / ng; i0 < i1; i0 += 2 * at_once) {
        uint4 vk[2], vv[2];
        uint32_t vs[2];
        float vw[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const long i = i0 + u * at_once;
            if (i >= i1) break;
            const size_t from = src.row(h, list ? __ldcg(list + i) : (int)i);
            vk[u] = __ldcg(reinterpret_cast<const uint4*>(src.k) + from * ng + piece);
            vv[u] = __ldcg(reinterpret_cast<const uint4*>(src.v) + from * ng + piece);
            vs[u] = __ldcg(reinterpret_cast<const uint32_t*>(src.scale) + from * ng + piece);
            vw[u] = piece == 0 ? __ldcg(src.weight + from) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const long i = i0 + u * at_once;
            if (i >= i1) break;
            const size_t to = dst.row(h, (int)i);
            reinterpret_cast<uint4*>(dst.k)[to * ng + piece] = vk[u];
            reinterpret_cast<uint4*>(dst.v)[to * ng + piece] = vv[u];
            reinterpret_cast<uint32_t*>(dst.scale)[to * ng + piece] = vs[u];
            if (piece == 0 && dst.weight) dst.weight[to] = vw[u];
        }
    }
}
template <int KEYS, bool MOVE>
__global__ void __launch_bounds__(CH_THREADS) kv4_choose_kernel(Kv4 src, Kv4 dst, int32_t* __restrict__ kept, int rows, int keep, int lo, int hi, int want, int CS) {
    __shared__ uint32_t hist[4][256], total[256], totals[2], found[3];
    __shared__ uint32_t warp_gt[32], warp_eq[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = blockIdx.x % CS, h = blockIdx.x / CS;
    for (int i = tid; i < 1024; i += CH_THREADS) (&hist[0][0])[i] = 0;
    pdl_launch_dependents();
    pdl_wait();
    auto meet = [&]() { if (CS > 1) { cluster_arrive(); cluster_wait(); } else __syncthreads(); };
    auto theirs = [&](const uint32_t* mine, int r) { return CS > 1 ? peer_load_u32(smem_u32(mine), (uint32_t)r) : *mine; };
    const int slice = (rows + CS - 1) / CS, per = (slice + CH_THREADS - 1) / CH_THREADS;
    const int r0 = rank * slice + tid * per, n = max(0, min(min(per, slice - tid * per), rows - r0));
    const float* w = src.weight + src.row(h, 0);
    uint32_t key[KEYS ? KEYS : 1];
    if constexpr (KEYS > 0) {
#pragma unroll
        for (int i = 0; i < KEYS; i += 4) {
            if (KEYS >= 4 && i + 4 <= n && ((uintptr_t)(w + r0) & 15) == 0) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(w + r0 + i));
                key[i] = weight_order(x.x); key[i + 1] = weight_order(x.y); key[i + 2] = weight_order(x.z); key[i + 3] = weight_order(x.w);
            } else {
#pragma unroll
                for (int u = 0; u < 4; u++) if (i + u < KEYS) key[i + u] = i + u < n ? weight_order(__ldcg(w + r0 + i + u)) : 0u;
            }
        }
    }
    // f(row, order, whether the row is one of those chosen from) for this thread's rows in order
    auto each = [&](auto f) {
        if constexpr (KEYS > 0) {
#pragma unroll
            for (int i = 0; i < KEYS; i++) if (i < n) f(r0 + i, key[i], r0 + i >= lo && r0 + i < hi);
        } else {
            for (int i0 = 0; i0 < n; i0 += 8) {                // eight on their way at a time
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = i0 + i < n ? __ldcg(w + r0 + i0 + i) : 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) if (i0 + i < n) f(r0 + i0 + i, weight_order(x[i]), r0 + i0 + i >= lo && r0 + i0 + i < hi);
            }
        }
    };
    uint32_t bound = 0, left = (uint32_t)want;                // rows still to be found among those that share the bound's bits so far
    __syncthreads();
    if (want > 0) {
        for (int round = 0; round < 4; round++) {
            const int shift = 24 - 8 * round;
            const uint32_t above = round ? 0xFFFFFFFFu << (shift + 8) : 0u;
            each([&](int, uint32_t k, bool in) { if (in && (k & above) == bound) atomicAdd(&hist[round][(k >> shift) & 255], 1u); });
            meet();
            if (tid < 256) {
                uint32_t t[CH_CLUSTER], sum = 0;               // all on their way at once
#pragma unroll
                for (int r = 0; r < CH_CLUSTER; r++) t[r] = r < CS ? theirs(&hist[round][tid], r) : 0u;
#pragma unroll
                for (int r = 0; r < CH_CLUSTER; r++) sum += t[r];
                total[tid] = sum;
            }
            __syncthreads();
            if (warp == 0) {                                  // lane l has bins 255 - 8 l .. 248 - 8 l
                uint32_t c[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) { c[i] = total[255 - 8 * lane - i]; sum += c[i]; }
                uint32_t before = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) { const uint32_t v = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += v; }
                before -= sum;
                if (before < left && before + sum >= left) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        if (before < left && before + c[i] >= left) { found[0] = 255 - 8 * lane - i; found[1] = before; found[2] = c[i]; }
                        before += c[i];
                    }
                }
            }
            __syncthreads();
            bound |= found[0] << shift;
            left -= found[1];
            if (found[2] == left && bound) {                  // all rows with these bits stay, whatever their other bits are: the same for every block
                bound--;
                left = 0;
                break;
            }
        }
    }
    // left: rows at the bound that stay, from the lowest. Who stays, and where it goes:
    uint32_t gt = 0, eq = 0;
    each([&](int, uint32_t k, bool in) { gt += !in || (want > 0 && k > bound); eq += in && want > 0 && k == bound; });
    uint32_t pgt = gt, peq = eq;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, pgt, o), b = __shfl_up_sync(0xffffffffu, peq, o);
        if (lane >= o) { pgt += a; peq += b; }
    }
    if (lane == 31) { warp_gt[warp] = pgt; warp_eq[warp] = peq; }
    __syncthreads();
    if (warp == 0) {
        uint32_t a = warp_gt[lane], b = warp_eq[lane];
        const uint32_t a0 = a, b0 = b;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
            if (lane >= o) { a += x; b += y; }
        }
        warp_gt[lane] = a - a0; warp_eq[lane] = b - b0;
        if (lane == 31) { totals[0] = a; totals[1] = b; }
    }
    meet();
    __syncthreads();
    uint32_t base = 0, eq_before = 0;                         // kept rows of the blocks below, and their rows at the bound
    uint32_t g[CH_CLUSTER], e[CH_CLUSTER];
#pragma unroll
    for (int r = 0; r < CH_CLUSTER; r++) { g[r] = r < rank ? theirs(&totals[0], r) : 0u; e[r] = r < rank ? theirs(&totals[1], r) : 0u; }
#pragma unroll
    for (int r = 0; r < CH_CLUSTER; r++) {
        base += g[r] + min(e[r], left - min(left, eq_before));
        eq_before += e[r];
    }
    const uint32_t room = left - min(left, eq_before);        // rows at the bound that stay in this block
    uint32_t at_gt = warp_gt[warp] + pgt - gt, at_eq = warp_eq[warp] + peq - eq;
    int32_t* mine = kept + (size_t)h * keep;
    each([&](int r, uint32_t k, bool in) {
        const bool sure = !in || (want > 0 && k > bound), tie = in && want > 0 && k == bound;
        if (sure || (tie && at_eq < room)) mine[base + at_gt + min(at_eq, room)] = r;
        at_gt += sure;
        at_eq += tie;
    });
    if (CS > 1) { cluster_arrive(); cluster_wait(); }         // nobody needs another block's shared memory any more, and the list is whole
    else __syncthreads();
    if (MOVE) move_rows(src, dst, h, mine, (long)keep * rank / CS, (long)keep * (rank + 1) / CS);        // equal parts of the list (the last rows, which all stay, would otherwise fall to the last block)
}

// The same copy by all SMs, where there is much of it. kept NULL: rows 0..keep-1. grid (parts, KV heads)
__global__ void __launch_bounds__(CH_THREADS) kv4_move_kernel(Kv4 src, Kv4 dst, const int32_t* __restrict__ kept, int keep) {
    pdl_launch_dependents();
    pdl_wait();
    const int h = blockIdx.y;
    move_rows(src, dst, h, kept ? kept + (size_t)h * keep : nullptr, (long)keep * blockIdx.x / gridDim.x, (long)keep * (blockIdx.x + 1) / gridDim.x);
}

Kv4 planes(const ibcu_kv4_t* t) { return Kv4{ t->k, t->v, (__half*)t->scale, t->weight, t->n_kv_heads, t->head_dim, t->max_rows }; }

int check_cache(ibcu_ctx* ctx, const ibcu_kv4_t* t, const char* call) {
    IBCU_REQUIRE(ctx, t && t->k && t->v && t->scale, "%s: null pointer", call);
    const int hd = t->head_dim;
    IBCU_REQUIRE(ctx, hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 192 || hd == 256, "%s: head_dim=%d (32, 64, 96, 128, 192 or 256)", call, hd);
    IBCU_REQUIRE(ctx, t->n_kv_heads >= 1 && t->n_kv_heads <= 1024 && t->max_rows >= 8 && t->max_rows <= (1 << 30) && t->max_rows % 8 == 0, "%s: n_kv_heads=%d max_rows=%d (rows in multiples of 8, up to 2^30)", call, t->n_kv_heads, t->max_rows);
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

}  // namespace

int kv4_prepare(ibcu_ctx* ctx, const Kv4& c, const Kv4Columns& t, const Kv4Place& at, const Kv4Prep& w) {
    PrepParams p = { c, t, at, w, 0, std::min(c.n_kv, (4 * ctx->sm_count + t.ntiles - 1) / t.ntiles), t.B <= 8 ? c.n_kv : 1, ctx->kern_err };
    if (w.q) p.qblocks = p.qparts * t.ntiles;
    const int nb = w.q ? std::min(16, 15 / t.group + 2) : 1;  // positions that a block may have to do with
    const size_t smem = w.rotate ? (size_t)nb * c.hd / 2 * sizeof(double2) : 0;
    auto kern = c.hd == 32 ? kv4_prep_kernel<1> : c.hd == 64 ? kv4_prep_kernel<2> : c.hd == 96 ? kv4_prep_kernel<3> : c.hd == 128 ? kv4_prep_kernel<4> : c.hd == 192 ? kv4_prep_kernel<6> : kv4_prep_kernel<8>;
    return ibcu_launch(ctx, kern, dim3(p.qblocks + (w.k ? t.B * p.wparts : 0)), dim3(128), smem, 1, true, p);
}

extern "C" int ibcu_kv4_write(ibcu_ctx* ctx, const ibcu_kv4_t* cache, const float* k, const float* v, int row0, int pos0, int B, float theta) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_cache(ctx, cache, "ibcu_kv4_write")) return rc;
    IBCU_REQUIRE(ctx, k && v, "ibcu_kv4_write: null pointer");
    if (int rc = check_rows(ctx, cache, row0, B, "ibcu_kv4_write")) return rc;
    if (int rc = check_rotation(ctx, pos0, B, theta, "ibcu_kv4_write")) return rc;
    return kv4_prepare(ctx, planes(cache), Kv4Columns{ cache->n_kv_heads, 1, B, 0, 1 }, Kv4Place{ row0, pos0, nullptr }, Kv4Prep{ nullptr, k, v, nullptr, nullptr, log2_of(theta), theta > 0.0f });
}

extern "C" int ibcu_kv4_read(ibcu_ctx* ctx, const ibcu_kv4_t* cache, float* k, float* v, int row0, int n) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_cache(ctx, cache, "ibcu_kv4_read")) return rc;
    IBCU_REQUIRE(ctx, k && v, "ibcu_kv4_read: null pointer");
    if (int rc = check_rows(ctx, cache, row0, n, "ibcu_kv4_read")) return rc;
    const int per_row = cache->n_kv_heads * (cache->head_dim / 8), at_once = std::max(1, 256 / per_row), hd = cache->head_dim;
    auto kern = hd == 32 ? kv4_read_kernel<1> : hd == 64 ? kv4_read_kernel<2> : hd == 96 ? kv4_read_kernel<3> : hd == 128 ? kv4_read_kernel<4> : hd == 192 ? kv4_read_kernel<6> : kv4_read_kernel<8>;
    return ibcu_launch(ctx, kern, dim3((int)std::min(((long)n + at_once - 1) / at_once, 16L * ctx->sm_count)), dim3(256), 0, 1, true, planes(cache), k, v, row0, n);
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
    return kv4_attend(ctx, planes(cache), cache->decay, Kv4Place{ row0, 0, nullptr }, q, nullptr, nullptr, out, n_heads, B, 0.0, 0);
}

extern "C" int ibcu_attention_decode_kv4(ibcu_ctx* ctx, const ibcu_kv4_t* cache, const float* q, const float* k, const float* v, float* out,
                                         int n_heads, int row0, int pos0, int B, float theta) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_cache(ctx, cache, "ibcu_attention_decode_kv4")) return rc;
    IBCU_REQUIRE(ctx, q && k && v && out, "ibcu_attention_decode_kv4: null pointer");
    if (int rc = check_rows(ctx, cache, row0, B, "ibcu_attention_decode_kv4")) return rc;
    if (int rc = check_heads(ctx, cache, n_heads, B, "ibcu_attention_decode_kv4")) return rc;
    if (int rc = check_rotation(ctx, pos0, B, theta, "ibcu_attention_decode_kv4")) return rc;
    return kv4_attend(ctx, planes(cache), cache->decay, Kv4Place{ row0, pos0, nullptr }, q, k, v, out, n_heads, B, log2_of(theta), theta > 0.0f);
}

extern "C" int ibcu_attention_decode_kv4_at(ibcu_ctx* ctx, const ibcu_kv4_t* cache, const float* q, const float* k, const float* v, float* out,
                                            int n_heads, const int* at_dev, int B, float theta) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_cache(ctx, cache, "ibcu_attention_decode_kv4_at")) return rc;
    IBCU_REQUIRE(ctx, q && k && v && out && at_dev, "ibcu_attention_decode_kv4_at: null pointer");
    if (int rc = check_rows(ctx, cache, 0, B, "ibcu_attention_decode_kv4_at")) return rc;
    if (int rc = check_heads(ctx, cache, n_heads, B, "ibcu_attention_decode_kv4_at")) return rc;
    if (int rc = check_rotation(ctx, 0, B, theta, "ibcu_attention_decode_kv4_at")) return rc;
    return kv4_attend(ctx, planes(cache), cache->decay, Kv4Place{ 0, 0, at_dev }, q, k, v, out, n_heads, B, log2_of(theta), theta > 0.0f);
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
    const bool in_place = src->k == dst->k;
    IBCU_REQUIRE(ctx, in_place ? src->v == dst->v && src->scale == dst->scale && src->weight == dst->weight && src->max_rows == dst->max_rows
                               : src->v != dst->v && src->scale != dst->scale && src->weight != dst->weight, "ibcu_kv4_evict: two caches that share some planes");
    // In place the kept rows go by way of scratch.
    Kv4 to = planes(dst);
    const bool by_way = in_place && keep < rows;
    auto round_up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    const size_t held = (size_t)nkv * keep, b_kept = kept ? 0 : round_up(held * sizeof(int32_t)), row_bytes = src->head_dim / 2, b_plane = round_up(held * row_bytes), b_scale = round_up(held * src->head_dim / 8);
    if (int rc = ibcu_reserve(ctx, &ctx->scratch, &ctx->scratch_bytes, b_kept + (by_way ? 2 * b_plane + b_scale + held * sizeof(float) : 0))) return rc;
    char* s = (char*)ctx->scratch;
    if (!kept) kept = (int32_t*)s;
    if (by_way) {
        s += b_kept;
        to.k = (uint8_t*)s; to.v = (uint8_t*)(s + b_plane); to.scale = (__half*)(s + 2 * b_plane); to.weight = (float*)(s + 2 * b_plane + b_scale);
        to.max_rows = keep;
    }
    // A block a thousand rows, up to eight, as long as all clusters run at once: 12 of eight blocks, 33 of four, 74 of two find their places (8192 rows of 32 heads
    // by eight blocks each 38 us, by four 14).
    int CS = 1;
    while (CS < CH_CLUSTER && rows > 1024 * CS && nkv <= (CS == 4 ? ctx->sm_count / 12 : CS == 2 ? ctx->sm_count * 9 / 40 : ctx->sm_count / 2)) CS *= 2;
    const bool move = !in_place || by_way, here = move && (long)keep / CS * src->head_dim <= CH_MOVE;
    const int per = ((rows + CS - 1) / CS + CH_THREADS - 1) / CH_THREADS;
    auto pick = [&](auto with, auto without) { return here ? with : without; };
    auto choose = per <= 1 ? pick(kv4_choose_kernel<1, true>, kv4_choose_kernel<1, false>) : per <= 8 ? pick(kv4_choose_kernel<8, true>, kv4_choose_kernel<8, false>)
                : per <= 16 ? pick(kv4_choose_kernel<16, true>, kv4_choose_kernel<16, false>) : pick(kv4_choose_kernel<0, true>, kv4_choose_kernel<0, false>);
    int rc = ibcu_launch(ctx, choose, dim3(CS * nkv), dim3(CH_THREADS), 0, CS, true, planes(src), to, kept, rows, keep, sink, rows - recent, keep - sink - recent, CS);
    const dim3 grid((unsigned)std::max(1, std::min(2 * ctx->sm_count / nkv, (keep + 255) / 256)), nkv);
    if (!rc && move && !here) rc = ibcu_launch(ctx, kv4_move_kernel, grid, dim3(CH_THREADS), 0, 1, true, planes(src), to, (const int32_t*)kept, keep);
    if (!rc && by_way) rc = ibcu_launch(ctx, kv4_move_kernel, grid, dim3(CH_THREADS), 0, 1, true, to, planes(dst), (const int32_t*)nullptr, keep);
    return rc;
}
