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
// kernels in tiles of 8 (all columns of a call, if they are no more than that) or of 16. A tile's queries lie in scratch as the A
// operand's fragments, two fp16 pieces of every value: [unit = KV head * tiles + tile][part][group of 32][step][half][lane] uint2. Tiles of 16 have two parts (high
// and low pieces), whose halves are columns 0-7 and 8-15; a tile of 8 has one, whose halves are the high and the low pieces.
// Beside them qc [unit][16]: the factor that turns a column's sums into exponents of 2.
struct Kv4Columns {
    int n_heads, group, B, large, ntiles;
    __host__ __device__ int cols() const { return large ? 16 : 8; }
};
__host__ __device__ constexpr size_t kv4_frag_uint2(int ng, bool large) { return (size_t)(large ? 2 : 1) * ng * 128; }     // of a unit

// where rows and positions of a call are: arguments, or {row0, pos0} in device memory
struct Kv4Place { int row0, pos0; const int* at; };
// Reads them where they are on the device. False, and the context's error word set, if the rows would not fit.
__device__ __forceinline__ bool kv4_place(const Kv4Place& p, int B, int max_rows, int* err, int& row0, int& pos0) {
    row0 = p.row0; pos0 = p.pos0;
    if (!p.at) return true;
    row0 = __ldcg(p.at); pos0 = __ldcg(p.at + 1);
    if (row0 >= 0 && pos0 >= 0 && row0 <= max_rows - B) return true;
    *err = IBCU_KV4_PLACE_ERR;
    return false;
}

// Prepares a call's queries (q != NULL) and writes its rows (k != NULL), one launch. Defined in kv4.cu.
struct Kv4Prep { const float *q, *k, *v; uint2* qf; float* qc; double log2_theta; int rotate; };
int kv4_prepare(ibcu_ctx* ctx, const Kv4& c, const Kv4Columns& t, const Kv4Place& at, const Kv4Prep& w);
// The attention of a call, with what it has to prepare. q, k, v as above (k NULL: the rows are there). Defined in kv4_attn.cu.
int kv4_attend(ibcu_ctx* ctx, const Kv4& c, float decay, const Kv4Place& at, const float* q, const float* k, const float* v, float* out, int n_heads, int B, double log2_theta, int rotate);
