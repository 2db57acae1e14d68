// INT8 weights x INT8 activations with one scale per output row and one per token: a prompt's projections as integer products, any
// number of tokens. Sums are exact 32-bit integers, so a result does not depend on how the work is cut.
#include "common.cuh"

namespace {

// one block per token: scale = max|x| * (1 / 127), codes rint(x * (1 / scale)); columns N..ldq-1 of the codes are zero
__global__ void __launch_bounds__(256) quantize_rows_kernel(const float* __restrict__ x, int8_t* __restrict__ q, float* __restrict__ scale, int N, int ldq) {
    __shared__ uint32_t red[8];
    pdl_launch_dependents();
    pdl_wait();
    const size_t b = blockIdx.x;
    const float* xb = x + b * N;
    uint32_t m = 0;
    for (int i = threadIdx.x; i < N; i += 256) m = max(m, __float_as_uint(xb[i]) & 0x7FFFFFFFu);
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < 8; w++) m = max(m, red[w]);
    float s = __fmul_rn(__uint_as_float(m), 1.0f / 127.0f), inv = __fdiv_rn(1.0f, s);
    if (m < 0x0D800000u) { s = 0.0f; inv = 0.0f; }            // below 2^-100: zeros
    if (m >= 0x7F800000u) { s = __uint_as_float(0x7FFFFFFFu); inv = 0.0f; }      // NaN or Inf: all results of the token are NaN
    for (int i = threadIdx.x; i < ldq; i += 256) q[b * ldq + i] = i < N && inv > 0.0f ? (int8_t)(int)rintf(__fmul_rn(xb[i], inv)) : (int8_t)0;
    if (threadIdx.x == 0) scale[b] = s;
}

// a warp per output row and token
__global__ void __launch_bounds__(256) w8a8_kernel(ibcu_linear_t t, const int8_t* __restrict__ xq, const float* __restrict__ sx, int N, int ldq) {
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const size_t b = blockIdx.y;
    if (row >= t.M) return;
    const int8_t* w = (const int8_t*)t.w + (size_t)row * N;
    int sum = 0;
    for (int i = lane; i < N; i += 32) sum += (int)w[i] * (int)xq[b * ldq + i];
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) {
        const float sw = t.scales_fp32 ? ((const float*)t.scales)[row] : __half2float(((const __half*)t.scales)[row]);
        float* o = t.out + b * t.out_stride + row;
        const float y = (float)sum * (sw * sx[b]);
        *o = t.epilogue == IBCU_EPI_ADD ? *o + y : y;
    }
}

int check_call(ibcu_ctx* ctx, const ibcu_linear_t* ts, int n, int N, int B, const char* call) {
    IBCU_REQUIRE(ctx, ts && n >= 1 && n <= 4, "%s: %d tensors (1 to 4)", call, n);
    IBCU_REQUIRE(ctx, N >= 1 && N <= 131072 && B >= 1 && B <= (1 << 20), "%s: N=%d (up to 131072) B=%d (up to %d)", call, N, B, 1 << 20);
    for (int i = 0; i < n; i++) {
        IBCU_REQUIRE(ctx, ts[i].w && ts[i].scales && ts[i].out, "%s: null pointer", call);
        IBCU_REQUIRE(ctx, ts[i].M >= 1 && ts[i].out_stride >= ts[i].M, "%s: M=%d out_stride=%d", call, ts[i].M, ts[i].out_stride);
        IBCU_REQUIRE(ctx, ts[i].epilogue == IBCU_EPI_STORE || ts[i].epilogue == IBCU_EPI_ADD, "%s: epilogue=%d", call, ts[i].epilogue);
    }
    return IBCU_OK;
}

int product(ibcu_ctx* ctx, const ibcu_linear_t* ts, int n, const int8_t* xq, const float* sx, int N, int ldq, int B) {
    for (int i = 0; i < n; i++)
        for (int b = 0; b < B; b += 65535) {
            ibcu_linear_t t = ts[i];
            t.out += (size_t)b * t.out_stride;
            if (int rc = ibcu_launch(ctx, w8a8_kernel, dim3((t.M + 7) / 8, B - b < 65535 ? B - b : 65535), dim3(256), 0, 1, true, t, xq + (size_t)b * ldq, sx + b, N, ldq)) return rc;
        }
    return IBCU_OK;
}

}  // namespace

extern "C" int ibcu_quantize_rows_int8(ibcu_ctx* ctx, const float* x, int8_t* q, float* scale, int N, int B) {
    IBCU_CHECK_CTX(ctx);
    IBCU_REQUIRE(ctx, x && q && scale, "ibcu_quantize_rows_int8: null pointer");
    IBCU_REQUIRE(ctx, N >= 1 && B >= 1, "ibcu_quantize_rows_int8: N=%d B=%d", N, B);
    return ibcu_launch(ctx, quantize_rows_kernel, dim3(B), dim3(256), 0, 1, true, x, q, scale, N, N);
}

extern "C" int ibcu_linear_w8a8(ibcu_ctx* ctx, const ibcu_linear_t* tensors, int n_tensors, const int8_t* xq, const float* sx, int N, int B) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_call(ctx, tensors, n_tensors, N, B, "ibcu_linear_w8a8")) return rc;
    IBCU_REQUIRE(ctx, xq && sx, "ibcu_linear_w8a8: null pointer");
    return product(ctx, tensors, n_tensors, xq, sx, N, N, B);
}

extern "C" int ibcu_linear_w8a8_fp32(ibcu_ctx* ctx, const ibcu_linear_t* tensors, int n_tensors, const float* x, int N, int B) {
    IBCU_CHECK_CTX(ctx);
    if (int rc = check_call(ctx, tensors, n_tensors, N, B, "ibcu_linear_w8a8_fp32")) return rc;
    IBCU_REQUIRE(ctx, x, "ibcu_linear_w8a8_fp32: null pointer");
    const int ldq = (N + 15) & ~15;
    const size_t qb = ((size_t)B * ldq + 255) & ~(size_t)255;
    int rc = ibcu_reserve(ctx, &ctx->xpack, &ctx->xpack_bytes, qb + (size_t)B * sizeof(float));
    if (rc) return rc;
    int8_t* q = (int8_t*)ctx->xpack;
    float* sx = (float*)((char*)ctx->xpack + qb);
    rc = ibcu_launch(ctx, quantize_rows_kernel, dim3(B), dim3(256), 0, 1, true, x, q, sx, N, ldq);
    if (!rc) rc = product(ctx, tensors, n_tensors, q, sx, N, ldq, B);
    return rc;
}
