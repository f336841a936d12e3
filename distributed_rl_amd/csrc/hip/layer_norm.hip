// Layer norm over the last axis and its backward pass.
//   y = (x - mean) rstd w + b;   dx = rstd (dn - mean(dn) - n mean(dn n)), n = (x - mean) rstd, dn = dy w
//   dw = sum over rows of dy n,  db = sum over rows of dy
// The variance is summed around the mean, not as E[x^2] - mean^2, which cancels for rows far from zero.
#include "ssm_math.h"

struct NormArgs {        // mirrored by ops/hip.py (_norm_args): 64-bit words in this order
    const void* x; long long x_r;
    const float *w, *b;
    void* y; long long y_r;
    float *mean, *rstd;
    long long M, D;
    const void* dy; long long dy_r;
    void* dx; long long dx_r;
    float *dw, *db, *ws;
    long long ws_n;
};

template <typename T>
__global__ __launch_bounds__(256) void k_norm_fwd(NormArgs p, float eps) {
    __shared__ float red[17];
    const long long r = blockIdx.x;
    const T* x = (const T*)p.x + r * p.x_r;
    float a = 0.f;
    for (long long c = threadIdx.x; c < p.D; c += 256) a += ld(x + c);
    const float mean = block_sum(a, red) / (float)p.D;
    a = 0.f;
    for (long long c = threadIdx.x; c < p.D; c += 256) { const float v = ld(x + c) - mean; a = fmaf(v, v, a); }
    const float rstd = 1.0f / sqrtf(block_sum(a, red) / (float)p.D + eps);
    for (long long c = threadIdx.x; c < p.D; c += 256)
        st((T*)p.y + r * p.y_r + c, fmaf((ld(x + c) - mean) * rstd, p.w[c], p.b ? p.b[c] : 0.f));
    if (threadIdx.x == 0 && p.mean) { p.mean[r] = mean; p.rstd[r] = rstd; }
}

template <typename T>
__global__ __launch_bounds__(256) void k_norm_dx(NormArgs p) {
    __shared__ float red[17];
    const long long r = blockIdx.x;
    const T *x = (const T*)p.x + r * p.x_r, *dy = (const T*)p.dy + r * p.dy_r;
    const float mean = p.mean[r], rstd = p.rstd[r];
    float a = 0.f, c2 = 0.f;
    for (long long c = threadIdx.x; c < p.D; c += 256) {
        const float dn = ld(dy + c) * p.w[c];
        a += dn;
        c2 = fmaf(dn, (ld(x + c) - mean) * rstd, c2);
    }
    const float m1 = block_sum(a, red) / (float)p.D;
    const float m2 = block_sum(c2, red) / (float)p.D;
    for (long long c = threadIdx.x; c < p.D; c += 256) {
        const float n = (ld(x + c) - mean) * rstd;
        st((T*)p.dx + r * p.dx_r + c, (ld(dy + c) * p.w[c] - m1 - n * m2) * rstd);
    }
}

#define NORM_STRIPS 256
template <typename T>
__global__ __launch_bounds__(256) void k_norm_dw(NormArgs p) {
    const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
    if (c >= p.D) return;
    float dw = 0.f, db = 0.f;
    for (long long r = blockIdx.y; r < p.M; r += gridDim.y) {
        const float g = ld((const T*)p.dy + r * p.dy_r + c);
        dw = fmaf(g, (ld((const T*)p.x + r * p.x_r + c) - p.mean[r]) * p.rstd[r], dw);
        db += g;
    }
    p.ws[blockIdx.y * 2 * p.D + c] = dw;
    p.ws[blockIdx.y * 2 * p.D + p.D + c] = db;
}
__global__ void k_norm_sum(const float* __restrict__ part, int R, long long D, float* __restrict__ dw, float* __restrict__ db) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= 2 * D) return;
    float v = 0.f;
    for (int r = 0; r < R; ++r) v += part[r * 2 * D + i];
    if (i < D) dw[i] = v;
    else if (db) db[i - D] = v;
}

static bool norm_ok(long long M, long long D) { return M > 0 && M < (1ll << 31) && D > 0 && D <= 16384; }
static int norm_strips(long long M) { return M < NORM_STRIPS ? (int)M : NORM_STRIPS; }

DRL_API int drl_norm_ws(long long M, long long D, long long* n) {
    if (!norm_ok(M, D)) return -1;
    *n = 2 * D * norm_strips(M);
    return 0;
}

DRL_API int drl_norm_fwd(const NormArgs* a, int bf16, float eps, hipStream_t s) {
    const NormArgs p = *a;
    if (!norm_ok(p.M, p.D)) return -1;
    if (bf16) k_norm_fwd<bf16_t><<<(unsigned)p.M, 256, 0, s>>>(p, eps);
    else k_norm_fwd<float><<<(unsigned)p.M, 256, 0, s>>>(p, eps);
    return (int)hipGetLastError();
}

DRL_API int drl_norm_bwd(const NormArgs* a, int bf16, hipStream_t s) {
    const NormArgs p = *a;
    long long need;
    if (drl_norm_ws(p.M, p.D, &need)) return -1;
    if (p.ws_n < need) return -2;
    const int R = norm_strips(p.M);
    const dim3 grid((unsigned)((p.D + 255) / 256), R);
    if (bf16) { k_norm_dx<bf16_t><<<(unsigned)p.M, 256, 0, s>>>(p); k_norm_dw<bf16_t><<<grid, 256, 0, s>>>(p); }
    else { k_norm_dx<float><<<(unsigned)p.M, 256, 0, s>>>(p); k_norm_dw<float><<<grid, 256, 0, s>>>(p); }
    k_norm_sum<<<(unsigned)((2 * p.D + 255) / 256), 256, 0, s>>>(p.ws, R, p.D, p.dw, p.db);
    return (int)hipGetLastError();
}
