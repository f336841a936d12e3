// Short causal depthwise convolution over time-major sequences (the mixing step in front of the state-space scan):
//   pre[t, d] = bias[d] + sum_k w[d, k] x[t - W + 1 + k, d],   y = silu(pre) (or pre),   2 <= W <= 4
// Steps before the first come from state_in [B, W - 1, D]; a set reset flag at t cuts every tap from t on off from the steps
// before t; steps from lengths[b] on are not read and write zeros.
//
// A thread owns one channel of one row and walks SEG steps with the last W - 1 inputs in registers.
#include "ssm_math.h"

#define SEG 16

struct ConvArgs {        // mirrored by ops/hip.py (_conv_args): 64-bit words in this order
    const void *x, *state_in;
    long long x_t, x_b;
    const float *w, *bias;
    const unsigned char* reset;
    const int* lengths;
    void *y, *state_out;
    long long y_t, y_b, T, B, D, W, silu;
    // backward
    const void *dy, *dstate_out;
    long long dy_t, dy_b;
    void *dx, *dstate_in;
    long long dx_t, dx_b;
    float *dw, *db, *ws;
    long long ws_n;
};

__device__ __forceinline__ int row_end(const ConvArgs& p, int b) {
    return p.lengths ? max(0, min(p.lengths[b], (int)p.T)) : (int)p.T;
}
// input row of time t (t < 0: the carried state)
template <typename T, int W>
__device__ __forceinline__ float input(const ConvArgs& p, int b, int t, int d) {
    if (t >= 0) return ld((const T*)p.x + t * p.x_t + b * p.x_b + d);
    return p.state_in ? ld((const T*)p.state_in + ((long long)b * (W - 1) + (t + W - 1)) * p.D + d) : 0.f;
}
__device__ __forceinline__ bool resets(const ConvArgs& p, int b, int t) { return t >= 0 && p.reset && p.reset[(long long)t * p.B + b] != 0; }

// xw = the inputs of times ta - W + 1 .. ta - 1, as a step at ta - 1 leaves them (resets applied); end > ta - 1
template <typename T, int W>
__device__ __forceinline__ void window(const ConvArgs& p, int b, int ta, int d, float (&xw)[W]) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        const int t = ta - W + 1 + k;
        if (resets(p, b, t)) {
#pragma unroll
            for (int q = 0; q < k; ++q) xw[q] = 0.f;
        }
        xw[k] = input<T, W>(p, b, t, d);
    }
}

template <typename T, int W>
__global__ __launch_bounds__(256) void k_conv_fwd(ConvArgs p) {
    const int d = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y, ta = blockIdx.z * SEG;
    if (d >= p.D) return;
    const int end = row_end(p, b), tb = min(ta + SEG, (int)p.T);
    float w[W], xw[W];
#pragma unroll
    for (int k = 0; k < W; ++k) w[k] = p.w[(long long)d * W + k];
    const float bias = p.bias ? p.bias[d] : 0.f;
    if (ta <= end) window<T, W>(p, b, ta, d, xw);
    for (int t = ta; t <= tb; ++t) {
        // the state a row leaves: the segment that holds its last step (the first one, for an empty row) writes it
        if (t == end && (t > ta || t == 0) && p.state_out) {
#pragma unroll
            for (int k = 0; k < W - 1; ++k) st((T*)p.state_out + ((long long)b * (W - 1) + k) * p.D + d, xw[k]);
        }
        if (t == tb) break;
        float v = 0.f;
        if (t < end) {
            if (resets(p, b, t)) {
#pragma unroll
                for (int k = 0; k < W - 1; ++k) xw[k] = 0.f;
            }
            xw[W - 1] = input<T, W>(p, b, t, d);
            v = bias;
#pragma unroll
            for (int k = 0; k < W; ++k) v = fmaf(w[k], xw[k], v);
            if (p.silu) v *= sigmoidf(v);
#pragma unroll
            for (int k = 0; k < W - 1; ++k) xw[k] = xw[k + 1];
        }
        st((T*)p.y + t * p.y_t + b * p.y_b + d, v);
    }
}

// dx[tau] collects w[k] dpre[tau + W - 1 - k]: one walk forward in time with W open sums. A segment emits the steps
// ta .. tb - 1 and runs W - 1 steps further for them; dw and db count its own steps only.
template <typename T, int W>
__global__ __launch_bounds__(256) void k_conv_bwd(ConvArgs p, float* __restrict__ part) {
    const int d = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y, ta = blockIdx.z * SEG;
    if (d >= p.D) return;
    const int end = row_end(p, b), tb = min(ta + SEG, (int)p.T);
    float w[W], xw[W], open[W], dw[W], db = 0.f;
    bool live[W];                                     // the window's step belongs to the current episode
#pragma unroll
    for (int k = 0; k < W; ++k) { w[k] = p.w[(long long)d * W + k]; open[k] = 0.f; dw[k] = 0.f; live[k] = true; xw[k] = 0.f; }
    const float bias = p.bias ? p.bias[d] : 0.f;
    if (ta < end) {
        window<T, W>(p, b, ta, d, xw);
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {             // a reset at a window step cuts the ones before it
            if (resets(p, b, ta - W + 1 + k)) {
#pragma unroll
                for (int q = 0; q < k; ++q) live[q] = false;
            }
        }
    }
    for (int t = ta; t < tb + W - 1; ++t) {
        if (t < end) {
            if (resets(p, b, t)) {
#pragma unroll
                for (int k = 0; k < W - 1; ++k) { xw[k] = 0.f; live[k] = false; }
            }
            xw[W - 1] = input<T, W>(p, b, t, d);
            live[W - 1] = true;
            float v = bias;
#pragma unroll
            for (int k = 0; k < W; ++k) v = fmaf(w[k], xw[k], v);
            float g = ld((const T*)p.dy + t * p.dy_t + b * p.dy_b + d);
            if (p.silu) { const float s = sigmoidf(v); g *= s * fmaf(v, 1.f - s, 1.f); }
            if (t < tb) {
#pragma unroll
                for (int k = 0; k < W; ++k) dw[k] = fmaf(g, xw[k], dw[k]);
                db += g;
            }
#pragma unroll
            for (int k = 0; k < W; ++k) if (live[k]) open[k] = fmaf(w[k], g, open[k]);
        } else if (t == end && p.dstate_out) {        // the state the row left = its last W - 1 inputs: their gradient comes in here
#pragma unroll
            for (int k = 0; k < W - 1; ++k)
                if (live[k]) open[k] += ld((const T*)p.dstate_out + ((long long)b * (W - 1) + k) * p.D + d);
        }
        const int tau = t - W + 1;                    // complete: no later step reaches back to it
        if (tau < 0) {
            if (p.dstate_in && ta == 0) st((T*)p.dstate_in + ((long long)b * (W - 1) + tau + W - 1) * p.D + d, open[0]);
        } else if (tau >= ta) {
            st((T*)p.dx + tau * p.dx_t + b * p.dx_b + d, open[0]);
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k) { xw[k] = xw[k + 1]; open[k] = open[k + 1]; live[k] = live[k + 1]; }
        open[W - 1] = 0.f;
    }
    float* q = part + ((long long)blockIdx.z * p.B + b) * (W + 1) * p.D + d;
#pragma unroll
    for (int k = 0; k < W; ++k) q[k * p.D] = dw[k];
    q[W * p.D] = db;
}

__global__ void k_conv_sum(const float* __restrict__ part, int R, int W, long long D, float* __restrict__ dw, float* __restrict__ db) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (W + 1) * D) return;
    const long long k = i / D, d = i - k * D;
    float v = 0.f;
    for (int r = 0; r < R; ++r) v += part[r * (W + 1) * D + i];
    if (k < W) dw[d * W + k] = v;
    else if (db) db[d] = v;
}

template <typename T, int W>
__global__ __launch_bounds__(256) void k_conv_step(ConvArgs p) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.B * p.D) return;
    const long long b = i / p.D, d = i - b * p.D;
    T* s = (T*)p.state_out + b * (W - 1) * p.D + d;
    const bool rs = p.reset && p.reset[b] != 0;
    const T* xp = (const T*)p.x + b * p.x_b + d;
    T row[W];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) row[k] = rs ? (T)0 : s[k * p.D];
    row[W - 1] = *xp;
    float v = p.bias ? p.bias[d] : 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) v = fmaf(p.w[d * W + k], ld(&row[k]), v);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) s[k * p.D] = row[k + 1];
    if (p.silu) v *= sigmoidf(v);
    st((T*)p.y + b * p.y_b + d, v);
}

#define CONV_W(NAME, T, GRID, ...)                                             \
    switch (p.W) {                                                              \
        case 2: NAME<T, 2><<<GRID, 256, 0, s>>>(__VA_ARGS__); break;            \
        case 3: NAME<T, 3><<<GRID, 256, 0, s>>>(__VA_ARGS__); break;            \
        default: NAME<T, 4><<<GRID, 256, 0, s>>>(__VA_ARGS__); break;           \
    }

static bool conv_ok(long long T, long long B, long long D, long long W) {
    return T > 0 && T <= 65535ll * SEG && B > 0 && B <= 65535 && D > 0 && D < (1ll << 31) && W >= 2 && W <= 4;
}

// floats of scratch of a backward pass
DRL_API int drl_short_conv_ws(long long T, long long B, long long D, long long W, long long* n) {
    if (!conv_ok(T, B, D, W)) return -1;
    *n = (T + SEG - 1) / SEG * B * (W + 1) * D;
    return 0;
}

DRL_API int drl_short_conv_fwd(const ConvArgs* a, int bf16, hipStream_t s) {
    const ConvArgs p = *a;
    if (!conv_ok(p.T, p.B, p.D, p.W)) return -1;
    const dim3 grid((unsigned)((p.D + 255) / 256), (unsigned)p.B, (unsigned)((p.T + SEG - 1) / SEG));
    if (bf16) { CONV_W(k_conv_fwd, bf16_t, grid, p) } else { CONV_W(k_conv_fwd, float, grid, p) }
    return (int)hipGetLastError();
}

DRL_API int drl_short_conv_bwd(const ConvArgs* a, int bf16, hipStream_t s) {
    const ConvArgs p = *a;
    long long need;
    if (drl_short_conv_ws(p.T, p.B, p.D, p.W, &need)) return -1;
    if (p.ws_n < need) return -2;
    const dim3 grid((unsigned)((p.D + 255) / 256), (unsigned)p.B, (unsigned)((p.T + SEG - 1) / SEG));
    if (bf16) { CONV_W(k_conv_bwd, bf16_t, grid, p, p.ws) } else { CONV_W(k_conv_bwd, float, grid, p, p.ws) }
    const long long n = (p.W + 1) * p.D;
    k_conv_sum<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(p.ws, (int)(grid.z * p.B), (int)p.W, p.D, p.dw, p.db);
    return (int)hipGetLastError();
}

DRL_API int drl_short_conv_step(const ConvArgs* a, int bf16, hipStream_t s) {
    const ConvArgs p = *a;
    if (!conv_ok(1, 1, p.D, p.W) || p.B <= 0) return -1;
    const long long nb = (p.B * p.D + 255) / 256;
    if (nb > 0x7fffffffll) return -1;
    const dim3 grid((unsigned)nb);
    if (bf16) { CONV_W(k_conv_step, bf16_t, grid, p) } else { CONV_W(k_conv_step, float, grid, p) }
    return (int)hipGetLastError();
}
