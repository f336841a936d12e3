// Short causal depthwise convolution over time-major sequences (the mixing step in front of the state-space scan):
//   pre[t, d] = bias[d] + sum_k w[d, k] x[t - W + 1 + k, d],   y = silu(pre) (or pre),   2 <= W <= 4
// Steps before the first come from state_in [B, W - 1, D]; a set reset flag at t cuts every tap from t on off from the steps
// before t; steps from lengths[b] on are not read and write zeros.
//
// Bound by memory: a thread owns V neighbouring channels of one row (4 of fp32, 2 of bf16, at any alignment; 1 where there are
// fewer) and a run of steps, reads FB (BB) steps ahead and keeps the last W - 1 inputs in registers. The last vector ends at
// the last channel: the channels that it has twice come out alike. Runs of one row are walked side by side; each starts by
// reading the W - 1 steps before it again. More channels a thread means fewer loads but also fewer waves on a SIMD: both
// passes of 120 x 64 x 1024 bf16 29 us with 2, 30 with 1, 33 with 4; of 1021 x 9 x 771 fp32 46 with 4, 51 with 2, 54 with 1.
#include "apart.h"
#include "ssm_math.h"
#include <type_traits>

#define FB 8             // steps read ahead by the forward
#define BB 6             // and by the backward (two tensors)

struct ConvArgs {        // mirrored by ops/hip.py (_CONV): 64-bit words in this order
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

struct ConvGrid { int L, seg, n_seg, rows; };       // L threads across channels, steps a run, runs a row, rows of partials

template <typename T, int V>
__device__ __forceinline__ void cload(const T* q, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = ld(q);
    } else if constexpr (V == 2 && sizeof(T) == 2) {
        uint32_t r;
        __builtin_memcpy(&r, q, 4);
        v[0] = __uint_as_float(r << 16); v[1] = __uint_as_float(r & 0xffff0000u);
    } else if constexpr (V == 2) {
        float2 r;
        __builtin_memcpy(&r, q, 8);
        v[0] = r.x; v[1] = r.y;
    } else if constexpr (sizeof(T) == 2) {
        uint2 r;
        __builtin_memcpy(&r, q, 8);
        v[0] = __uint_as_float(r.x << 16); v[1] = __uint_as_float(r.x & 0xffff0000u);
        v[2] = __uint_as_float(r.y << 16); v[3] = __uint_as_float(r.y & 0xffff0000u);
    } else {
        float4 r;
        __builtin_memcpy(&r, q, 16);
        v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
    }
}
template <typename T, int V>
__device__ __forceinline__ void cstore(T* q, const float (&v)[V]) {
    if constexpr (V == 1) {
        st(q, v[0]);
    } else if constexpr (V == 2 && sizeof(T) == 2) {
        const uint32_t r = pack_bf2(v[0], v[1]);
        __builtin_memcpy(q, &r, 4);
    } else if constexpr (V == 2) {
        const float2 r = make_float2(v[0], v[1]);
        __builtin_memcpy(q, &r, 8);
    } else if constexpr (sizeof(T) == 2) {
        const uint2 r = make_uint2(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]));
        __builtin_memcpy(q, &r, 8);
    } else {
        const float4 r = make_float4(v[0], v[1], v[2], v[3]);
        __builtin_memcpy(q, &r, 16);
    }
}
template <int V>
__device__ __forceinline__ void czero(float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
}

__device__ __forceinline__ int row_end(const ConvArgs& p, int b) {
    return p.lengths ? max(0, min(p.lengths[b], (int)p.T)) : (int)p.T;
}

// WIDE: 64 or more threads across the channels, so a wave has one row and one run, whose steps and flags are scalars.
template <bool WIDE>
__device__ __forceinline__ int uniform(int v) { return WIDE ? __builtin_amdgcn_readfirstlane(v) : v; }

// bit q: step t0 + q (0 <= it < stop) has its reset flag set. WIDE: a lane reads a flag, every lane of the wave takes part.
template <int N, bool WIDE>
__device__ __forceinline__ unsigned reset_bits(const ConvArgs& p, int b, int t0, int stop) {
    if (!p.reset) return 0;
    if constexpr (WIDE) {
        const int q = threadIdx.x & 63;
        return (unsigned)__ballot(q < N && t0 + q >= 0 && t0 + q < stop && p.reset[(long long)(t0 + q) * p.B + b] != 0);
    }
    unsigned rm = 0;
#pragma unroll
    for (int q = 0; q < N; ++q) rm |= (t0 + q >= 0 && t0 + q < stop && p.reset[(long long)(t0 + q) * p.B + b] != 0 ? 1u : 0u) << q;
    return rm;
}

// xw[0 .. W - 2] = the inputs of times ta - W + 1 .. ta - 1 as the step at ta - 1 leaves them (what a reset cut off is 0 and
// not live); needs ta <= the row's end
template <typename T, int V, int W, bool WIDE>
__device__ __forceinline__ void window(const ConvArgs& p, int b, int ta, int d, float (&xw)[W][V], bool (&live)[W]) {
    const unsigned rm = reset_bits<W - 1, WIDE>(p, b, ta - W + 1, ta);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        const int t = ta - W + 1 + k;
        if (t >= 0) cload<T, V>((const T*)p.x + t * p.x_t + b * p.x_b + d, xw[k]);
        else if (p.state_in) cload<T, V>((const T*)p.state_in + ((long long)b * (W - 1) + (t + W - 1)) * p.D + d, xw[k]);
        else czero(xw[k]);
    }
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        live[k] = rm >> (k + 1) == 0;                                          // no episode starts behind it
        if (!live[k]) czero(xw[k]);
    }
}
template <int V, int W>
__device__ __forceinline__ void load_w(const ConvArgs& p, int d, float (&w)[W][V], float (&bias)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < W; ++k) w[k][i] = p.w[(long long)(d + i) * W + k];
        bias[i] = p.bias ? p.bias[d + i] : 0.f;
    }
}

// 120 x 64 x 1024 bf16 10.5 us (3.0 TB/s), 1021 x 9 x 771 fp32 12.7 us (4.5 TB/s): bound by the three memory latencies that a
// wave's run has one after the other (flags and window, steps, stores), of which too few waves are on the way at a time.
template <typename T, int V, int W, bool WIDE>
__global__ __launch_bounds__(256) void k_conv_fwd(ConvArgs p, ConvGrid cg) {
    int d = (blockIdx.x * cg.L + threadIdx.x % cg.L) * V, run = blockIdx.z * (256 / cg.L) + threadIdx.x / cg.L;
    const bool ok = d < p.D && run < cg.n_seg;                                 // idle lanes walk the last channels or run 0 and write nothing
    d = min(d, (int)p.D - V);
    if (run >= cg.n_seg) run = 0;                                              // (a whole wave's, where it has one run)
    run = uniform<WIDE>(run);
    const int b = blockIdx.y, ta = run * cg.seg;
    const int end = row_end(p, b), tb = min(ta + cg.seg, (int)p.T), stop = min(tb, end);
    float w[W][V], bias[V], xw[W][V];
    bool live[W];
    const bool silu = p.silu != 0;
    T* y = (T*)p.y + b * p.y_b + d;
    const auto put_state = [&] {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) cstore<T, V>((T*)p.state_out + ((long long)b * (W - 1) + k) * p.D + d, xw[k]);
    };
    if (ta <= end) {
        load_w<V, W>(p, d, w, bias);
        window<T, V, W, WIDE>(p, b, ta, d, xw, live);
        if (ta == 0 && end == 0 && p.state_out && ok) put_state();             // an empty row passes its state on
    }
    const T* x = (const T*)p.x + b * p.x_b + d;
    for (int t0 = ta; t0 < stop; t0 += FB) {
        float in[FB][V];
#pragma unroll
        for (int q = 0; q < FB; ++q) cload<T, V>(x + min(t0 + q, stop - 1) * p.x_t, in[q]);      // beyond the run: read again, not used
        const unsigned rm = reset_bits<FB, WIDE>(p, b, t0, stop);
        // a whole batch without a reset is straight code, in which the window moves by renaming
        const auto steps = [&](auto plain) {
#pragma unroll
            for (int q = 0; q < FB; ++q) {
                if (!plain && t0 + q >= stop) break;
                if (!plain && (rm >> q & 1)) {
#pragma unroll
                    for (int k = 0; k < W - 1; ++k) czero(xw[k]);
                }
                float v[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    xw[W - 1][i] = in[q][i];
                    v[i] = bias[i];
#pragma unroll
                    for (int k = 0; k < W; ++k) v[i] = fmaf(w[k][i], xw[k][i], v[i]);
                    if (silu) v[i] *= sigmoidf(v[i]);
#pragma unroll
                    for (int k = 0; k < W - 1; ++k) xw[k][i] = xw[k + 1][i];
                }
                if (ok) cstore<T, V>(y + (t0 + q) * p.y_t, v);
            }
        };
        if (__all(rm == 0 && t0 + FB <= stop)) steps(std::true_type{}); else steps(std::false_type{});
    }
    if (!ok) return;
    if (stop == end && stop > ta && p.state_out) put_state();                  // the row's last step was this run's
    float zero[V];
    czero(zero);
    for (int t = max(ta, stop); t < tb; ++t) cstore<T, V>(y + t * p.y_t, zero);
}

// dx[tau] collects w[k] dpre[tau + W - 1 - k]: one walk forward in time with W open sums. A run emits its steps ta .. tb - 1
// and goes W - 1 steps further for them; dw and db count its own steps only and stay in registers over all the runs that a
// thread takes (every cg.rows-th). Bound as the forward is, with half of its waves (the sums' registers).
template <typename T, int V, int W, bool WIDE>
__global__ __launch_bounds__(256) void k_conv_bwd(ConvArgs p, ConvGrid cg) {
    __shared__ float acc[W + 1][256 * V];
    const int lx = threadIdx.x % cg.L, ly = threadIdx.x / cg.L, per = 256 / cg.L;
    const bool dv = (blockIdx.x * cg.L + lx) * V < p.D;                         // idle lanes walk the last channels and write nothing
    const int d = min((int)(blockIdx.x * cg.L + lx) * V, (int)p.D - V);
    float w[W][V], bias[V], dw[W][V], db[V];
    load_w<V, W>(p, d, w, bias);
#pragma unroll
    for (int k = 0; k < W; ++k) czero(dw[k]);
    czero(db);
    const bool silu = p.silu != 0;
    const unsigned B = (unsigned)p.B, n_runs = (unsigned)cg.n_seg * B;      // T B <= 2^31
    for (unsigned r = blockIdx.y * per + ly; r < n_runs; r += cg.rows * per) {
        const int run = uniform<WIDE>((int)(r / B)), b = uniform<WIDE>((int)(r % B)), ta = run * cg.seg;
        const int end = row_end(p, b), tb = min(ta + cg.seg, (int)p.T), last = tb + W - 1, stop = min(last, end);
        float xw[W][V], open[W][V];
        bool live[W];
#pragma unroll
        for (int k = 0; k < W; ++k) { czero(open[k]); czero(xw[k]); live[k] = true; }
        if (ta < end) window<T, V, W, WIDE>(p, b, ta, d, xw, live);
        const T *x = (const T*)p.x + b * p.x_b + d, *dy = (const T*)p.dy + b * p.dy_b + d;
        T* dx = (T*)p.dx + b * p.dx_b + d;
        // tau = t - W + 1 is complete once step t is through: no later step reaches back to it
        const auto emit = [&](int t) {
            const int tau = t - W + 1;
            if (tau < 0) {
                if (p.dstate_in && ta == 0 && dv) cstore<T, V>((T*)p.dstate_in + ((long long)b * (W - 1) + tau + W - 1) * p.D + d, open[0]);
            } else if (tau >= ta && dv) {
                cstore<T, V>(dx + tau * p.dx_t, open[0]);
            }
#pragma unroll
            for (int k = 0; k < W - 1; ++k) {
                live[k] = live[k + 1];
#pragma unroll
                for (int i = 0; i < V; ++i) { xw[k][i] = xw[k + 1][i]; open[k][i] = open[k + 1][i]; }
            }
            czero(open[W - 1]);
        };
        for (int t0 = ta; t0 < stop; t0 += BB) {
            float in[BB][V], gy[BB][V];
#pragma unroll
            for (int q = 0; q < BB; ++q) {
                const int t = min(t0 + q, stop - 1);
                cload<T, V>(x + t * p.x_t, in[q]);
                cload<T, V>(dy + t * p.dy_t, gy[q]);
            }
            const unsigned rm = reset_bits<BB, WIDE>(p, b, t0, stop);
            // a whole batch of the run's own steps in one episode is straight code, see k_conv_fwd
            const auto steps = [&](auto plain) {
#pragma unroll
                for (int q = 0; q < BB; ++q) {
                    const int t = t0 + q;
                    if (!plain && t >= stop) break;
                    if (!plain && (rm >> q & 1)) {
#pragma unroll
                        for (int k = 0; k < W - 1; ++k) { czero(xw[k]); live[k] = false; }
                    }
                    live[W - 1] = true;
                    const bool mine = plain || t < tb;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        xw[W - 1][i] = in[q][i];
                        float v = bias[i], g = gy[q][i];
#pragma unroll
                        for (int k = 0; k < W; ++k) v = fmaf(w[k][i], xw[k][i], v);
                        if (silu) { const float s = sigmoidf(v); g *= s * fmaf(v, 1.f - s, 1.f); }
#pragma unroll
                        for (int k = 0; k < W; ++k) open[k][i] = plain || live[k] ? fmaf(w[k][i], g, open[k][i]) : open[k][i];
                        if (mine) {
                            db[i] += g;
#pragma unroll
                            for (int k = 0; k < W; ++k) dw[k][i] = fmaf(g, xw[k][i], dw[k][i]);
                        }
                    }
                    emit(t);
                }
            };
            bool whole = rm == 0 && t0 + BB <= min(stop, tb);
#pragma unroll
            for (int k = 0; k < W - 1; ++k) whole = whole && live[k];
            if (__all(whole)) steps(std::true_type{}); else steps(std::false_type{});
        }
        for (int t = max(ta, stop); t < last; ++t) {
            if (t == end && p.dstate_out) {           // the state the row left = its last W - 1 inputs: their gradient comes in here
#pragma unroll
                for (int k = 0; k < W - 1; ++k) {
                    if (!live[k]) continue;
                    float g[V];
                    cload<T, V>((const T*)p.dstate_out + ((long long)b * (W - 1) + k) * p.D + d, g);
#pragma unroll
                    for (int i = 0; i < V; ++i) open[k][i] += g[i];
                }
            }
            emit(t);
        }
    }
    // the block's sums: its `per` groups one after the other, then a row of partials [W + 1][D]
    for (int t = 0; t < per; ++t) {
        if (ly == t) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
#pragma unroll
                for (int k = 0; k < W; ++k) acc[k][lx * V + i] = (t ? acc[k][lx * V + i] : 0.f) + dw[k][i];
                acc[W][lx * V + i] = (t ? acc[W][lx * V + i] : 0.f) + db[i];
            }
        }
        if (per > 1) __syncthreads();
    }
    if (ly == 0 && dv) {
        float* q = p.ws + (long long)blockIdx.y * (W + 1) * p.D + d;
#pragma unroll
        for (int k = 0; k <= W; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) q[k * p.D + i] = acc[k][lx * V + i];
    }
}

// R rows of partials [W + 1][D] -> dw [D, W], db: 32 columns by 32 groups of rows a block, in a fixed order
__global__ __launch_bounds__(1024) void k_conv_sum(const float* __restrict__ part, int R, int W, long long D, float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float acc[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const long long n = (W + 1) * D, c = (long long)blockIdx.x * 32 + x;
    float v = 0.f;
    if (c < n) {
#pragma unroll 8
        for (int r = y; r < R; r += 32) v += part[r * n + c];
    }
    acc[y][x] = v;
    __syncthreads();
    if (y == 0 && c < n) {
        v = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) v += acc[k][x];
        const long long k = c / D, d = c - k * D;
        if (k < W) dw[d * W + k] = v;
        else if (db) db[d] = v;
    }
}

// One step. A thread per V channels of a row. Bound by memory: 4096 x 1024 bf16 12 us (5.5 TB/s).
template <typename T, int V, int W>
__global__ __launch_bounds__(256) void k_conv_step(ConvArgs p) {
    const long long i = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x, cv = (p.D + V - 1) / V;
    if (i >= p.B * cv) return;
    const long long b = i / cv, c = (i - b * cv) * V, d = min(c, p.D - V);
    const int dup = (int)(c - d);           // the state changes in place: what the vector before has is not written twice
    T* s = (T*)p.state_out + b * (W - 1) * p.D + d;
    const bool rs = p.reset && p.reset[b] != 0;
    float row[W][V], w[W][V], v[V];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) cload<T, V>(s + k * p.D, row[k]);
    cload<T, V>((const T*)p.x + b * p.x_b + d, row[W - 1]);
    load_w<V, W>(p, (int)d, w, v);
    if (rs) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) czero(row[k]);
    }
#pragma unroll
    for (int q = 0; q < V; ++q) {
#pragma unroll
        for (int k = 0; k < W; ++k) v[q] = fmaf(w[k][q], row[k][q], v[q]);
        if (p.silu) v[q] *= sigmoidf(v[q]);
    }
    T* y = (T*)p.y + b * p.y_b + d;
    if (dup == 0) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k) cstore<T, V>(s + k * p.D, row[k + 1]);
        cstore<T, V>(y, v);
        return;
    }
#pragma unroll
    for (int q = 1; q < V; ++q) {
        if (q < dup) continue;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) st(s + k * p.D + q, row[k + 1][q]);
        st(y + q, v[q]);
    }
}

static bool conv_ok(long long T, long long B, long long D, long long W) {
    return T > 0 && T <= 1000000 && B > 0 && B <= 65535 && T * B <= (1ll << 31) && D > 0 && D <= (1ll << 22) && W >= 2 && W <= 4;
}

// channels a thread of the sequence kernels, see above; a single step has two (4 096 x 1 024: bf16 12 us against 14 with one and
// 17 with four, fp32 21 against 23 with four)
#define V_BF16 2
#define V_F32 4
#define V_STEP 2
static long long conv_cols(long long D, int V) { return D < V ? D : (D + V - 1) / V; }
static int conv_v(int bf16) { return bf16 ? V_BF16 : V_F32; }

// Runs of 8 steps, longer ones (up to 64: fewer steps are read twice) where they still give the chip 4 096 waves: the forward of
// 120 x 64 x 1024 bf16 takes 10.5 us in runs of 16 and 10.7 of 8. The backward walks W - 1 steps more than a run has: its
// runs are that much short of 12 (below 1 024 waves), 18 (both passes of the above 29.5 us against 31.7 with 12), 36 or 60.
// A block of the backward takes every rows-th run: 1 024 rows of partials at most (29.5 us; 512 33, 2 048 29.5).
static ConvGrid conv_grid(long long T, long long B, long long D, int bf16, int extra) {
    const long long cv = conv_cols(D, conv_v(bf16));
    int L = 1;
    while (L < cv && L < 256) L *= 2;
    const long long waves = (cv + L - 1) / L * L * B / 64;                    // of one run a row
    const int choice[2][4] = {{8, 16, 32, 64}, {12 - extra, 18 - extra, 36 - extra, 60 - extra}};
    int k = 0;
    while (k < 3 && waves * ((T + choice[extra > 0][k + 1] - 1) / choice[extra > 0][k + 1]) >= (extra && k == 0 ? 1024 : 4096)) ++k;
    const int seg = choice[extra > 0][k];
    const long long n_seg = (T + seg - 1) / seg, blocks = (n_seg * B + 256 / L - 1) / (256 / L), cols = (cv + L - 1) / L;
    long long rows = (1024 + cols - 1) / cols;
    if (rows > blocks) rows = blocks;
    return {L, seg, (int)n_seg, (int)rows};
}

// floats of scratch of a backward pass
DRL_API int drl_short_conv_ws(long long T, long long B, long long D, long long W, long long* n) {
    if (!conv_ok(T, B, D, W)) return -1;
    const int a = conv_grid(T, B, D, 0, (int)W - 1).rows, b = conv_grid(T, B, D, 1, (int)W - 1).rows;
    *n = (a > b ? a : b) * (W + 1) * D;
    return 0;
}

template <typename T, int V, int W, bool WIDE>
static void launch_conv(const ConvArgs& p, const ConvGrid& cg, bool bwd, dim3 grid, hipStream_t s) {
    if (bwd) k_conv_bwd<T, V, W, WIDE><<<grid, 256, 0, s>>>(p, cg);
    else k_conv_fwd<T, V, W, WIDE><<<grid, 256, 0, s>>>(p, cg);
}
template <typename T, int V, int W>
static void launch_conv_step(const ConvArgs& p, dim3 grid, hipStream_t s) { k_conv_step<T, V, W><<<grid, 256, 0, s>>>(p); }
// F<T, V, W>(...) for the call's type, channels and taps
#define CONV_W(F, T, V, ...)                                           \
    switch (p.W) {                                                      \
        case 2: F(T, V, 2, __VA_ARGS__); break;                         \
        case 3: F(T, V, 3, __VA_ARGS__); break;                         \
        default: F(T, V, 4, __VA_ARGS__); break;                        \
    }
#define CONV_ALL(F, VB, VF, ...)                                                                                            \
    if (bf16) { if (p.D >= VB) { CONV_W(F, bf16_t, VB, __VA_ARGS__) } else { CONV_W(F, bf16_t, 1, __VA_ARGS__) } }         \
    else { if (p.D >= VF) { CONV_W(F, float, VF, __VA_ARGS__) } else { CONV_W(F, float, 1, __VA_ARGS__) } }
#define CONV_SEQ(T, V, W, BWD) cg.L >= 64 ? launch_conv<T, V, W, true>(p, cg, BWD, grid, s) : launch_conv<T, V, W, false>(p, cg, BWD, grid, s)
#define CONV_ONE(T, V, W, _) launch_conv_step<T, V, W>(p, grid, s)

// a [T, B, D] tensor (e bytes an element) and what else a call reads
static View seq_view(const ConvArgs& p, const void* q, long long st, long long sb, long long e) { return {q, p.D * e, p.T, st * e, p.B, sb * e}; }
static View state_view(const ConvArgs& p, const void* q, long long e) { return {q, p.B * (p.W - 1) * p.D * e}; }

DRL_API int drl_short_conv_fwd(const ConvArgs* a, int bf16, hipStream_t s) {
    const ConvArgs p = *a;
    if (!conv_ok(p.T, p.B, p.D, p.W)) return -1;
    const long long e = bf16 ? 2 : 4;
    if (!apart({seq_view(p, p.y, p.y_t, p.y_b, e), state_view(p, p.state_out, e)},
               {seq_view(p, p.x, p.x_t, p.x_b, e), state_view(p, p.state_in, e), {p.w, p.D * p.W * 4}, {p.bias, p.D * 4}, {p.reset, p.T * p.B},
                {p.lengths, p.B * 4}})) return -3;
    const ConvGrid cg = conv_grid(p.T, p.B, p.D, bf16, 0);
    const long long cv = conv_cols(p.D, conv_v(bf16)), per = 256 / cg.L;
    if ((cg.n_seg + per - 1) / per > 65535) return -1;
    const dim3 grid((unsigned)((cv + cg.L - 1) / cg.L), (unsigned)p.B, (unsigned)((cg.n_seg + per - 1) / per));
    CONV_ALL(CONV_SEQ, V_BF16, V_F32, false)
    return (int)hipGetLastError();
}

DRL_API int drl_short_conv_bwd(const ConvArgs* a, int bf16, hipStream_t s) {
    const ConvArgs p = *a;
    long long need;
    if (drl_short_conv_ws(p.T, p.B, p.D, p.W, &need)) return -1;
    if (p.ws_n < need) return -2;
    const long long e = bf16 ? 2 : 4;
    if (!apart({seq_view(p, p.dx, p.dx_t, p.dx_b, e), state_view(p, p.dstate_in, e), {p.dw, p.D * p.W * 4}, {p.db, p.D * 4}, {p.ws, need * 4}},
               {seq_view(p, p.x, p.x_t, p.x_b, e), seq_view(p, p.dy, p.dy_t, p.dy_b, e), state_view(p, p.state_in, e), state_view(p, p.dstate_out, e),
                {p.w, p.D * p.W * 4}, {p.bias, p.D * 4}, {p.reset, p.T * p.B}, {p.lengths, p.B * 4}})) return -3;
    const ConvGrid cg = conv_grid(p.T, p.B, p.D, bf16, (int)p.W - 1);
    const long long cv = conv_cols(p.D, conv_v(bf16)), n = (p.W + 1) * p.D;
    const dim3 grid((unsigned)((cv + cg.L - 1) / cg.L), (unsigned)cg.rows);
    CONV_ALL(CONV_SEQ, V_BF16, V_F32, true)
    k_conv_sum<<<(unsigned)((n + 31) / 32), 1024, 0, s>>>(p.ws, cg.rows, (int)p.W, p.D, p.dw, p.db);
    return (int)hipGetLastError();
}

DRL_API int drl_short_conv_step(const ConvArgs* a, int bf16, hipStream_t s) {
    const ConvArgs p = *a;
    if (!conv_ok(1, 1, p.D, p.W) || p.B <= 0) return -1;
    const long long e = bf16 ? 2 : 4;
    if (!apart({{p.y, p.D * e, p.B, p.y_b * e}, state_view(p, p.state_out, e)},
               {{p.x, p.D * e, p.B, p.x_b * e}, {p.w, p.D * p.W * 4}, {p.bias, p.D * 4}, {p.reset, p.B}})) return -3;
    const long long nb = (p.B * conv_cols(p.D, V_STEP) + 255) / 256;
    if (nb >= 1ll << 38) return -1;
    const long long x = nb < (1 << 23) ? nb : 1 << 23;
    const dim3 grid((unsigned)x, (unsigned)((nb + x - 1) / x));
    CONV_ALL(CONV_ONE, V_STEP, V_STEP, 0)
    return (int)hipGetLastError();
}
