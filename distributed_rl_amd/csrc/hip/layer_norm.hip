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

// A team of TW waves owns a row and keeps it in registers, 16 values a lane at most (D <= 1 024 TW): one read, the mean, the
// spread around it, one write. V values travel per load (16 bytes, or 1 value where an address or a stride does not allow it).
template <typename T, int V>
__device__ __forceinline__ void load_v(const T* q, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = ld(q);
    } else if constexpr (sizeof(T) == 2) {
        const uint4 r = *reinterpret_cast<const uint4*>(q);
        const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
    } else {
        const float4 r = *reinterpret_cast<const float4*>(q);
        v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* q, const float (&v)[V]) {
    if constexpr (V == 1) st(q, v[0]);
    else if constexpr (sizeof(T) == 2) *reinterpret_cast<uint4*>(q) = make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
    else *reinterpret_cast<float4*>(q) = make_float4(v[0], v[1], v[2], v[3]);
}
// fp32 parameters of V columns (zeros for a null pointer)
template <int V>
__device__ __forceinline__ void load_p(const float* q, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = q[0];
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) { const float4 r = *reinterpret_cast<const float4*>(q + i); v[i] = r.x; v[i + 1] = r.y; v[i + 2] = r.z; v[i + 3] = r.w; }
    }
}

// sums of K values over the team's TW waves; slot: LDS of TW x K floats, another one for each use in flight
template <int TW, int K>
__device__ __forceinline__ void team_sum(float (&v)[K], float* slot) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lane_sum(v[k]);
    if constexpr (TW > 1) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) slot[k * TW + w] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < TW; ++i) t += slot[k * TW + i];
            v[k] = t;
        }
    }
}

// TW = 1: four rows a block. NV vectors a lane.
template <typename T, int V, int NV, int TW>
__global__ __launch_bounds__(TW > 1 ? 64 * TW : 256) void k_norm_fwd(NormArgs p, float eps) {
    __shared__ float slot[2][TW];
    const int lane = TW > 1 ? threadIdx.x : threadIdx.x & 63;
    const long long r = TW > 1 ? blockIdx.x : (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= p.M) return;                              // TW = 1 only: a whole wave, and nothing waits for it
    const int D = (int)p.D;
    const T* x = (const T*)p.x + r * p.x_r;
    float v[NV][V], s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * 64 * TW + lane) * V;
        if (c < D) load_v<T, V>(x + c, v[k]);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if ((k * 64 * TW + lane) * V < D) {
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] += v[k][i];
        }
    }
    team_sum<TW, 1>(s, slot[0]);
    const float mean = s[0] / (float)D;
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if ((k * 64 * TW + lane) * V < D) {
#pragma unroll
            for (int i = 0; i < V; ++i) { v[k][i] -= mean; s[0] = fmaf(v[k][i], v[k][i], s[0]); }
        }
    }
    team_sum<TW, 1>(s, slot[1]);
    const float rstd = 1.0f / sqrtf(s[0] / (float)D + eps);
    T* y = (T*)p.y + r * p.y_r;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * 64 * TW + lane) * V;
        if (c < D) {
            float w[V], b[V];
            load_p<V>(p.w + c, w);
#pragma unroll
            for (int i = 0; i < V; ++i) b[i] = 0.f;
            if (p.b) load_p<V>(p.b + c, b);
#pragma unroll
            for (int i = 0; i < V; ++i) v[k][i] = fmaf(v[k][i] * rstd, w[i], b[i]);
            store_v<T, V>(y + c, v[k]);
        }
    }
    if (lane == 0 && p.mean) { p.mean[r] = mean; p.rstd[r] = rstd; }
}

// A team walks every n_teams-th row, the next row's loads under way: dx of the row, and dw, db of its columns in registers.
// The block's sums leave as one row of partials [2 D].
template <typename T, int V, int NV, int TW>
__global__ __launch_bounds__(TW > 1 ? 64 * TW : 256) void k_norm_bwd(NormArgs p) {
    __shared__ float slot[2][2 * TW];
    const int wave = threadIdx.x >> 6, lane = TW > 1 ? threadIdx.x : threadIdx.x & 63;
    const int D = (int)p.D;
    const long long n_teams = TW > 1 ? gridDim.x : (long long)gridDim.x * 4;
    float w[NV][V], dw[NV][V], db[NV][V], x[NV][V], dy[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * 64 * TW + lane) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) { w[k][i] = dw[k][i] = db[k][i] = x[k][i] = dy[k][i] = 0.f; }
        if (c < D) load_p<V>(p.w + c, w[k]);
    }
    const float inv = 1.0f / (float)D;
    int par = 0;
    for (long long r = TW > 1 ? blockIdx.x : (long long)blockIdx.x * 4 + wave; r < p.M; r += n_teams, par ^= 1) {
        const T *xp = (const T*)p.x + r * p.x_r, *dyp = (const T*)p.dy + r * p.dy_r;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * 64 * TW + lane) * V;
            if (c < D) { load_v<T, V>(xp + c, x[k]); load_v<T, V>(dyp + c, dy[k]); }
        }
        const float mean = p.mean[r], rstd = p.rstd[r];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if ((k * 64 * TW + lane) * V < D) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    x[k][i] = (x[k][i] - mean) * rstd;
                    dw[k][i] = fmaf(dy[k][i], x[k][i], dw[k][i]);
                    db[k][i] += dy[k][i];
                    dy[k][i] *= w[k][i];
                    s[0] += dy[k][i];
                    s[1] = fmaf(dy[k][i], x[k][i], s[1]);
                }
            }
        }
        team_sum<TW, 2>(s, slot[par]);
        const float m1 = s[0] * inv, m2 = s[1] * inv;
        T* dx = (T*)p.dx + r * p.dx_r;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * 64 * TW + lane) * V;
            if (c < D) {
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = (dy[k][i] - m1 - x[k][i] * m2) * rstd;
                store_v<T, V>(dx + c, o);
            }
        }
    }
    if constexpr (TW == 1) {                           // the block's four teams, one after the other
        __shared__ float acc[2][1024];
        for (int t = 0; t < 4; ++t) {
            if (wave == t) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int c = (k * 64 + lane) * V;
                    if (c < D) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            acc[0][c + i] = (t ? acc[0][c + i] : 0.f) + dw[k][i];
                            acc[1][c + i] = (t ? acc[1][c + i] : 0.f) + db[k][i];
                        }
                    }
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < 2 * D; c += 256) p.ws[(long long)blockIdx.x * 2 * D + c] = c < D ? acc[0][c] : acc[1][c - D];
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * 64 * TW + lane) * V;
            if (c < D) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    p.ws[(long long)blockIdx.x * 2 * D + c + i] = dw[k][i];
                    p.ws[(long long)blockIdx.x * 2 * D + D + c + i] = db[k][i];
                }
            }
        }
    }
}

// R rows of partials -> dw, db: 32 columns by 32 groups of rows a block, in a fixed order
__global__ __launch_bounds__(1024) void k_norm_sum(const float* __restrict__ part, int R, int D, float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float acc[32][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
    float v = 0.f;
    if (c < 2 * D) {
#pragma unroll 8
        for (int r = y; r < R; r += 32) v += part[(long long)r * 2 * D + c];
    }
    acc[y][x] = v;
    __syncthreads();
    if (y == 0 && c < 2 * D) {
        v = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) v += acc[k][x];
        if (c < D) dw[c] = v;
        else if (db) db[c - D] = v;
    }
}

static bool norm_ok(long long M, long long D) { return M > 0 && M < (1ll << 31) && D > 0 && D <= 16384; }
static int team_waves(long long D) { return D <= 1024 ? 1 : D <= 4096 ? 4 : 16; }
// blocks of the backward = rows of partials
static int norm_blocks(long long M, long long D) {
    const long long rows = team_waves(D) == 1 ? (M + 3) / 4 : M;
    return (int)(rows < 512 ? rows : 512);
}

DRL_API int drl_norm_ws(long long M, long long D, long long* n) {
    if (!norm_ok(M, D)) return -1;
    *n = 2 * D * norm_blocks(M, D);
    return 0;
}

static bool by16(const void* q, long long stride_bytes) { return (((uintptr_t)q | (uintptr_t)stride_bytes) & 15) == 0; }

template <typename T, int V, int NV>
static void norm_launch(const NormArgs& p, bool bwd, float eps, hipStream_t s) {
    const int tw = team_waves(p.D);
    const unsigned g1 = (unsigned)((p.M + 3) / 4), gn = (unsigned)p.M, gb = (unsigned)norm_blocks(p.M, p.D);
    if (!bwd) {
        if (tw == 1) k_norm_fwd<T, V, NV, 1><<<g1, 256, 0, s>>>(p, eps);
        else if (tw == 4) k_norm_fwd<T, V, NV, 4><<<gn, 256, 0, s>>>(p, eps);
        else k_norm_fwd<T, V, NV, 16><<<gn, 1024, 0, s>>>(p, eps);
    } else {
        if (tw == 1) k_norm_bwd<T, V, NV, 1><<<gb, 256, 0, s>>>(p);
        else if (tw == 4) k_norm_bwd<T, V, NV, 4><<<gb, 256, 0, s>>>(p);
        else k_norm_bwd<T, V, NV, 16><<<gb, 1024, 0, s>>>(p);
    }
}

template <typename T>
static void norm_dispatch(const NormArgs& p, bool bwd, float eps, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const long long e = sizeof(T);
    const bool vec = p.D % V == 0 && by16(p.x, p.x_r * e) && by16(p.w, 0) && by16(p.b, 0)
                     && (bwd ? by16(p.dy, p.dy_r * e) && by16(p.dx, p.dx_r * e) : by16(p.y, p.y_r * e));
    const long long n = (p.D + 64 * team_waves(p.D) - 1) / (64 * team_waves(p.D));        // values a lane, one at a time: 1 .. 16
    if (vec) {
        const long long nv = (n + V - 1) / V;
        if constexpr (sizeof(T) == 2) {
            if (nv == 1) norm_launch<T, V, 1>(p, bwd, eps, s);
            else norm_launch<T, V, 2>(p, bwd, eps, s);
        } else {
            if (nv == 1) norm_launch<T, V, 1>(p, bwd, eps, s);
            else if (nv == 2) norm_launch<T, V, 2>(p, bwd, eps, s);
            else norm_launch<T, V, 4>(p, bwd, eps, s);
        }
    } else if (n <= 4) {
        norm_launch<T, 1, 4>(p, bwd, eps, s);
    } else {
        norm_launch<T, 1, 16>(p, bwd, eps, s);
    }
}

DRL_API int drl_norm_fwd(const NormArgs* a, int bf16, float eps, hipStream_t s) {
    const NormArgs p = *a;
    if (!norm_ok(p.M, p.D)) return -1;
    if (bf16) norm_dispatch<bf16_t>(p, false, eps, s);
    else norm_dispatch<float>(p, false, eps, s);
    return (int)hipGetLastError();
}

DRL_API int drl_norm_bwd(const NormArgs* a, int bf16, hipStream_t s) {
    const NormArgs p = *a;
    long long need;
    if (drl_norm_ws(p.M, p.D, &need)) return -1;
    if (p.ws_n < need) return -2;
    if (bf16) norm_dispatch<bf16_t>(p, true, 0.f, s);
    else norm_dispatch<float>(p, true, 0.f, s);
    k_norm_sum<<<(unsigned)((2 * p.D + 31) / 32), 1024, 0, s>>>(p.ws, norm_blocks(p.M, p.D), (int)p.D, p.dw, p.db);
    return (int)hipGetLastError();
}
