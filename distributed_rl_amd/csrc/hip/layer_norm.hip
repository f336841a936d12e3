// Layer norm over the last axis and its backward pass.
//   y = (x - mean) rstd w + b;   dx = rstd (dn - mean(dn) - n mean(dn n)), n = (x - mean) rstd, dn = dy w
//   dw = sum over rows of dy n,  db = sum over rows of dy
// The variance is summed around the mean, not as E[x^2] - mean^2, which cancels for rows far from zero.
#include "apart.h"
#include "ssm_math.h"

struct NormArgs {        // mirrored by ops/hip.py (_NORM): 64-bit words in this order
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

// A team of L lanes (4 to 64, or 64 x TW of TW waves) owns a row and keeps it in registers, NV vectors a lane: one read, the
// mean, the spread around it, one write. V values (16 bytes) travel per load. AL: every vector lies at a multiple of 16 bytes
// and D is a multiple of V; otherwise vectors start anywhere (the memory system takes them), and a row's last one ends at the
// row's end: its first `dup` columns are the vector before's, left out of the sums and stored twice with the same value.
// Bound by memory. Forward and backward of 10 M values, bf16 / fp32: D = 17 55 / 86 us, 40 33 / 58, 100 36 / 51, 130 41 / 59,
// 256 28 / 45, 350 36 / 53, 511 37 / 47, 768 30 / 46; of 20 M values 512 55 / 83, 4001 81 / 100, 4096 69 / 88 (4.6 TB/s).
template <typename T, int V, bool AL>
__device__ __forceinline__ void load_v(const T* q, int n, float (&v)[V]) {
    if (AL || n >= V) {
        uint4 r;
        if constexpr (AL) r = *reinterpret_cast<const uint4*>(q);
        else __builtin_memcpy(&r, q, 16);
        const uint32_t u[4] = {r.x, r.y, r.z, r.w};
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < n ? ld(q + i) : 0.f;
    }
}
template <typename T, int V, bool AL>
__device__ __forceinline__ void store_v(T* q, int n, const float (&v)[V]) {
    if (AL || n >= V) {
        uint4 r;
        if constexpr (sizeof(T) == 2) r = make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
        else r = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        if constexpr (AL) *reinterpret_cast<uint4*>(q) = r;
        else __builtin_memcpy(q, &r, 16);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) if (i < n) st(q + i, v[i]);
    }
}
// column where vector c of a row of D starts, and how many of its columns the vector before has
template <int V, bool AL>
__device__ __forceinline__ int col_of(int c, int D, int& dup) {
    const int cb = AL || D < V ? c : min(c, D - V);
    dup = AL ? 0 : c - cb;
    return cb;
}

// fp32 parameters of n columns
template <int V, bool AL>
__device__ __forceinline__ void load_p(const float* q, int n, float (&v)[V]) {
    if (AL || n >= V) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            float4 r;
            if constexpr (AL) r = *reinterpret_cast<const float4*>(q + i);
            else __builtin_memcpy(&r, q + i, 16);
            v[i] = r.x; v[i + 1] = r.y; v[i + 2] = r.z; v[i + 3] = r.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < n ? q[i] : 0.f;
    }
}

// sums of K values over a team; slot: LDS of TW x K floats, another one for each use in flight
template <int L, int TW, int K>
__device__ __forceinline__ void team_sum(float (&v)[K], float* slot) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lane_sum<L>(v[k]);
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

// [7680, 512] bf16 5.9 us (2.7 TB/s), [7680, 3136] fp32 37 us (5.2 TB/s, as a copy of that size); [256, 512] 3.0 us, of which
// 2.5 are any kernel's. NV vectors a lane; blocks of 256 threads, or of the one team where it has more than a wave. Teams behind the last row stand
// in for it and write nothing, so that whole waves take part in every sum.
template <typename T, int V, int NV, int L, int TW, bool AL>
__global__ __launch_bounds__(TW > 1 ? 64 * TW : 256) void k_norm_fwd(NormArgs p, float eps) {
    __shared__ float slot[2][TW];
    const int lane = TW > 1 ? threadIdx.x : threadIdx.x % L, D = (int)p.D;
    const long long r0 = TW > 1 ? blockIdx.x : (long long)blockIdx.x * (256 / L) + threadIdx.x / L, r = min(r0, p.M - 1);
    const T* x = (const T*)p.x + r * p.x_r;
    float v[NV][V], s[1] = {0.f};
    int dup[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * L * TW + lane) * V, cb = col_of<V, AL>(c, D, dup[k]);
        if (c < D) load_v<T, V, AL>(x + cb, D - cb, v[k]);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if ((k * L * TW + lane) * V < D) {
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] += AL || i >= dup[k] ? v[k][i] : 0.f;
        }
    }
    team_sum<L, TW, 1>(s, slot[0]);
    const float mean = s[0] / (float)D;
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * L * TW + lane) * V;
        if (c < D) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k][i] -= mean;
                if (AL || (i >= dup[k] && c - dup[k] + i < D)) s[0] = fmaf(v[k][i], v[k][i], s[0]);
            }
        }
    }
    team_sum<L, TW, 1>(s, slot[1]);
    if (r0 >= p.M) return;
    const float rstd = 1.0f / sqrtf(s[0] / (float)D + eps);
    T* y = (T*)p.y + r * p.y_r;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * L * TW + lane) * V;
        if (c < D) {
            const int cb = c - dup[k];
            float w[V], b[V];
            load_p<V, AL>(p.w + cb, D - cb, w);
#pragma unroll
            for (int i = 0; i < V; ++i) b[i] = 0.f;
            if (p.b) load_p<V, AL>(p.b + cb, D - cb, b);
#pragma unroll
            for (int i = 0; i < V; ++i) v[k][i] = fmaf(v[k][i] * rstd, w[i], b[i]);
            store_v<T, V, AL>(y + cb, D - cb, v[k]);
        }
    }
    if (lane == 0 && p.mean) { p.mean[r] = mean; p.rstd[r] = rstd; }
}

// A team walks every n_teams-th row: dx of the row, and dw, db of its columns in registers. The block's sums leave as one row
// of partials [2 D]. [7680, 512] bf16 9.3 us, [7680, 3136] fp32 64 us (4.5 TB/s).
template <typename T, int V, int NV, int L, int TW, bool AL>
__global__ __launch_bounds__(TW > 1 ? 64 * TW : 256) void k_norm_bwd(NormArgs p) {
    constexpr int TEAMS = TW > 1 ? 1 : 256 / L, COLS = NV * L * TW * V;
    __shared__ float slot[2][2 * TW];
    const int team = TW > 1 ? 0 : threadIdx.x / L, lane = TW > 1 ? threadIdx.x : threadIdx.x % L, D = (int)p.D;
    float w[NV][V], dw[NV][V], db[NV][V], x[NV][V], dy[NV][V];
    int dup[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * L * TW + lane) * V, cb = col_of<V, AL>(c, D, dup[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) { w[k][i] = dw[k][i] = db[k][i] = x[k][i] = dy[k][i] = 0.f; }
        if (c < D) load_p<V, AL>(p.w + cb, D - cb, w[k]);
    }
    const float inv = 1.0f / (float)D;
    int par = 0;
    for (long long rb = (long long)blockIdx.x * TEAMS; rb < p.M; rb += (long long)gridDim.x * TEAMS, par ^= 1) {
        const bool ok = rb + team < p.M;
        const long long r = ok ? rb + team : p.M - 1;
        const T *xp = (const T*)p.x + r * p.x_r, *dyp = (const T*)p.dy + r * p.dy_r;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * L * TW + lane) * V;
            const int cb = c - dup[k];
            if (c < D) { load_v<T, V, AL>(xp + cb, D - cb, x[k]); load_v<T, V, AL>(dyp + cb, D - cb, dy[k]); }
        }
        const float mean = p.mean[r], rstd = p.rstd[r];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * L * TW + lane) * V;
            if (c < D) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    x[k][i] = (x[k][i] - mean) * rstd;             // columns behind the end (D < V) have dy = 0 and w = 0
                    const bool mine = AL || i >= dup[k];
                    const float g = ok && mine ? dy[k][i] : 0.f;
                    dw[k][i] = fmaf(g, x[k][i], dw[k][i]);
                    db[k][i] += g;
                    dy[k][i] *= w[k][i];
                    const float dn = mine ? dy[k][i] : 0.f;
                    s[0] += dn;
                    s[1] = fmaf(dn, x[k][i], s[1]);
                }
            }
        }
        team_sum<L, TW, 2>(s, slot[par]);
        const float m1 = s[0] * inv, m2 = s[1] * inv;
        T* dx = (T*)p.dx + r * p.dx_r;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * L * TW + lane) * V;
            if (c < D && ok) {
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = (dy[k][i] - m1 - x[k][i] * m2) * rstd;
                store_v<T, V, AL>(dx + c - dup[k], D - c + dup[k], o);
            }
        }
    }
    float* part = p.ws + (long long)blockIdx.x * 2 * D;
    if constexpr (TEAMS > 1) {                         // the block's teams, in order: one tensor at a time through LDS
        __shared__ __align__(16) float acc[TEAMS][COLS];
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
            if (pass) __syncthreads();
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (AL || i >= dup[k]) acc[team][(k * L + lane) * V - dup[k] + i] = pass ? db[k][i] : dw[k][i];
            __syncthreads();
            for (int c = threadIdx.x; c < D; c += 256) {
                float v = 0.f;
#pragma unroll 8
                for (int t = 0; t < TEAMS; ++t) v += acc[t][c];
                part[pass * D + c] = v;
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * L * TW + lane) * V;
            if (c < D) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int q = c - dup[k] + i;
                    if (AL || (i >= dup[k] && q < D)) { part[q] = dw[k][i]; part[D + q] = db[k][i]; }
                }
            }
        }
    }
}

// R rows of partials -> dw, db: 32 columns by 32 groups of rows a block, in a fixed order. 512 rows of 2 x 512 3.3 us, of
// 2 x 3136 4.8 us.
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
// Lanes and vectors of a row's team: as few idle lanes as the powers of two allow, one vector a lane where they are full, three
// where that saves a quarter of them (10 M fp32 values: D = 130 59 us with 3 x 16 lanes, 92 with 64; 17 86 with 8, 144 with
// 16), four waves beyond 1 024 columns and 16 beyond 4 096.
struct Team { int L, TW, NV; };
static Team team_of(long long D, int V) {
    const long long n = (D + V - 1) / V;               // vectors a row
    if (n <= 4) return {4, 1, 1};
    if (n <= 8) return {8, 1, 1};
    if (n <= 16) return {16, 1, 1};
    if (n <= 24) return {8, 1, 3};
    if (n <= 32) return {32, 1, 1};
    if (n <= 48) return {16, 1, 3};
    if (n > 64 && n <= 96) return {32, 1, 3};
    const int TW = D <= 1024 ? 1 : D <= 4096 ? 4 : 16;
    const int nv = (int)((n + 64 * TW - 1) / (64 * TW));
    return {64, TW, nv > 2 ? 4 : nv};
}
// blocks of the backward = rows of partials
static int norm_blocks(long long M, long long D, int V) {
    const Team t = team_of(D, V);
    const long long rows = t.TW > 1 ? M : (M + 256 / t.L - 1) / (256 / t.L);
    return (int)(rows < 512 ? rows : 512);
}

// floats of scratch of a backward pass, whichever type
DRL_API int drl_norm_ws(long long M, long long D, long long* n) {
    if (!norm_ok(M, D)) return -1;
    const int a = norm_blocks(M, D, 4), b = norm_blocks(M, D, 8);
    *n = 2 * D * (a > b ? a : b);
    return 0;
}

static bool by16(const void* q, long long stride_bytes) { return (((uintptr_t)q | (uintptr_t)stride_bytes) & 15) == 0; }

template <typename T, int NV, int L, int TW, bool AL>
static void norm_launch(const NormArgs& p, bool bwd, float eps, hipStream_t s) {
    constexpr int V = 16 / sizeof(T), threads = TW > 1 ? 64 * TW : 256;
    constexpr long long rows = TW > 1 ? 1 : 256 / L, most = 1ll << 21;   // a launch has fewer than 2^32 threads
    if (bwd) {
        k_norm_bwd<T, V, NV, L, TW, AL><<<(unsigned)norm_blocks(p.M, p.D, V), threads, 0, s>>>(p);
        return;
    }
    for (long long r = 0; r < p.M; r += most * rows) {
        NormArgs q = p;
        q.M = p.M - r < most * rows ? p.M - r : most * rows;
        q.x = (const T*)p.x + r * p.x_r;
        q.y = (T*)p.y + r * p.y_r;
        if (p.mean) { q.mean = p.mean + r; q.rstd = p.rstd + r; }
        k_norm_fwd<T, V, NV, L, TW, AL><<<(unsigned)((q.M + rows - 1) / rows), threads, 0, s>>>(q, eps);
    }
}

template <typename T, bool AL>
static void norm_team(const NormArgs& p, bool bwd, float eps, hipStream_t s) {
    const Team t = team_of(p.D, 16 / sizeof(T));
    if (t.L == 4) return norm_launch<T, 1, 4, 1, AL>(p, bwd, eps, s);
    if (t.L == 8) return t.NV == 1 ? norm_launch<T, 1, 8, 1, AL>(p, bwd, eps, s) : norm_launch<T, 3, 8, 1, AL>(p, bwd, eps, s);
    if (t.L == 16) return t.NV == 1 ? norm_launch<T, 1, 16, 1, AL>(p, bwd, eps, s) : norm_launch<T, 3, 16, 1, AL>(p, bwd, eps, s);
    if (t.L == 32) return t.NV == 1 ? norm_launch<T, 1, 32, 1, AL>(p, bwd, eps, s) : norm_launch<T, 3, 32, 1, AL>(p, bwd, eps, s);
#define NORM_NV(TW)                                                                                                   \
    if (t.NV == 1) return norm_launch<T, 1, 64, TW, AL>(p, bwd, eps, s);                                              \
    if constexpr (sizeof(T) == 4) { if (t.NV == 4) return norm_launch<T, 4, 64, TW, AL>(p, bwd, eps, s); }            \
    return norm_launch<T, 2, 64, TW, AL>(p, bwd, eps, s);
    if (t.TW == 1) { NORM_NV(1) }
    if (t.TW == 4) { NORM_NV(4) }
    NORM_NV(16)
#undef NORM_NV
}

template <typename T>
static void norm_dispatch(const NormArgs& p, bool bwd, float eps, hipStream_t s) {
    const long long e = sizeof(T);
    const bool al = p.D * e % 16 == 0 && by16(p.x, p.x_r * e) && by16(p.w, 0) && by16(p.b, 0)
                    && (bwd ? by16(p.dy, p.dy_r * e) && by16(p.dx, p.dx_r * e) : by16(p.y, p.y_r * e));
    if (al) norm_team<T, true>(p, bwd, eps, s);
    else norm_team<T, false>(p, bwd, eps, s);
}

DRL_API int drl_norm_fwd(const NormArgs* a, int bf16, float eps, hipStream_t s) {
    const NormArgs p = *a;
    if (!norm_ok(p.M, p.D)) return -1;
    const long long e = bf16 ? 2 : 4, cols = p.D * 4, rows = p.M * 4;
    if (!apart({{p.y, p.D * e, p.M, p.y_r * e}, {p.mean, rows}, {p.rstd, rows}}, {{p.x, p.D * e, p.M, p.x_r * e}, {p.w, cols}, {p.b, cols}})) return -3;
    if (bf16) norm_dispatch<bf16_t>(p, false, eps, s);
    else norm_dispatch<float>(p, false, eps, s);
    return (int)hipGetLastError();
}

DRL_API int drl_norm_bwd(const NormArgs* a, int bf16, hipStream_t s) {
    const NormArgs p = *a;
    long long need;
    if (drl_norm_ws(p.M, p.D, &need)) return -1;
    if (p.ws_n < need) return -2;
    const long long e = bf16 ? 2 : 4, cols = p.D * 4, rows = p.M * 4;
    if (!apart({{p.dx, p.D * e, p.M, p.dx_r * e}, {p.dw, cols}, {p.db, cols}, {p.ws, need * 4}},
               {{p.x, p.D * e, p.M, p.x_r * e}, {p.dy, p.D * e, p.M, p.dy_r * e}, {p.w, cols}, {p.mean, rows}, {p.rstd, rows}})) return -3;
    if (bf16) norm_dispatch<bf16_t>(p, true, 0.f, s);
    else norm_dispatch<float>(p, true, 0.f, s);
    k_norm_sum<<<(unsigned)((2 * p.D + 31) / 32), 1024, 0, s>>>(p.ws, norm_blocks(p.M, p.D, bf16 ? 8 : 4), (int)p.D, p.dw, p.db);
    return (int)hipGetLastError();
}
