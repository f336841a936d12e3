// Selective state-space scan: a recurrence with one decay per channel and state, whose step size, input and read-out are
// functions of the data. Time-major, per row b and channel d with N states:
//   s = softplus(dt + bias)   a_n = exp(s A[d,n])   h_n <- a_n h_n + s u B_n   y = (sum_n C_n h_n + D u) silu(z)
// A step whose reset flag is set starts from h = 0 (episode ends inside stored sequences); steps from lengths[b] on leave h
// alone, are not read, and write zeros.
//
// A wave owns 16 channels of one row: lane = 16 g + j holds channel j and the NS states n = NS g .. NS g + NS - 1 in
// registers and walks the time in chunks of 16 steps. What depends on (step, channel) only is computed once - lane (g, j) has
// the steps 4 i + g - and handed round through LDS; B and C of the chunk are staged in LDS as well.
#include "ssm_math.h"

#define KC 16            // steps per chunk = distance of the saved states

struct SsmArgs {         // mirrored by ops/hip.py (_ssm_args): 64-bit words in this order
    const void *u, *dt, *z, *Bm, *Cm;
    long long u_t, u_b, dt_t, dt_b, z_t, z_b, B_t, B_b, C_t, C_b;
    const float *A, *Dp, *bias, *h0;
    const unsigned char* reset;
    const int* lengths;
    void* y; long long y_t, y_b;
    float *hT, *ckpt, *ws; long long ws_n;
    long long T, B, D, N, softplus;
    // backward
    const void* dy; long long dy_t, dy_b;
    const float* dhT;
    void *du, *ddt, *dz, *dBm, *dCm;
    long long du_t, du_b, ddt_t, ddt_b, dz_t, dz_b, dB_t, dB_b, dC_t, dC_b;
    float *dA, *dD, *dbias, *dh0;
};

// LDS writes of a wave become visible to its own lanes: one wave, no barrier
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// B and C rows of a chunk -> LDS (fp32, NP = 4 NS columns each, zeros beyond N and beyond the row's end)
template <typename T, int NS>
__device__ __forceinline__ void stage_bc(const SsmArgs& p, int b, int t0, int end, int lane, float* bc) {
    constexpr int NP = 4 * NS;
#pragma unroll
    for (int k = 0; k < KC * NP / 64; ++k) {
        const int e = k * 64 + lane, s = e / NP, n = e % NP, t = t0 + s;
        const bool ok = t < end && n < p.N;
        bc[s * 2 * NP + n] = ok ? ld((const T*)p.Bm + t * p.B_t + b * p.B_b + n) : 0.f;
        bc[s * 2 * NP + NP + n] = ok ? ld((const T*)p.Cm + t * p.C_t + b * p.C_b + n) : 0.f;
    }
}

__device__ __forceinline__ unsigned reset_mask(const SsmArgs& p, int b, int t0, int end, int lane) {
    if (!p.reset) return 0;
    const int t = t0 + lane;
    return (unsigned)__ballot(lane < KC && t < end && p.reset[(long long)t * p.B + b] != 0) & 0xffffu;
}

// Sums over the four lane groups (rows of 16 lanes): group g ends with the sum of v[g]. Swapping rows adds two values at a
// time: 3 swaps + 3 adds for four sums, where a butterfly of each value would take 8 of each.
__device__ __forceinline__ float add_swap16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);     // rows a0+a1, b0+b1, a2+a3, b2+b3
}
__device__ __forceinline__ float add_swap32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);     // rows a0+a2, a1+a3, b0+b2, b1+b3
}
__device__ __forceinline__ float sum_groups(float v0, float v1, float v2, float v3) {
    return add_swap32(add_swap16(v0, v1), add_swap16(v2, v3));
}

// Keeps a value's computation where it is written: left to itself the compiler moves sums to their use, behind the next loop,
// and holds all of their terms in registers until then.
__device__ __forceinline__ void pin(float& v) { asm volatile("" : "+v"(v)); }

// Sums over the 16 lanes of a row, four at a time: quad 0 of r ends with the sum of be, quad 1 bo, quad 2 ce, quad 3 co. The
// first two levels fold two values into one register (a bank mask writes half of the quads each), so a value costs 2 adds
// instead of 4. The waits between a write and a cross-lane read of it (2 states) are the other registers' adds or s_nop.
__device__ __forceinline__ void sum_rows2(const float (&be)[2], const float (&ce)[2], const float (&bo)[2], const float (&co)[2], float (&r)[2]) {
    float t0, t1;
    asm volatile("s_nop 1\n"
        "v_add_f32_dpp %0, %4, %4 row_mirror row_mask:0xf bank_mask:0x3\n"
        "v_add_f32_dpp %1, %5, %5 row_mirror row_mask:0xf bank_mask:0x3\n"
        "v_add_f32_dpp %2, %6, %6 row_mirror row_mask:0xf bank_mask:0x3\n"
        "v_add_f32_dpp %3, %7, %7 row_mirror row_mask:0xf bank_mask:0x3\n"
        "v_add_f32_dpp %0, %8, %8 row_mirror row_mask:0xf bank_mask:0xc\n"
        "v_add_f32_dpp %1, %9, %9 row_mirror row_mask:0xf bank_mask:0xc\n"
        "v_add_f32_dpp %2, %10, %10 row_mirror row_mask:0xf bank_mask:0xc\n"
        "v_add_f32_dpp %3, %11, %11 row_mirror row_mask:0xf bank_mask:0xc\n"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(t0), "=&v"(t1)
        : "v"(be[0]), "v"(be[1]), "v"(bo[0]), "v"(bo[1]), "v"(ce[0]), "v"(ce[1]), "v"(co[0]), "v"(co[1]));
    float q0, q1;
    asm volatile("s_nop 1\n"
        "v_add_f32_dpp %0, %2, %2 row_half_mirror row_mask:0xf bank_mask:0x5\n"
        "v_add_f32_dpp %1, %3, %3 row_half_mirror row_mask:0xf bank_mask:0x5\n"
        "v_add_f32_dpp %0, %4, %4 row_half_mirror row_mask:0xf bank_mask:0xa\n"
        "v_add_f32_dpp %1, %5, %5 row_half_mirror row_mask:0xf bank_mask:0xa\n"
        "s_nop 0\n"
        "v_add_f32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
        "v_add_f32_dpp %1, %1, %1 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
        "s_nop 0\n"
        "v_add_f32_dpp %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
        "v_add_f32_dpp %1, %1, %1 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
        : "=&v"(q0), "=&v"(q1) : "v"(r[0]), "v"(r[1]), "v"(t0), "v"(t1));
    r[0] = q0; r[1] = q1;
}

// A long time axis with few rows is cut into segments that run side by side: what a segment does to the state is
// h -> P h + e with P = exp(A sum of s) and e its end state from h = 0 (k_ssm_carry), the segments are joined in order
// (k_ssm_join), and then every segment runs from its true state. The backward does the same against the time with
// G -> P G + e. ``seg`` points at [S, B, D, N] carries (nullptr: one segment), [S, B, D] sums of s follow them.
template <typename T, int NS, bool BWD>
__global__ __launch_bounds__(256) void k_ssm_carry(SsmArgs p, int seg_len, float* __restrict__ carry, float* __restrict__ sums) {
    constexpr int NP = 4 * NS;
    __shared__ __align__(16) float2 pw_s[4][KC][16];
    __shared__ __align__(16) float bc_s[4][KC * NP];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
    const int b = blockIdx.y, seg = BWD ? blockIdx.z + 1 : blockIdx.z;          // the last one (the first one) passes nothing on
    const int d = (blockIdx.x * 4 + w) * 16 + j;
    const bool dv = d < p.D;
    const int end = p.lengths ? max(0, min(p.lengths[b], (int)p.T)) : (int)p.T;
    const int ta = seg * seg_len, tb = min(ta + seg_len, (int)p.T);
    float A2[NS], h[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        A2[i] = dv && g * NS + i < p.N ? p.A[(long long)d * p.N + g * NS + i] * LOG2E : 0.f;
        h[i] = 0.f;
    }
    const float bias = dv && p.bias ? p.bias[d] : 0.f;
    float sum = 0.f;
    bool cut = false;
    const int n_chunks = (min(tb, end) - ta + KC - 1) / KC;
    for (int c = 0; c < n_chunks; ++c) {
        const int t0 = ta + (BWD ? n_chunks - 1 - c : c) * KC;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = 4 * i + g, t = t0 + s;
            const bool ok = dv && t < end;
            float v;
            if (BWD) {
                v = ok ? ld((const T*)p.dy + t * p.dy_t + b * p.dy_b + d) : 0.f;
                if (p.z && ok) { const float z = ld((const T*)p.z + t * p.z_t + b * p.z_b + d); v *= z * sigmoidf(z); }
            } else {
                v = ok ? ld((const T*)p.u + t * p.u_t + b * p.u_b + d) : 0.f;
            }
            float sp = ok ? ld((const T*)p.dt + t * p.dt_t + b * p.dt_b + d) + bias : 0.f;
            if (ok && p.softplus) sp = softplus_from(sp, exp_neg_abs(sp));
            sum += sp;
            pw_s[w][s][j] = make_float2(sp, BWD ? v : sp * v);
        }
#pragma unroll
        for (int k = 0; k < KC * NP / 64; ++k) {
            const int e = k * 64 + lane, n = e % NP, t = t0 + e / NP;
            const bool ok = t < end && n < p.N;
            bc_s[w][e] = !ok ? 0.f : BWD ? ld((const T*)p.Cm + t * p.C_t + b * p.C_b + n) : ld((const T*)p.Bm + t * p.B_t + b * p.B_b + n);
        }
        const unsigned rm = reset_mask(p, b, t0, end, lane);
        cut |= rm != 0;
        wave_sync();
#pragma unroll 4
        for (int k = 0; k < KC; ++k) {
            const int s = BWD ? KC - 1 - k : k;
            const float2 pw = pw_s[w][s][j];
            const float* bc = bc_s[w] + s * NP + g * NS;
            const bool rs = rm >> s & 1;
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const float a = __builtin_amdgcn_exp2f(pw.x * A2[i]);
                h[i] = BWD ? (rs ? 0.f : a * fmaf(pw.y, bc[i], h[i])) : fmaf(a, rs ? 0.f : h[i], pw.y * bc[i]);
            }
        }
        wave_sync();
    }
    sum += __shfl_xor(sum, 16, WAVE);
    sum += __shfl_xor(sum, 32, WAVE);
    if (!dv) return;
    const long long o = ((long long)seg * p.B + b) * p.D + d;
#pragma unroll
    for (int i = 0; i < NS; ++i) if (g * NS + i < p.N) carry[o * p.N + g * NS + i] = h[i];
    if (g == 0) sums[o] = cut ? __builtin_inff() : sum;
}

// carry[seg]: what a segment adds -> what it starts from
template <bool BWD>
__global__ __launch_bounds__(256) void k_ssm_join(SsmArgs p, int S, float* __restrict__ carry, const float* __restrict__ sums) {
    const long long n = p.B * p.D * p.N, i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long r = i / p.N;
    const float A2 = p.A[r % p.D * p.N + i % p.N] * LOG2E;
    const float* h0 = BWD ? p.dhT : p.h0;
    float h = h0 ? h0[i] : 0.f;
#pragma unroll 4
    for (int k = 0; k < S; ++k) {
        const int s = BWD ? S - 1 - k : k;
        const bool last = k == S - 1;
        const float e = last ? 0.f : carry[s * n + i], sum = last ? 0.f : sums[s * p.B * p.D + r];
        carry[s * n + i] = h;
        h = fmaf(sum == __builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(sum * A2), h, e);
    }
}

template <typename T, int NS>
__global__ __launch_bounds__(256) void k_ssm_fwd(SsmArgs p, int seg_len, const float* __restrict__ carry) {
    constexpr int NP = 4 * NS;
    __shared__ __align__(16) float2 pw_s[4][KC][16];
    __shared__ __align__(16) float bc_s[4][KC * 2 * NP];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
    const int b = blockIdx.y;
    const int d = (blockIdx.x * 4 + w) * 16 + j;
    const bool dv = d < p.D;
    const int end = p.lengths ? max(0, min(p.lengths[b], (int)p.T)) : (int)p.T;
    const long long so = ((long long)b * p.D + d) * p.N + g * NS;          // this lane's states in a [B, D, N] tensor
    float A2[NS], h[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const bool ok = dv && g * NS + i < p.N;
        A2[i] = ok ? p.A[(long long)d * p.N + g * NS + i] * LOG2E : 0.f;
        h[i] = !ok ? 0.f : carry ? carry[(long long)blockIdx.z * p.B * p.D * p.N + so + i] : p.h0 ? p.h0[so + i] : 0.f;
    }
    const float Dd = dv && p.Dp ? p.Dp[d] : 0.f, bias = dv && p.bias ? p.bias[d] : 0.f;
    const int ta = blockIdx.z * seg_len, tb = min(ta + seg_len, (int)p.T);
    for (int t0 = ta; t0 < tb; t0 += KC) {
        float u[4], zz[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = 4 * i + g, t = t0 + s;
            const bool ok = dv && t < end;
            u[i] = ok ? ld((const T*)p.u + t * p.u_t + b * p.u_b + d) : 0.f;
            zz[i] = ok && p.z ? ld((const T*)p.z + t * p.z_t + b * p.z_b + d) : 0.f;
            float sp = ok ? ld((const T*)p.dt + t * p.dt_t + b * p.dt_b + d) + bias : 0.f;
            if (ok && p.softplus) sp = softplus_from(sp, exp_neg_abs(sp));
            pw_s[w][s][j] = make_float2(sp, sp * u[i]);
        }
        stage_bc<T, NS>(p, b, t0, end, lane, bc_s[w]);
        const unsigned rm = reset_mask(p, b, t0, end, lane);
        wave_sync();
        if (p.ckpt && dv) {
            float* c = p.ckpt + (long long)(t0 / KC) * p.B * p.D * p.N + so;
#pragma unroll
            for (int i = 0; i < NS; ++i) if (g * NS + i < p.N) c[i] = h[i];
        }
        float y[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float part[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int s = 4 * q + r;
                const float2 pw = pw_s[w][s][j];
                if (rm >> s & 1) {
#pragma unroll
                    for (int i = 0; i < NS; ++i) h[i] = 0.f;
                }
                const float* bc = bc_s[w] + s * 2 * NP + g * NS;
                float acc = 0.f;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    h[i] = fmaf(__builtin_amdgcn_exp2f(pw.x * A2[i]), h[i], pw.y * bc[i]);
                    acc = fmaf(bc[NP + i], h[i], acc);
                }
                part[r] = acc;
            }
            y[q] = sum_groups(part[0], part[1], part[2], part[3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = t0 + 4 * i + g;
            if (!dv || t >= p.T) continue;
            float v = 0.f;
            if (t < end) {
                v = fmaf(Dd, u[i], y[i]);
                if (p.z) v *= zz[i] * sigmoidf(zz[i]);
            }
            st((T*)p.y + t * p.y_t + b * p.y_b + d, v);
        }
        wave_sync();                                        // the next chunk overwrites the LDS images
    }
    if (p.hT && dv && blockIdx.z == gridDim.z - 1) {
#pragma unroll
        for (int i = 0; i < NS; ++i) if (g * NS + i < p.N) p.hT[so + i] = h[i];
    }
}

// Backward. g_t = C ds + a_{t+1} g_{t+1} runs against the time; the states it needs are recomputed chunk by chunk from the
// saved ones and kept in registers (16 steps x NS, next to the decays). The sums over channels of dB and dC leave as partials
// of 64 channels (a block), the sums over rows of dA, dD and the bias as partials of a row: second launches add them in a
// fixed order.
template <typename T, int NS>
__global__ __launch_bounds__(256, 2) void k_ssm_bwd(SsmArgs p, int seg_len, const float* __restrict__ carry,
                                                    float* __restrict__ part_bc, float* __restrict__ part_a, float* __restrict__ part_d) {
    constexpr int NP = 4 * NS;
    constexpr int KH = NS > 4 ? 64 / NS : KC;               // steps whose states are held at a time
    __shared__ __align__(16) float4 pw_s[4][KC][16];
    __shared__ __align__(16) float bc_s[4][KC * 2 * NP];
    __shared__ __align__(16) float red_s[4][KC * 2 * NP];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
    const int b = blockIdx.y;
    const int d = (blockIdx.x * 4 + w) * 16 + j;
    const bool dv = d < p.D;
    const int end = p.lengths ? max(0, min(p.lengths[b], (int)p.T)) : (int)p.T;
    const long long so = ((long long)b * p.D + d) * p.N + g * NS;
    float An[NS], G[NS], dA[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const bool ok = dv && g * NS + i < p.N;
        An[i] = ok ? p.A[(long long)d * p.N + g * NS + i] : 0.f;
        // a_{t+1} g_{t+1}: dL/dh_t from the steps behind
        G[i] = !ok ? 0.f : carry ? carry[(long long)blockIdx.z * p.B * p.D * p.N + so + i] : p.dhT ? p.dhT[so + i] : 0.f;
        dA[i] = 0.f;
    }
    const float Dd = dv && p.Dp ? p.Dp[d] : 0.f, bias = dv && p.bias ? p.bias[d] : 0.f;
    float dD = 0.f, dbias = 0.f;
    const int ta = blockIdx.z * seg_len, tb = min(ta + seg_len, (int)p.T);
    for (int t0 = ta + (tb - ta - 1) / KC * KC; t0 >= ta; t0 -= KC) {
        float u[4], zz[4], dy[4], sp[4], sg[4], ds[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = 4 * i + g, t = t0 + s;
            const bool ok = dv && t < end;
            u[i] = ok ? ld((const T*)p.u + t * p.u_t + b * p.u_b + d) : 0.f;
            zz[i] = ok && p.z ? ld((const T*)p.z + t * p.z_t + b * p.z_b + d) : 0.f;
            dy[i] = ok ? ld((const T*)p.dy + t * p.dy_t + b * p.dy_b + d) : 0.f;
            sp[i] = ok ? ld((const T*)p.dt + t * p.dt_t + b * p.dt_b + d) + bias : 0.f;
            sg[i] = ok ? 1.f : 0.f;
            if (ok && p.softplus) {
                const float e = exp_neg_abs(sp[i]);
                sg[i] = sigmoid_from(sp[i], e);
                sp[i] = softplus_from(sp[i], e);
            }
            ds[i] = p.z ? dy[i] * zz[i] * sigmoidf(zz[i]) : dy[i];
            pw_s[w][s][j] = make_float4(sp[i], sp[i] * u[i], ds[i], 0.f);
        }
        stage_bc<T, NS>(p, b, t0, end, lane, bc_s[w]);
        const unsigned rm = reset_mask(p, b, t0, end, lane);
        wave_sync();
        float yq[4], gb[4], wa[4], dAc[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) dAc[i] = 0.f;
        // pieces of KH steps, last one first: the states are run up to the piece, then kept through it
        for (int s0 = KC - KH; s0 >= 0; s0 -= KH) {
            float hs[KH + 1][NS], a[KH][NS];
            const float* c = p.ckpt + (long long)(t0 / KC) * p.B * p.D * p.N + so;
#pragma unroll
            for (int i = 0; i < NS; ++i) hs[0][i] = dv && g * NS + i < p.N ? c[i] : 0.f;
            for (int s = 0; s < s0; ++s) {
                const float4 pw = pw_s[w][s][j];
                const float* bc = bc_s[w] + s * 2 * NP + g * NS;
                const bool rs = rm >> s & 1;
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    hs[0][i] = fmaf(__builtin_amdgcn_exp2f(pw.x * (An[i] * LOG2E)), rs ? 0.f : hs[0][i], pw.y * bc[i]);
            }
            float part[4];
#pragma unroll
            for (int k = 0; k < KH; ++k) {
                const int s = s0 + k;
                const float4 pw = pw_s[w][s][j];
                const float* bc = bc_s[w] + s * 2 * NP + g * NS;
                const bool rs = rm >> s & 1;                // hs[k] stays: dC of the step before needs it
                float acc = 0.f;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    a[k][i] = __builtin_amdgcn_exp2f(pw.x * (An[i] * LOG2E));
                    hs[k + 1][i] = fmaf(a[k][i], rs ? 0.f : hs[k][i], pw.y * bc[i]);
                    acc = fmaf(bc[NP + i], hs[k + 1][i], acc);
                }
                part[k & 3] = acc;
                if ((k & 3) == 3) {
                    float sy = sum_groups(part[0], part[1], part[2], part[3]);
                    pin(sy);
#pragma unroll
                    for (int i = 0; i < 4; ++i) if (i == s / 4) yq[i] = sy;
                }
            }
            int again = 0;                                  // hides that B, C and the step's scalars are read a second time:
            asm volatile("" : "+v"(again));                 // kept from the first, they would fill the registers
            float pb[4], pa[4];
#pragma unroll
            for (int k = KH - 2; k >= 0; k -= 2) {          // two steps at a time: k + 1, then k
                float vB[2][NS], vC[2][NS];
#pragma unroll
                for (int o = 1; o >= 0; --o) {
                    const int s = s0 + k + o, c = (k + o) & 3;
                    const float4 pw = pw_s[w][s][j + again];
                    const float* bc = bc_s[w] + s * 2 * NP + g * NS + again;
                    const bool rs = rm >> s & 1;
                    pb[c] = 0.f; pa[c] = 0.f;
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        const float gh = fmaf(pw.z, bc[NP + i], G[i]);
                        vB[o][i] = gh * pw.y;
                        vC[o][i] = pw.z * hs[k + o + 1][i];
                        pb[c] = fmaf(gh, bc[i], pb[c]);
                        const float q = rs ? 0.f : gh * a[k + o][i], x = q * hs[k + o][i];
                        G[i] = q;
                        pa[c] = fmaf(x, An[i], pa[c]);
                        dAc[i] = fmaf(x, pw.x, dAc[i]);
                        pin(dAc[i]);
                    }
                    pin(pb[c]); pin(pa[c]);
                }
                float* red = red_s[w] + (s0 + k + (j >> 2 & 1)) * 2 * NP + (j >> 3) * NP + g * NS;
#pragma unroll
                for (int i = 0; i < NS; i += 2) {
                    float r[2];
                    sum_rows2({vB[0][i], vB[0][i + 1]}, {vC[0][i], vC[0][i + 1]}, {vB[1][i], vB[1][i + 1]}, {vC[1][i], vC[1][i + 1]}, r);
                    if ((j & 3) == 0) { red[i] = r[0]; red[i + 1] = r[1]; }
                }
                if ((k & 3) == 0) {
                    float sb = sum_groups(pb[0], pb[1], pb[2], pb[3]), sa = sum_groups(pa[0], pa[1], pa[2], pa[3]);
                    pin(sb); pin(sa);
#pragma unroll
                    for (int i = 0; i < 4; ++i) if (i == (s0 + k) / 4) { gb[i] = sb; wa[i] = sa; }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) dA[i] += dAc[i];
        float dDc = 0.f, dbc = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = t0 + 4 * i + g;
            const float dpre = fmaf(u[i], gb[i], wa[i]) * sg[i];
            dDc = fmaf(ds[i], u[i], dDc);
            dbc += dpre;
            if (!dv || t >= p.T) continue;
            st((T*)p.du + t * p.du_t + b * p.du_b + d, fmaf(Dd, ds[i], sp[i] * gb[i]));
            st((T*)p.ddt + t * p.ddt_t + b * p.ddt_b + d, dpre);
            if (p.z) {
                const float sz = sigmoidf(zz[i]);
                st((T*)p.dz + t * p.dz_t + b * p.dz_b + d, t < end ? dy[i] * fmaf(Dd, u[i], yq[i]) * sz * (1.f + zz[i] * (1.f - sz)) : 0.f);
            }
        }
        dD += dDc; dbias += dbc;
        __syncthreads();
        for (int e = threadIdx.x; e < KC * 2 * NP; e += 256) {
            const int t = t0 + e / (2 * NP);
            if (t < p.T)
                part_bc[(((long long)t * p.B + b) * gridDim.x + blockIdx.x) * (2 * NP) + e % (2 * NP)] =
                    (red_s[0][e] + red_s[1][e]) + (red_s[2][e] + red_s[3][e]);
        }
        __syncthreads();
    }
    dD += __shfl_xor(dD, 16, WAVE); dD += __shfl_xor(dD, 32, WAVE);
    dbias += __shfl_xor(dbias, 16, WAVE); dbias += __shfl_xor(dbias, 32, WAVE);
    if (!dv) return;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        if (g * NS + i >= p.N) continue;
        part_a[(long long)blockIdx.z * p.B * p.D * p.N + so + i] = dA[i];
        if (p.dh0 && blockIdx.z == 0) p.dh0[so + i] = G[i];
    }
    if (g == 0) {
        const long long r = (long long)blockIdx.z * p.B + b;
        part_d[r * p.D + d] = dD;
        part_d[((long long)gridDim.z * p.B + r) * p.D + d] = dbias;
    }
}

// out[i] = sum over r < R of part[r][i], in order
__global__ void k_sum_rows(const float* __restrict__ part, int R, long long n, float* __restrict__ out) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    float v = 0.f;
    for (int r = 0; r < R; ++r) v += part[r * n + i];
    out[i] = v;
}
template <typename T>
__global__ void k_ssm_sum_bc(SsmArgs p, const float* __restrict__ part, int nblk, int NP) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long row = i / (2 * p.N);
    if (row >= p.T * p.B) return;
    const int c = (int)(i % (2 * p.N)), isC = c >= p.N, n = isC ? c - (int)p.N : c;
    const float* q = part + row * nblk * 2 * NP + isC * NP + n;
    float v = 0.f;
    for (int k = 0; k < nblk; ++k) v += q[(long long)k * 2 * NP];
    const long long t = row / p.B, b = row % p.B;
    if (isC) st((T*)p.dCm + t * p.dC_t + b * p.dC_b + n, v);
    else st((T*)p.dBm + t * p.dB_t + b * p.dB_b + n, v);
}

// One step: h [B, D, N] is read and written once, the rest is small. A thread per (row, channel).
template <typename T>
__global__ __launch_bounds__(256) void k_ssm_step(SsmArgs p) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= p.B * p.D) return;
    const long long b = i / p.D, d = i - b * p.D;
    const float u = ld((const T*)p.u + b * p.u_b + d);
    float sp = ld((const T*)p.dt + b * p.dt_b + d) + (p.bias ? p.bias[d] : 0.f);
    if (p.softplus) sp = softplus_from(sp, exp_neg_abs(sp));
    const bool rs = p.reset && p.reset[b] != 0;
    float y = 0.f;
    for (int n = 0; n < p.N; ++n) {
        float* hp = p.hT + i * p.N + n;
        const float h = fmaf(__builtin_amdgcn_exp2f(sp * (p.A[d * p.N + n] * LOG2E)), rs ? 0.f : *hp,
                             sp * u * ld((const T*)p.Bm + b * p.B_b + n));
        *hp = h;
        y = fmaf(ld((const T*)p.Cm + b * p.C_b + n), h, y);
    }
    if (p.Dp) y = fmaf(p.Dp[d], u, y);
    if (p.z) { const float z = ld((const T*)p.z + b * p.z_b + d); y *= z * sigmoidf(z); }
    st((T*)p.y + b * p.y_b + d, y);
}

static int ns_of(long long N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

// Segments: one where the rows alone give the chip 768 waves, else as many as bring it to 2 048, of at least 64 steps. A cut
// costs the carry pass (the recurrence without its read-out), so rows that fill the chip are never cut.
struct Segs { int n, len; };
static Segs segments(long long T, long long B, long long D) {
    const long long waves = (D + 15) / 16 * B, chunks = (T + KC - 1) / KC;
    long long n = 1;
    if (waves < 768) {
        n = (2048 + waves - 1) / waves;
        if (n > chunks / 4) n = chunks / 4;
        if (n < 1) n = 1;
    }
    const long long len = (chunks + n - 1) / n * KC;
    return {(int)((T + len - 1) / len), (int)len};
}

// floats of scratch that a forward (train = 0) or a forward and its backward (1) need
DRL_API int drl_ssm_ws(long long T, long long B, long long D, long long N, int train, long long* n) {
    if (T <= 0 || T >= (1ll << 31) || B <= 0 || D <= 0 || N <= 0 || N > 64 || B > 65535) return -1;
    const long long nblk = (D + 63) / 64, S = segments(T, B, D).n;
    *n = S > 1 ? S * B * D * (N + 1) : 0;
    if (train) *n += T * B * nblk * 8 * ns_of(N) + S * B * D * (N + 2);
    return 0;
}

template <typename T, int NS, bool BWD>
static const float* launch_carry(const SsmArgs& p, Segs sg, hipStream_t s) {
    if (sg.n == 1) return nullptr;
    float *carry = p.ws, *sums = carry + sg.n * p.B * p.D * p.N;
    k_ssm_carry<T, NS, BWD><<<dim3((unsigned)((p.D + 63) / 64), (unsigned)p.B, (unsigned)(sg.n - 1)), 256, 0, s>>>(p, sg.len, carry, sums);
    k_ssm_join<BWD><<<(unsigned)((p.B * p.D * p.N + 255) / 256), 256, 0, s>>>(p, sg.n, carry, sums);
    return carry;
}

template <typename T, int NS>
static void launch_fwd(const SsmArgs& p, hipStream_t s) {
    const Segs sg = segments(p.T, p.B, p.D);
    const float* carry = launch_carry<T, NS, false>(p, sg, s);
    k_ssm_fwd<T, NS><<<dim3((unsigned)((p.D + 63) / 64), (unsigned)p.B, (unsigned)sg.n), 256, 0, s>>>(p, sg.len, carry);
}

template <typename T, int NS>
static void launch_bwd(const SsmArgs& p, hipStream_t s) {
    const Segs sg = segments(p.T, p.B, p.D);
    const float* carry = launch_carry<T, NS, true>(p, sg, s);
    const int nblk = (int)((p.D + 63) / 64), NP = 4 * NS;
    const long long rows = sg.n * p.B;
    float* part_bc = p.ws + (sg.n > 1 ? rows * p.D * (p.N + 1) : 0);
    float* part_a = part_bc + p.T * p.B * nblk * 2 * NP;
    float* part_d = part_a + rows * p.D * p.N;
    k_ssm_bwd<T, NS><<<dim3((unsigned)nblk, (unsigned)p.B, (unsigned)sg.n), 256, 0, s>>>(p, sg.len, carry, part_bc, part_a, part_d);
    const long long nbc = p.T * p.B * 2 * p.N, na = p.D * p.N;
    k_ssm_sum_bc<T><<<(unsigned)((nbc + 255) / 256), 256, 0, s>>>(p, part_bc, nblk, NP);
    k_sum_rows<<<(unsigned)((na + 255) / 256), 256, 0, s>>>(part_a, (int)rows, na, p.dA);
    if (p.dD) k_sum_rows<<<(unsigned)((p.D + 255) / 256), 256, 0, s>>>(part_d, (int)rows, p.D, p.dD);
    if (p.dbias) k_sum_rows<<<(unsigned)((p.D + 255) / 256), 256, 0, s>>>(part_d + rows * p.D, (int)rows, p.D, p.dbias);
}

#define SSM_NS(NAME, T)                       \
    switch (ns_of(p.N)) {                     \
        case 2: NAME<T, 2>(p, s); break;      \
        case 4: NAME<T, 4>(p, s); break;      \
        case 8: NAME<T, 8>(p, s); break;      \
        default: NAME<T, 16>(p, s); break;    \
    }

DRL_API int drl_ssm_fwd(const SsmArgs* a, int bf16, hipStream_t s) {
    const SsmArgs p = *a;
    long long need;
    if (drl_ssm_ws(p.T, p.B, p.D, p.N, 0, &need)) return -1;
    if (p.ws_n < need) return -2;
    if (bf16) { SSM_NS(launch_fwd, bf16_t) } else { SSM_NS(launch_fwd, float) }
    return (int)hipGetLastError();
}

DRL_API int drl_ssm_bwd(const SsmArgs* a, int bf16, hipStream_t s) {
    const SsmArgs p = *a;
    long long need;
    if (drl_ssm_ws(p.T, p.B, p.D, p.N, 1, &need) || !p.ckpt) return -1;
    if (p.ws_n < need) return -2;
    if (bf16) { SSM_NS(launch_bwd, bf16_t) } else { SSM_NS(launch_bwd, float) }
    return (int)hipGetLastError();
}

DRL_API int drl_ssm_step(const SsmArgs* a, int bf16, hipStream_t s) {
    const SsmArgs p = *a;
    if (p.B <= 0 || p.D <= 0 || p.N <= 0 || p.N > 64) return -1;
    const long long nb = (p.B * p.D + 255) / 256;
    if (nb > 0x7fffffffll) return -1;
    if (bf16) k_ssm_step<bf16_t><<<(unsigned)nb, 256, 0, s>>>(p);
    else k_ssm_step<float><<<(unsigned)nb, 256, 0, s>>>(p);
    return (int)hipGetLastError();
}
