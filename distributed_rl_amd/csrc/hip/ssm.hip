// Selective state-space scan: a recurrence with one decay per channel and state, whose step size, input and read-out are
// functions of the data. Time-major, per row b and channel d with N states:
//   s = softplus(dt + bias)   a_n = exp(s A[d,n])   h_n <- a_n h_n + s u B_n   y = (sum_n C_n h_n + D u) silu(z)
// A step whose reset flag is set starts from h = 0 (episode ends inside stored sequences); steps from lengths[b] on leave h
// alone, are not read, and write zeros.
//
// A wave owns 16 channels of one row: lane = 16 g + j holds channel j and the NS states n = NS g .. NS g + NS - 1 in
// registers and walks the time in chunks of 16 steps. What depends on (step, channel) only is computed once - lane (g, j) has
// the steps 4 i + g - and handed round through LDS; B and C of the chunk are staged in LDS as well.
//
// Bound by vector issue: a state and step cost an exp (2.5 issue slots) and four more instructions forward, an exp and twelve
// backward. Four lanes a channel keep 16 states at 4 registers a lane of each kind, and the sums over states at a row swap and
// an add a step.
#include "apart.h"
#include "ssm_math.h"
#include <type_traits>

#define KC 16            // steps per chunk
#define SAVE 8           // distance of the states that the forward saves for the backward (ops/hip.py SSM_SAVE)

struct SsmArgs {         // mirrored by ops/hip.py (_SSM): 64-bit words in this order
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
// a barrier that orders LDS only: loads and stores of global memory stay in flight
__device__ __forceinline__ void block_sync_lds() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Rows of a chunk of a [T, B, C] tensor through a buffer descriptor: uniform 64-bit base of the chunk's first step, 32-bit
// offsets inside the chunk. A lane whose element does not exist takes the offset OOB: its load gives 0 and its store does
// nothing, without a branch.
#define OOB 0x80000000u
template <typename T>
struct Rows {
    const char* base;            // the chunk's first step of row b
    unsigned four;               // bytes over 4 steps (the host keeps 16 steps under 2^31 bytes)
    __device__ __forceinline__ Rows(const void* q, long long st, long long sb, int b, int t0)
        : base((const char*)q + (t0 * st + b * sb) * (long long)sizeof(T)), four((unsigned)st * (unsigned)(4 * sizeof(T))) {}
    __device__ __forceinline__ void next() { base += 4ull * four; }
    __device__ __forceinline__ void back() { base -= 4ull * four; }
    __device__ __forceinline__ auto rsrc() const { return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000); }
    static __device__ __forceinline__ unsigned offset(long long st, int s, long long c) { return ((unsigned)s * (unsigned)st + (unsigned)c) * (unsigned)sizeof(T); }
    template <typename R> static __device__ __forceinline__ unsigned load(R r, unsigned voff, unsigned soff) {
        if constexpr (sizeof(T) == 2) return (unsigned)__builtin_amdgcn_raw_buffer_load_b16(r, voff, soff, 0);
        else return __builtin_amdgcn_raw_buffer_load_b32(r, voff, soff, 0);
    }
    static __device__ __forceinline__ float value(unsigned raw) { return __uint_as_float(sizeof(T) == 2 ? raw << 16 : raw); }
    template <typename R> static __device__ __forceinline__ void store(R r, unsigned voff, unsigned soff, float v) {
        if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16((short)f2bf(v), r, voff, soff, 0);
        else __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, voff, soff, 0);
    }
};

// What a block of four waves needs of B and C in a chunk: NV values of each per thread, fetched ahead and written to LDS as
// fp32, [step][B: NP | C: NP], zeros beyond N and beyond the row's end. WHICH: 1 = B, 2 = C, 3 = both.
template <typename T, int NS, int WHICH>
struct StageBC {
    static constexpr int NP = 4 * NS, STEP = 256 / NP < KC ? 256 / NP : KC, NV = (KC + STEP - 1) / STEP, ROW = WHICH == 3 ? 2 * NP : NP;
    Rows<T> B, C;
    unsigned ob, oc, rb[WHICH & 1 ? NV : 1], rc[WHICH & 2 ? NV : 1];
    __device__ __forceinline__ StageBC(const SsmArgs& p, int b, int t0)
        : B(p.Bm, p.B_t, p.B_b, b, t0), C(p.Cm, p.C_t, p.C_b, b, t0) {
        const int n = threadIdx.x % NP, s = threadIdx.x / NP;
        const bool in = n < p.N && s < STEP;
        ob = in ? Rows<T>::offset(p.B_t, s, n) : OOB;
        oc = in ? Rows<T>::offset(p.C_t, s, n) : OOB;
    }
    // live: steps of the chunk before the row's end
    __device__ __forceinline__ void fetch(int live) {
        const int s = threadIdx.x / NP;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const unsigned bad = s + k * STEP < min(live, KC) ? 0u : OOB;
            if (WHICH & 1) rb[k] = Rows<T>::load(B.rsrc(), ob | bad, k * STEP * (B.four / 4));
            if (WHICH & 2) rc[k] = Rows<T>::load(C.rsrc(), oc | bad, k * STEP * (C.four / 4));
        }
    }
    __device__ __forceinline__ void put(float* bc) const {
        const int n = threadIdx.x % NP, s = threadIdx.x / NP;
        if (s >= STEP) return;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (KC % STEP && s + k * STEP >= KC) break;
            float* q = bc + (s + k * STEP) * ROW + n;
            if (WHICH & 1) *q = Rows<T>::value(rb[k]);
            if (WHICH & 2) q[WHICH == 3 ? NP : 0] = Rows<T>::value(rc[k]);
        }
    }
};
// NS consecutive values of an LDS image
template <int NS>
__device__ __forceinline__ void lds_row(const float* q, float (&v)[NS]) {
    if constexpr (NS % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NS; i += 4) { const float4 x = *reinterpret_cast<const float4*>(q + i); v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w; }
    } else if constexpr (NS == 2) {
        const float2 x = *reinterpret_cast<const float2*>(q);
        v[0] = x.x; v[1] = x.y;
    } else {
        v[0] = *q;
    }
}

// reset flags of a chunk, one byte in each of the first 16 lanes, and as a bit mask
__device__ __forceinline__ unsigned fetch_resets(const SsmArgs& p, int b, int t0, int end, int lane) {
    if (!p.reset) return 0;
    const int t = t0 + (lane & 15);
    return t < end ? p.reset[(long long)t * p.B + b] : 0;
}
__device__ __forceinline__ unsigned reset_mask(unsigned flag) { return (unsigned)__ballot(flag != 0) & 0xffffu; }

__device__ __forceinline__ int row_end(const SsmArgs& p, int b) { return p.lengths ? max(0, min(p.lengths[b], (int)p.T)) : (int)p.T; }

// The row of a block. Rows of unequal length are taken longest first, so that no long one starts when the others are through
// (120 x 64 x 1024, lengths of 30 .. 120: backward 120 us instead of 147): slot k of the grid gets the row with k longer ones, found by
// counting, 256 rows at most.
#define SORT_ROWS 256
__device__ __forceinline__ int block_row(const SsmArgs& p, int* len_s) {
    const int slot = blockIdx.y, B = (int)p.B;
    if (!p.lengths || B > SORT_ROWS) return slot;
    const int r = threadIdx.x;
    if (r < B) len_s[r] = p.lengths[r];
    __syncthreads();
    if (r < B) {
        const int mine = len_s[r];
        int rank = 0;
        for (int k = 0; k < B; ++k) rank += len_s[k] > mine || (len_s[k] == mine && k < r);
        if (rank == slot) len_s[SORT_ROWS] = r;
    }
    __syncthreads();
    const int b = __builtin_amdgcn_readfirstlane(len_s[SORT_ROWS]);
    __syncthreads();                                        // len_s is another array's memory
    return b;
}

// the states of a lane in a [.., B, D, N] tensor, four at a time (v4: N and the tensor's address allow it, see vec4)
__host__ __device__ __forceinline__ bool vec4(const float* q, long long N) { return (N & 3) == 0 && ((uintptr_t)q & 15) == 0; }
template <int NS>
__device__ __forceinline__ void put_states(float* q, const float (&h)[NS], int n0, int N, bool v4) {
    if (NS % 4 == 0 && v4) {
#pragma unroll
        for (int i = 0; i + 3 < NS; i += 4) if (n0 + i < N) *reinterpret_cast<float4*>(q + i) = make_float4(h[i], h[i + 1], h[i + 2], h[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < NS; ++i) if (n0 + i < N) q[i] = h[i];
    }
}
template <int NS>
__device__ __forceinline__ void get_states(const float* q, float (&h)[NS], int n0, int N, bool ok, bool v4) {
#pragma unroll
    for (int i = 0; i < NS; ++i) h[i] = 0.f;
    if (!ok) return;
    if (NS % 4 == 0 && v4) {
#pragma unroll
        for (int i = 0; i + 3 < NS; i += 4)
            if (n0 + i < N) { const float4 v = *reinterpret_cast<const float4*>(q + i); h[i] = v.x; h[i + 1] = v.y; h[i + 2] = v.z; h[i + 3] = v.w; }
    } else {
#pragma unroll
        for (int i = 0; i < NS; ++i) if (n0 + i < N) h[i] = q[i];
    }
}

// Sums over the four lane groups (rows of 16 lanes): group g ends with the sum of v[g]. Swapping rows adds two values at a
// time: 3 swaps + 3 adds for four sums, where a butterfly of each value would take 8 of each.
__device__ __forceinline__ float sum_groups(float v0, float v1, float v2, float v3) {
    return add_swap32(add_swap16(v0, v1), add_swap16(v2, v3));
}

// Keeps a value's computation where it is written: left to itself the compiler moves sums to their use, behind the next loop,
// and holds all of their terms in registers until then.
__device__ __forceinline__ void pin(float& v) { asm volatile("" : "+v"(v)); }

// Sums over the 16 lanes of a row, NS x 4 of them at a time: quad 0 holds the sums of be, quad 1 bo, quad 2 ce, quad 3 co, and
// lane q of a quad the one of index q (q & 1 where there are two, any lane where there is one). Every level folds two values into one register - by
// bank masks, which write half of the quads each, or within quads by exchanging what the other lane keeps - so a value costs
// 2 to 2.3 instructions instead of 4 adds. Between a write and a cross-lane read of it there are 2 wait states: the other
// registers' adds, or s_nop.
#define DPP(D, S, CTRL, BANK) "v_add_f32_dpp %" #D ", %" #S ", %" #S " " CTRL " row_mask:0xf bank_mask:" BANK "\n"
template <int CTRL>
__device__ __forceinline__ float quad_fold(bool odd, float v0, float v1) {
    const float keep = odd ? v1 : v0, give = odd ? v0 : v1;
    return keep + __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(give), CTRL, 0xf, 0xf, true));
}
#define QUAD_XOR1 0xB1
#define QUAD_XOR2 0x4E
template <int CTRL>
__device__ __forceinline__ float quad_add(float v) { return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true)); }
__device__ __forceinline__ float sum_rows1(const float* be, const float* ce, const float* bo, const float* co) {
    float t0, t1, r;
    asm volatile("s_nop 1\n"
        DPP(0, 2, "row_mirror", "0x3") DPP(1, 3, "row_mirror", "0x3") DPP(0, 4, "row_mirror", "0xc") DPP(1, 5, "row_mirror", "0xc")
        : "=&v"(t0), "=&v"(t1) : "v"(be[0]), "v"(bo[0]), "v"(ce[0]), "v"(co[0]));
    asm volatile("s_nop 1\n" DPP(0, 1, "row_half_mirror", "0x5") DPP(0, 2, "row_half_mirror", "0xa") "s_nop 1\n"
        : "=&v"(r) : "v"(t0), "v"(t1));
    return quad_add<QUAD_XOR2>(quad_add<QUAD_XOR1>(r));
}
__device__ __forceinline__ float sum_rows2(const float* be, const float* ce, const float* bo, const float* co, int j) {
    float t0, t1, t2, t3, r0, r1;
    asm volatile("s_nop 1\n"
        DPP(0, 4, "row_mirror", "0x3") DPP(1, 5, "row_mirror", "0x3") DPP(2, 6, "row_mirror", "0x3") DPP(3, 7, "row_mirror", "0x3")
        DPP(0, 8, "row_mirror", "0xc") DPP(1, 9, "row_mirror", "0xc") DPP(2, 10, "row_mirror", "0xc") DPP(3, 11, "row_mirror", "0xc")
        : "=&v"(t0), "=&v"(t1), "=&v"(t2), "=&v"(t3)
        : "v"(be[0]), "v"(be[1]), "v"(bo[0]), "v"(bo[1]), "v"(ce[0]), "v"(ce[1]), "v"(co[0]), "v"(co[1]));
    asm volatile("s_nop 1\n"
        DPP(0, 2, "row_half_mirror", "0x5") DPP(1, 3, "row_half_mirror", "0x5")
        DPP(0, 4, "row_half_mirror", "0xa") DPP(1, 5, "row_half_mirror", "0xa") "s_nop 1\n"
        : "=&v"(r0), "=&v"(r1) : "v"(t0), "v"(t1), "v"(t2), "v"(t3));
    return quad_add<QUAD_XOR2>(quad_fold<QUAD_XOR1>(j & 1, r0, r1));
}
__device__ __forceinline__ float sum_rows4(const float* be, const float* ce, const float* bo, const float* co, int j) {
    float t[8], r[4];
    asm volatile("s_nop 1\n"
        DPP(0, 8, "row_mirror", "0x3") DPP(1, 9, "row_mirror", "0x3") DPP(2, 10, "row_mirror", "0x3") DPP(3, 11, "row_mirror", "0x3")
        DPP(4, 12, "row_mirror", "0x3") DPP(5, 13, "row_mirror", "0x3") DPP(6, 14, "row_mirror", "0x3") DPP(7, 15, "row_mirror", "0x3")
        DPP(0, 16, "row_mirror", "0xc") DPP(1, 17, "row_mirror", "0xc") DPP(2, 18, "row_mirror", "0xc") DPP(3, 19, "row_mirror", "0xc")
        DPP(4, 20, "row_mirror", "0xc") DPP(5, 21, "row_mirror", "0xc") DPP(6, 22, "row_mirror", "0xc") DPP(7, 23, "row_mirror", "0xc")
        : "=&v"(t[0]), "=&v"(t[1]), "=&v"(t[2]), "=&v"(t[3]), "=&v"(t[4]), "=&v"(t[5]), "=&v"(t[6]), "=&v"(t[7])
        : "v"(be[0]), "v"(be[1]), "v"(be[2]), "v"(be[3]), "v"(bo[0]), "v"(bo[1]), "v"(bo[2]), "v"(bo[3]),
          "v"(ce[0]), "v"(ce[1]), "v"(ce[2]), "v"(ce[3]), "v"(co[0]), "v"(co[1]), "v"(co[2]), "v"(co[3]));
    asm volatile("s_nop 1\n"
        DPP(0, 4, "row_half_mirror", "0x5") DPP(1, 5, "row_half_mirror", "0x5") DPP(2, 6, "row_half_mirror", "0x5") DPP(3, 7, "row_half_mirror", "0x5")
        DPP(0, 8, "row_half_mirror", "0xa") DPP(1, 9, "row_half_mirror", "0xa") DPP(2, 10, "row_half_mirror", "0xa") DPP(3, 11, "row_half_mirror", "0xa")
        "s_nop 1\n"                               // what follows may read the sums across lanes
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
        : "v"(t[0]), "v"(t[1]), "v"(t[2]), "v"(t[3]), "v"(t[4]), "v"(t[5]), "v"(t[6]), "v"(t[7]));
    return quad_fold<QUAD_XOR2>(j & 2, quad_fold<QUAD_XOR1>(j & 1, r[0], r[1]), quad_fold<QUAD_XOR1>(j & 1, r[2], r[3]));
}
#undef DPP

// A long time axis with few rows is cut into segments that run side by side: what a segment does to the state is
// h -> P h + e with P = exp(A sum of s) and e its end state from h = 0 (k_ssm_carry), the segments are joined in order
// (k_ssm_join), and then every segment runs from its true state. The backward does the same against the time with
// G -> P G + e. ``carry`` points at [S, B, D, N] carries (nullptr: one segment), [S, B, D] sums of s follow them. 4096 x 2 x 1024
// fp32, 16 states: 36 us (38 backward) beside 51 (147) of the true pass and 6 (8) of the join.
template <typename T, int NS, bool BWD>
__global__ __launch_bounds__(256) void k_ssm_carry(SsmArgs p, int seg_len, float* __restrict__ carry, float* __restrict__ sums) {
    constexpr int NP = 4 * NS;
    using R = Rows<T>;
    __shared__ __align__(16) float2 pw_s[4][KC][16];
    __shared__ __align__(16) float bc_s[2][KC * NP];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
    const int b = blockIdx.y, seg = BWD ? blockIdx.z + 1 : blockIdx.z;          // the last one (the first one) passes nothing on
    const int d = (blockIdx.x * 4 + w) * 16 + j;
    const bool dv = d < p.D;
    const int end = row_end(p, b), ta = seg * seg_len, tb = min(ta + seg_len, (int)p.T);
    float A2[NS], h[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        A2[i] = dv && g * NS + i < p.N ? rate(p.A[(long long)d * p.N + g * NS + i], LOG2E) : 0.f;
        h[i] = 0.f;
    }
    const float bias = dv && p.bias ? p.bias[d] : 0.f;
    const void* v_p = BWD ? p.dy : p.u;
    const long long v_t = BWD ? p.dy_t : p.u_t, v_b = BWD ? p.dy_b : p.u_b;
    const unsigned ov = R::offset(v_t, g, d), od = R::offset(p.dt_t, g, d), oz = R::offset(p.z_t, g, d);
    const int n_chunks = max(0, (min(tb, end) - ta + KC - 1) / KC);
    float sum = 0.f;
    bool cut = false;
    const bool has_z = p.z != nullptr, soft = p.softplus != 0;
    unsigned rv[4], rd[4], rz[4], rr;
    const int t_first = BWD ? ta + max(0, n_chunks - 1) * KC : ta;
    R xv(v_p, v_t, v_b, b, t_first), xd(p.dt, p.dt_t, p.dt_b, b, t_first), xz(p.z, p.z_t, p.z_b, b, t_first);
    StageBC<T, NS, BWD ? 2 : 1> st(p, b, t_first);
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned bad = dv && t0 + 4 * i + g < end ? 0u : OOB;
            rv[i] = R::load(xv.rsrc(), ov | bad, i * xv.four);
            rd[i] = R::load(xd.rsrc(), od | bad, i * xd.four);
            if (BWD && has_z) rz[i] = R::load(xz.rsrc(), oz | bad, i * xz.four);
        }
        st.fetch(end - t0);
        rr = fetch_resets(p, b, t0, end, lane);
        if (BWD) { xv.back(); xd.back(); xz.back(); st.C.back(); } else { xv.next(); xd.next(); st.B.next(); }
    };
    if (n_chunks) fetch(t_first);
    for (int c = 0; c < n_chunks; ++c) {
        const int t0 = ta + (BWD ? n_chunks - 1 - c : c) * KC;
        // the flags are asked once, outside: the four elements' chains of operations then overlap
        float v[4], sp[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = R::value(rv[i]); sp[i] = R::value(rd[i]) + bias; }
        if (BWD && has_z) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { const float z = R::value(rz[i]); v[i] *= z * sigmoidf(z); }
        }
        if (soft) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sp[i] = softplus(sp[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sp[i] = dv && t0 + 4 * i + g < end ? sp[i] : 0.f;
            sum += sp[i];
            pw_s[w][4 * i + g][j] = make_float2(sp[i], BWD ? v[i] : sp[i] * v[i]);
        }
        float* bcb = bc_s[c & 1];
        st.put(bcb);
        const unsigned rm = reset_mask(rr);
        cut |= rm != 0;
        if (c + 1 < n_chunks) fetch(BWD ? t0 - KC : t0 + KC);
        block_sync_lds();
        auto steps = [&](auto has) {
#pragma unroll 4
            for (int k = 0; k < KC; ++k) {
                const int s = BWD ? KC - 1 - k : k;
                const float2 pw = pw_s[w][s][j];
                float bc[NS];
                lds_row<NS>(bcb + s * NP + g * NS, bc);
                const bool rs = has && (rm >> s & 1);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const float a = __builtin_amdgcn_exp2f(pw.x * A2[i]);
                    h[i] = BWD ? (rs ? 0.f : a * fmaf(pw.y, bc[i], h[i])) : fmaf(a, rs ? 0.f : h[i], pw.y * bc[i]);
                }
            }
        };
        if (rm) steps(std::true_type{}); else steps(std::false_type{});
        wave_sync();
    }
    sum += __shfl_xor(sum, 16, WAVE);
    sum += __shfl_xor(sum, 32, WAVE);
    if (!dv) return;
    const long long o = ((long long)seg * p.B + b) * p.D + d;
    put_states<NS>(carry + o * p.N + g * NS, h, g * NS, p.N, vec4(carry, p.N));
    if (g == 0) sums[o] = cut ? __builtin_inff() : sum;
}

// carry[seg]: what a segment adds -> what it starts from
template <bool BWD>
__global__ __launch_bounds__(256) void k_ssm_join(SsmArgs p, int S, float* __restrict__ carry, const float* __restrict__ sums) {
    const long long n = p.B * p.D * p.N, i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long r = i / p.N;
    // P as the square of R: it may leave the range where P h does not. R is finite: an empty state stays empty.
    const float A2 = rate(p.A[r % p.D * p.N + i % p.N], 0.5f * LOG2E);
    const float* h0 = BWD ? p.dhT : p.h0;
    float h = h0 ? h0[i] : 0.f;
    constexpr int AHEAD = 16;                               // loads in flight: a carry is overwritten only after its batch is read
    for (int k0 = 0; k0 < S; k0 += AHEAD) {
        float e[AHEAD], sum[AHEAD], R[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int s = BWD ? S - 1 - k0 - k : k0 + k;
            const bool in = k0 + k < S - 1;
            e[k] = in ? carry[s * n + i] : 0.f;
            sum[k] = in ? sums[s * p.B * p.D + r] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) R[k] = fminf(__builtin_amdgcn_exp2f(sum[k] * A2), 3.402823466e38f);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (k0 + k >= S) break;
            carry[(BWD ? S - 1 - k0 - k : k0 + k) * n + i] = h;
            h = sum[k] == __builtin_inff() ? e[k] : fmaf(R[k], R[k] * h, e[k]);
        }
    }
}

// 120 x 64 x 1024 bf16, 16 states: 41 to 45 us, its vector units busy 89 % of the time, 1.6 TB/s; 32 states 68 us, 4
// states 28 us.
template <typename T, int NS>
__global__ __launch_bounds__(256) void k_ssm_fwd(SsmArgs p, int seg_len, const float* __restrict__ carry) {
    constexpr int NP = 4 * NS;
    using R = Rows<T>;
    __shared__ __align__(16) float2 pw_s[4][KC][16];
    __shared__ __align__(16) float bc_s[2][KC * 2 * NP];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
    static_assert(sizeof(pw_s) > SORT_ROWS * sizeof(int), "block_row");
    const int b = block_row(p, (int*)pw_s);
    const int d = (blockIdx.x * 4 + w) * 16 + j;
    const bool dv = d < p.D;
    const int end = row_end(p, b), ta = blockIdx.z * seg_len, tb = min(ta + seg_len, (int)p.T);
    const long long so = ((long long)b * p.D + d) * p.N + g * NS;          // this lane's states in a [B, D, N] tensor
    const long long BDN = p.B * p.D * p.N;
    float A2[NS], h[NS];
    const float* hp = carry ? carry + blockIdx.z * BDN : p.h0;
    get_states<NS>(hp + so, h, g * NS, p.N, dv && hp, vec4(hp, p.N));
#pragma unroll
    for (int i = 0; i < NS; ++i) A2[i] = dv && g * NS + i < p.N ? rate(p.A[(long long)d * p.N + g * NS + i], LOG2E) : 0.f;
    const float Dd = dv && p.Dp ? p.Dp[d] : 0.f, bias = dv && p.bias ? p.bias[d] : 0.f;
    const unsigned ou = R::offset(p.u_t, g, d), od = R::offset(p.dt_t, g, d), oz = R::offset(p.z_t, g, d), oy = R::offset(p.y_t, g, d);
    const bool has_z = p.z != nullptr, soft = p.softplus != 0, ck4 = vec4(p.ckpt, p.N);
    unsigned ru[4], rd[4], rz[4], rr;
    R xu(p.u, p.u_t, p.u_b, b, ta), xd(p.dt, p.dt_t, p.dt_b, b, ta), xz(p.z, p.z_t, p.z_b, b, ta), xy(p.y, p.y_t, p.y_b, b, ta);
    StageBC<T, NS, 3> st(p, b, ta);
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned bad = dv && t0 + 4 * i + g < end ? 0u : OOB;
            ru[i] = R::load(xu.rsrc(), ou | bad, i * xu.four);
            rd[i] = R::load(xd.rsrc(), od | bad, i * xd.four);
            if (has_z) rz[i] = R::load(xz.rsrc(), oz | bad, i * xz.four);
        }
        st.fetch(end - t0);
        rr = fetch_resets(p, b, t0, end, lane);
        xu.next(); xd.next(); xz.next(); st.B.next(); st.C.next();
    };
    const int live = min(tb, end);                          // padding is not walked: its rows are zeroed below
    if (live > ta) fetch(ta);
    for (int t0 = ta, c = 0; t0 < live; t0 += KC, ++c) {
        float u[4], zz[4], sp[4];                           // flags outside: see k_ssm_carry
#pragma unroll
        for (int i = 0; i < 4; ++i) { u[i] = R::value(ru[i]); zz[i] = 1.f; sp[i] = R::value(rd[i]) + bias; }
        if (has_z) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { const float z = R::value(rz[i]); zz[i] = z * sigmoidf(z); }
        }
        if (soft) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sp[i] = softplus(sp[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sp[i] = dv && t0 + 4 * i + g < end ? sp[i] : 0.f;
            pw_s[w][4 * i + g][j] = make_float2(sp[i], sp[i] * u[i]);
        }
        float* bcb = bc_s[c & 1];
        st.put(bcb);
        const unsigned rm = reset_mask(rr);
        if (t0 + KC < live) fetch(t0 + KC);
        block_sync_lds();                 // B and C of this chunk are there; the image of the chunk before last is free again
        float y[4] = {0.f, 0.f, 0.f, 0.f};
        auto steps = [&](auto has) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (q == 2 && t0 + 8 >= live) break;        // the row ends in the chunk's first half
                if (4 * q % SAVE == 0 && p.ckpt && dv && t0 + 4 * q < p.T)
                    put_states<NS>(p.ckpt + (t0 / SAVE + 4 * q / SAVE) * BDN + so, h, g * NS, p.N, ck4);
                float part[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int s = 4 * q + r;
                    const float2 pw = pw_s[w][s][j];
                    const bool rs = has && (rm >> s & 1);
                    float Bv[NS], Cv[NS];
                    lds_row<NS>(bcb + s * 2 * NP + g * NS, Bv);
                    lds_row<NS>(bcb + s * 2 * NP + NP + g * NS, Cv);
                    float acc = 0.f;
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        h[i] = fmaf(__builtin_amdgcn_exp2f(pw.x * A2[i]), rs ? 0.f : h[i], pw.y * Bv[i]);
                        acc = fmaf(Cv[i], h[i], acc);
                    }
                    part[r] = acc;
                }
                y[q] = sum_groups(part[0], part[1], part[2], part[3]);
            }
        };
        if (rm) steps(std::true_type{}); else steps(std::false_type{});
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = t0 + 4 * i + g;
            // dead steps: u = 0 and C = 0, so the sum is 0 but for what a diverged state makes of it
            R::store(xy.rsrc(), dv && t < p.T ? oy : OOB, i * xy.four, t < end ? fmaf(Dd, u[i], y[i]) * zz[i] : 0.f);
        }
        xy.next();
        wave_sync();                                        // the next chunk overwrites this wave's LDS image
    }
    for (int t0 = ta + (max(live - ta, 0) + KC - 1) / KC * KC; t0 < tb; t0 += KC) {
#pragma unroll
        for (int i = 0; i < 4; ++i) R::store(xy.rsrc(), dv && t0 + 4 * i + g < tb ? oy : OOB, i * xy.four, 0.f);
        xy.next();
    }
    if (p.hT && dv && blockIdx.z == gridDim.z - 1) put_states<NS>(p.hT + so, h, g * NS, p.N, vec4(p.hT, p.N));
}

// Backward. g_t = C ds + a_{t+1} g_{t+1} runs against the time; the states it needs are recomputed from the saved ones, KH = 8
// steps at a time (4 from 17 states on), and kept in registers next to the decays. The sums over channels of dB and dC leave as partials
// of 64 channels (a block), the sums over rows of dA, dD and the bias as partials of a row: a second launch adds them in a
// fixed order. 120 x 64 x 1024 bf16, 16 states, resets and lengths of 30 .. 120: 102 to 107 us, vector units busy 74 % of the
// time with two waves a SIMD. Three fit 168 registers only with spills or with LDS reads one step at a time: 3 to 8 % slower.
//
// KH steps of a chunk, s0 .. s0 + KH - 1, from the state before them: forward with the states and decays kept, then back.
// mid() is called half way back, when half of those registers are free again: the next chunk's loads start there. emit(s, gB, wA)
// gets the sums over the states for the lane's own step of each four that are done (s = their first).
//
// A reset chooses zeros for what passes it, the state forward and its gradient back: a factor of zero would make NaN of an
// episode that diverged on the other side. By a select for each state, or from 17 states on by one branch a step (120 x 64 x
// 1024 with resets, both passes, selects and branch: 4 states 81.0 and 84.1 us, 32 states 319 and 307, 64 states 772 and 759).
template <int NS, int KH, bool RS, typename F, typename E>
__device__ __forceinline__ void bwd_piece(const float4 (&pw_w)[KC][16], const float* bcb, float* red_w, unsigned rm, int s0, int g, int j,
                                          const float (&An)[NS], float (&hs)[KH + 1][NS], float (&G)[NS], float (&dAc)[NS],
                                          float (&y_w)[KC][16], F mid, E emit) {
    constexpr int NP = 4 * NS;
    constexpr bool BRANCH = RS && NS > 4;
    // What a step reads from LDS. Forward a step ahead; back as it is needed: two steps ahead took registers that 32 states do
    // not have (120 x 64 x 1024 both passes 340 us, so 297) and gained nothing with fewer.
    struct In { float4 pw; float B[NS], C[NS]; };
    auto load = [&](int s, int again) {
        In x;
        x.pw = pw_w[s][j + again];
        lds_row<NS>(bcb + s * 2 * NP + g * NS + again, x.B);
        lds_row<NS>(bcb + s * 2 * NP + NP + g * NS + again, x.C);
        return x;
    };
    float a[KH][NS], part[4];
    In x = load(s0, 0);
#pragma unroll
    for (int k = 0; k < KH; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        const int s = s0 + k;
        In nx;
        if (k + 1 < KH) nx = load(s + 1, 0);
        const bool rs = RS && (rm >> s & 1);        // hs[k] itself stays: dC of the step before needs it
        float acc = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const float e = __builtin_amdgcn_exp2f(x.pw.x * An[i]), in = x.pw.y * x.B[i], n = fmaf(e, hs[k][i], in);
            a[k][i] = e;
            hs[k + 1][i] = rs ? in : n;
            acc = fmaf(x.C[i], hs[k + 1][i], acc);
        }
        part[k & 3] = acc;
        if ((k & 3) == 3) y_w[s - 3 + g][j] = sum_groups(part[0], part[1], part[2], part[3]);
        if (k + 1 < KH) x = nx;
    }
    int again = 0;                                  // hides that B, C and the step's scalars are read a second time:
    asm volatile("" : "+v"(again));                 // kept from the first, they would fill the registers
    float pb[4], pa[4];
#pragma unroll
    for (int k = KH - 2; k >= 0; k -= 2) {          // two steps at a time: k + 1, then k
        float vB[2][NS], vC[2][NS];
        __builtin_amdgcn_sched_barrier(0);
        if (k == (KH == 4 ? 0 : KH / 2 - 2)) mid();
        const In xs[2] = {load(s0 + k, again), load(s0 + k + 1, again)};
#pragma unroll
        for (int o = 1; o >= 0; --o) {
            const int c = (k + o) & 3;
            const float4 pw = xs[o].pw;
            pb[c] = 0.f; pa[c] = 0.f;
            const bool rs = RS && (rm >> (s0 + k + o) & 1);
            const auto back = [&](int i, float gh, bool cut) {  // through the decay, to the step before
                const float q = gh * a[k + o][i], y = cut ? 0.f : q * hs[k + o][i];
                G[i] = cut ? 0.f : q;
                pa[c] = fmaf(y, An[i], pa[c]);
                dAc[i] = fmaf(y, pw.x, dAc[i]);
                pin(dAc[i]);
            };
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const float gh = fmaf(pw.z, xs[o].C[i], G[i]);
                vB[o][i] = gh * pw.y;
                vC[o][i] = pw.z * hs[k + o + 1][i];
                pb[c] = fmaf(gh, xs[o].B[i], pb[c]);
                if constexpr (BRANCH) G[i] = gh;
                else back(i, gh, rs);
            }
            if constexpr (BRANCH) {
                if (rs) {
#pragma unroll
                    for (int i = 0; i < NS; ++i) G[i] = 0.f;
                } else {
#pragma unroll
                    for (int i = 0; i < NS; ++i) back(i, G[i], false);
                }
            }
            pin(pb[c]); pin(pa[c]);
        }
        float* red = red_w + (s0 + k + (j >> 2 & 1)) * 2 * NP + (j >> 3) * NP + g * NS;
        if constexpr (NS % 4 == 0) {
#pragma unroll
            for (int i = 0; i < NS; i += 4) red[i + (j & 3)] = sum_rows4(vB[0] + i, vC[0] + i, vB[1] + i, vC[1] + i, j);
        } else if constexpr (NS == 2) {
            red[j & 1] = sum_rows2(vB[0], vC[0], vB[1], vC[1], j);
        } else {
            red[0] = sum_rows1(vB[0], vC[0], vB[1], vC[1]);
        }
        if ((k & 3) == 0) {
            emit(s0 + k, sum_groups(pb[0], pb[1], pb[2], pb[3]), sum_groups(pa[0], pa[1], pa[2], pa[3]));
        }
    }
}

// Four waves a SIMD for 5 to 8 states: 120 x 64 x 1024 both passes 130 -> 117 us, though up to 4 registers spill. Up to 4 states
// they fit without being asked for.
// HAS: the call has reset flags. (A branch on each chunk's flags instead holds the registers of both paths: spills.)
template <typename T, int NS, bool HAS>
__global__ __launch_bounds__(256, NS > 8 ? 1 : NS == 2 ? 4 : 2) void k_ssm_bwd(SsmArgs p, int seg_len, const float* __restrict__ carry,
                                                    float* __restrict__ part_bc, float* __restrict__ part_a) {
    constexpr int NP = 4 * NS;
    constexpr int KH = NS > 4 ? 4 : 8;                      // steps whose states are held at a time
    using R = Rows<T>;
    __shared__ __align__(16) float4 pw_s[4][KC][16];        // s log2(e), s u, ds, u
    __shared__ __align__(16) float2 ex_s[4][KC][16];        // dy silu'(z), ds/d(pre)
    __shared__ float y_s[4][KC][16];                        // sum_n C h
    __shared__ __align__(16) float bc_s[2][KC * 2 * NP];
    __shared__ __align__(16) float red_s[2][4][KC * 2 * NP];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
    static_assert(sizeof(pw_s) > SORT_ROWS * sizeof(int), "block_row");
    const int b = block_row(p, (int*)pw_s);
    const int d = (blockIdx.x * 4 + w) * 16 + j;
    const bool dv = d < p.D;
    const int end = row_end(p, b), ta = blockIdx.z * seg_len, tb = min(ta + seg_len, (int)p.T);
    const long long so = ((long long)b * p.D + d) * p.N + g * NS, BDN = p.B * p.D * p.N;
    float An[NS], G[NS], dA[NS];                            // G = a_{t+1} g_{t+1}: dL/dh_t from the steps behind
    const float* Gp = carry ? carry + blockIdx.z * BDN : p.dhT;
    get_states<NS>(Gp + so, G, g * NS, p.N, dv && Gp, vec4(Gp, p.N));
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        An[i] = dv && g * NS + i < p.N ? rate(p.A[(long long)d * p.N + g * NS + i], 1.f) : 0.f;
        dA[i] = 0.f;
    }
    const float Dd = dv && p.Dp ? p.Dp[d] : 0.f, bias = dv && p.bias ? p.bias[d] : 0.f;
    float dD = 0.f, dbias = 0.f;
    const bool has_z = p.z != nullptr, soft = p.softplus != 0;
    const int n_t = (int)p.T;
    const unsigned ou = R::offset(p.u_t, g, d), od = R::offset(p.dt_t, g, d), oz = R::offset(p.z_t, g, d), oy = R::offset(p.dy_t, g, d);
    const unsigned odu = R::offset(p.du_t, g, d), odd = R::offset(p.ddt_t, g, d), odz = R::offset(p.dz_t, g, d);
    unsigned ru[4], rd[4], rz[4], ry[4], rr;
    float hc0[NS], hc1[NS];                                 // the saved states before steps 0 and 8 of the chunk
    const int live = min(tb, end), t_last = ta + max(live - ta - 1, 0) / KC * KC;       // padding is not walked, see below
    R xu(p.u, p.u_t, p.u_b, b, t_last), xd(p.dt, p.dt_t, p.dt_b, b, t_last), xz(p.z, p.z_t, p.z_b, b, t_last), xy(p.dy, p.dy_t, p.dy_b, b, t_last);
    R wu(p.du, p.du_t, p.du_b, b, t_last), wd(p.ddt, p.ddt_t, p.ddt_b, b, t_last), wz(p.dz, p.dz_t, p.dz_b, b, t_last);
    StageBC<T, NS, 3> st(p, b, t_last);
    const float* ck = p.ckpt + t_last / SAVE * BDN;
    const bool ck4 = vec4(p.ckpt, p.N);
    auto fetch = [&](int t0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned bad = dv && t0 + 4 * i + g < end ? 0u : OOB;
            ru[i] = R::load(xu.rsrc(), ou | bad, i * xu.four);
            rd[i] = R::load(xd.rsrc(), od | bad, i * xd.four);
            ry[i] = R::load(xy.rsrc(), oy | bad, i * xy.four);
            if (has_z) rz[i] = R::load(xz.rsrc(), oz | bad, i * xz.four);
        }
        st.fetch(end - t0);
        if (HAS) rr = fetch_resets(p, b, t0, end, lane);
        get_states<NS>(ck + so, hc0, g * NS, p.N, dv, ck4);
        get_states<NS>(ck + BDN + so, hc1, g * NS, p.N, dv && t0 + SAVE < live, ck4);
        xu.back(); xd.back(); xz.back(); xy.back(); st.B.back(); st.C.back(); ck -= 2 * BDN;
    };
    // sums of the block's four waves over a finished chunk's dB, dC
    const long long prow = p.B * gridDim.x * 2 * NP;        // partials of a step
    auto put_partials = [&](int t0, const float (*red)[KC * 2 * NP]) {
        constexpr int RS = 256 / (2 * NP) < KC ? 256 / (2 * NP) : KC;       // steps that the block covers at a time
        const int x = threadIdx.x % (2 * NP), y = threadIdx.x / (2 * NP);
        float* q = part_bc + (t0 + y) * prow + ((long long)b * gridDim.x + blockIdx.x) * (2 * NP) + x;
#pragma unroll
        for (int k = 0; k < (KC + RS - 1) / RS; ++k) {
            const int s = y + k * RS, e = s * 2 * NP + x;
            if (y < RS && s < KC && t0 + s < live) q[k * RS * prow] = (red[0][e] + red[1][e]) + (red[2][e] + red[3][e]);
        }
    };
    for (int t0 = live > ta ? t_last + KC : ta; t0 < tb; t0 += KC) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned bad = dv && t0 + 4 * i + g < tb ? 0u : OOB;
            const R qu(p.du, p.du_t, p.du_b, b, t0), qd(p.ddt, p.ddt_t, p.ddt_b, b, t0), qz(p.dz, p.dz_t, p.dz_b, b, t0);
            R::store(qu.rsrc(), odu | bad, i * qu.four, 0.f);
            R::store(qd.rsrc(), odd | bad, i * qd.four, 0.f);
            if (has_z) R::store(qz.rsrc(), odz | bad, i * qz.four, 0.f);
        }
    }
    if (live > ta) fetch(t_last);
    int c = 0;
    for (int t0 = live > ta ? t_last : ta - 1; t0 >= ta; t0 -= KC, ++c) {
        {
            float sp[4], ds[4], sg[4], dz[4];               // flags outside: see k_ssm_carry
#pragma unroll
            for (int i = 0; i < 4; ++i) { sp[i] = R::value(rd[i]) + bias; ds[i] = R::value(ry[i]); sg[i] = 1.f; dz[i] = 0.f; }
            if (has_z) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float z = R::value(rz[i]), sz = sigmoidf(z);
                    dz[i] = ds[i] * sz * fmaf(z, 1.f - sz, 1.f);
                    ds[i] *= z * sz;
                }
            }
            if (soft) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sp[i] = softplus(sp[i], &sg[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = R::value(ru[i]);
                sp[i] = dv && t0 + 4 * i + g < end ? sp[i] : 0.f;
                pw_s[w][4 * i + g][j] = make_float4(sp[i] * LOG2E, sp[i] * u, ds[i], u);
                ex_s[w][4 * i + g][j] = make_float2(dz[i], sg[i]);
            }
        }
        float* bcb = bc_s[c & 1];
        st.put(bcb);
        const unsigned rm = HAS ? reset_mask(rr) : 0;
        float hs[KH + 1][NS], h0[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) h0[i] = HAS && (rm & 1) ? 0.f : hc0[i];
        auto next = [&] {
            asm volatile("" ::: "memory");                  // not earlier
            if (t0 > ta) fetch(t0 - KC);
        };
        block_sync_lds();
        if (c) put_partials(t0 + KC, red_s[(c - 1) & 1]);
        float dAc[NS], dDc = 0.f, dbc = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) dAc[i] = 0.f;
        float* red = red_s[c & 1][w];
        auto emit = [&](int s, float gB, float wA) {
            const float4 pw = pw_s[w][s + g][j];
            const float2 ex = ex_s[w][s + g][j];
            const float yq = y_s[w][s + g][j];
            const int t = t0 + s + g;
            const float dpre = t < end ? fmaf(pw.w, gB, wA) * ex.y : 0.f;
            dDc = fmaf(pw.z, pw.w, dDc);
            dbc += dpre;
            const unsigned bad = dv && t < n_t ? 0u : OOB;
            R::store(wu.rsrc(), odu | bad, (unsigned)(s / 4) * wu.four, t < end ? fmaf(Dd, pw.z, pw.x * LN2 * gB) : 0.f);
            R::store(wd.rsrc(), odd | bad, (unsigned)(s / 4) * wd.four, dpre);
            if (has_z) R::store(wz.rsrc(), odz | bad, (unsigned)(s / 4) * wz.four, t < end ? ex.x * fmaf(Dd, pw.w, yq) : 0.f);
        };
        auto from = [&](const float (&h)[NS]) {
#pragma unroll
            for (int i = 0; i < NS; ++i) hs[0][i] = h[i];
        };
        auto piece = [&](int s0, auto mid) { bwd_piece<NS, KH, HAS>(pw_s[w], bcb, red, rm, s0, g, j, An, hs, G, dAc, y_s[w], mid, emit); };
        auto nothing = [] {};
        const bool half = t0 + SAVE >= live;                // the row ends in the chunk's first half: the other is zeros
        if (half) {
#pragma unroll
            for (int i = 2; i < 4; ++i) {
                const unsigned bad = dv && t0 + 4 * i + g < n_t ? 0u : OOB;
                R::store(wu.rsrc(), odu | bad, i * wu.four, 0.f);
                R::store(wd.rsrc(), odd | bad, i * wd.four, 0.f);
                if (has_z) R::store(wz.rsrc(), odz | bad, i * wz.four, 0.f);
            }
        }
        if constexpr (KH == SAVE) {
            if (!half) {
                from(hc1);
                piece(SAVE, nothing);
            }
            from(h0);
            piece(0, next);
        } else {                                            // two pieces from each saved state: its steps are run up to the second
            auto run = [&](int s0) {
#pragma unroll
                for (int s = s0; s < s0 + KH; ++s) {
                    const float4 pw = pw_s[w][s][j];
                    float Bv[NS];
                    lds_row<NS>(bcb + s * 2 * NP + g * NS, Bv);
                    const bool rs = HAS && (rm >> s & 1);
#pragma unroll
                    for (int i = 0; i < NS; ++i) hs[0][i] = fmaf(__builtin_amdgcn_exp2f(pw.x * An[i]), rs ? 0.f : hs[0][i], pw.y * Bv[i]);
                }
            };
            if (!half) {
                from(hc1); run(SAVE); piece(SAVE + KH, nothing);
                from(hc1); piece(SAVE, nothing);
            }
            from(h0); run(0); piece(KH, nothing);
            from(h0); piece(0, next);
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) dA[i] += dAc[i];
        dD += dDc; dbias += dbc;
        wu.back(); wd.back(); wz.back();
        wave_sync();
    }
    if (c) {
        block_sync_lds();
        put_partials(ta, red_s[(c - 1) & 1]);
    }
    dD += __shfl_xor(dD, 16, WAVE); dD += __shfl_xor(dD, 32, WAVE);
    dbias += __shfl_xor(dbias, 16, WAVE); dbias += __shfl_xor(dbias, 32, WAVE);
    if (!dv) return;
#pragma unroll
    for (int i = 0; i < NS; ++i) dA[i] *= LN2;              // the step sizes were carried times log2(e)
    // a row of partials: dA [D, N], dD [D], dbias [D]
    const long long cols = p.D * (p.N + 2);
    float* q = part_a + ((long long)blockIdx.z * p.B + b) * cols;
    put_states<NS>(q + (long long)d * p.N + g * NS, dA, g * NS, p.N, vec4(q, p.N));
    if (p.dh0 && blockIdx.z == 0) put_states<NS>(p.dh0 + so, G, g * NS, p.N, vec4(p.dh0, p.N));
    if (g == 0) { q[p.D * p.N + d] = dD; q[p.D * (p.N + 1) + d] = dbias; }
}

// Second launch of the backward: blocks [0, n_bc) add the channel blocks' partials of dB and dC, the others the rows' partials
// of dA, dD and the bias, 32 columns by 8 groups of rows each, all in a fixed order. 120 x 64 x 1024, 16 states: 4.9 us.
template <typename T>
__global__ __launch_bounds__(256) void k_ssm_finish(SsmArgs p, const float* __restrict__ part_bc, int nblk, int NP, unsigned n_bc,
                                                    const float* __restrict__ part_a, int rows) {
    if (blockIdx.x < n_bc) {
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x;; i += (long long)n_bc * 256) {
            const long long row = i / (2 * p.N);
            if (row >= p.T * p.B) return;
            const int c = (int)(i - row * 2 * p.N), isC = c >= p.N, n = isC ? c - (int)p.N : c;
            const float* q = part_bc + row * nblk * 2 * NP + isC * NP + n;
            const long long t = row / p.B, b = row - t * p.B;
            float v = 0.f;
            if (t < row_end(p, (int)b)) {                   // padding has no partials
#pragma unroll 4
                for (int k = 0; k < nblk; ++k) v += q[(long long)k * 2 * NP];
            }
            if (isC) st((T*)p.dCm + t * p.dC_t + b * p.dC_b + n, v);
            else st((T*)p.dBm + t * p.dB_t + b * p.dB_b + n, v);
        }
    }
    __shared__ float acc[8][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const long long DN = p.D * p.N, cols = DN + 2 * p.D, i = (long long)(blockIdx.x - n_bc) * 32 + x;
    float v = 0.f;
    if (i < cols) {
#pragma unroll 4
        for (int r = y; r < rows; r += 8) v += part_a[r * cols + i];
    }
    acc[y][x] = v;
    __syncthreads();
    if (y || i >= cols) return;
    v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += acc[k][x];
    if (i < DN) p.dA[i] = v;
    else if (i < DN + p.D) { if (p.dD) p.dD[i - DN] = v; }
    else if (p.dbias) p.dbias[i - DN - p.D] = v;
}

// One step: h [B, D, N] is read and written once and is nearly all of the bytes. Consecutive lanes own V consecutive states (four,
// 16 bytes, where N is a power of two from 4 on and the addresses allow it, otherwise one), L = 2^k >= N / V lanes a channel,
// and add up the read-out with cross-lane adds; what depends on the channel only is computed by each of its lanes. A thread
// takes R channels with the loads of all of them under way. 4096 x 1024 bf16, 16 states: 119 us (4.8 TB/s), 64 x 1024 4.2 us.
// One state a lane means a channel's step size in 32 or 64 lanes and idle ones: 24 states 566 us, 40 states 1 106 (1.2 TB/s).
template <typename T, int V, int L, int R>
__global__ __launch_bounds__(256) void k_ssm_step(SsmArgs p) {
    const int lane = threadIdx.x % L, n0 = lane * V, N = (int)p.N, D = (int)p.D;
    const long long total = p.B * p.D, step = (long long)gridDim.x * gridDim.y * (256 / L);
    const long long i0 = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * (256 / L) + threadIdx.x / L;
    float h[R][V], A[R][V], Bv[R][V], Cv[R][V], u[R], dt[R], z[R], Dd[R];
    bool rs[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const long long i = min(i0 + k * step, total - 1), b = (unsigned long long)i / (unsigned)D;
        const int d = (int)(i - b * D);
        u[k] = ld((const T*)p.u + b * p.u_b + d);
        dt[k] = ld((const T*)p.dt + b * p.dt_b + d) + (p.bias ? p.bias[d] : 0.f);
        z[k] = p.z ? ld((const T*)p.z + b * p.z_b + d) : 0.f;
        Dd[k] = p.Dp ? p.Dp[d] : 0.f;
        rs[k] = p.reset && p.reset[b] != 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const bool in = V > 1 || n0 < N;
            h[k][v] = A[k][v] = Bv[k][v] = Cv[k][v] = 0.f;
            if (V == 1 && in) { h[k][v] = p.hT[i * N + n0]; A[k][v] = p.A[(long long)d * N + n0]; }
            if (in) { Bv[k][v] = ld((const T*)p.Bm + b * p.B_b + n0 + v); Cv[k][v] = ld((const T*)p.Cm + b * p.C_b + n0 + v); }
        }
        if constexpr (V == 4) {
            const float4 x = *reinterpret_cast<const float4*>(p.hT + i * N + n0), a = *reinterpret_cast<const float4*>(p.A + (long long)d * N + n0);
            h[k][0] = x.x; h[k][1] = x.y; h[k][2] = x.z; h[k][3] = x.w;
            A[k][0] = a.x; A[k][1] = a.y; A[k][2] = a.z; A[k][3] = a.w;
        }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const long long i = i0 + k * step;
        float s = dt[k], y = 0.f;
        if (p.softplus) s = softplus(s);
        const float s2 = s * LOG2E;                         // (A log2(e) may leave the range, and a step of size 0 holds the state)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float e = __builtin_amdgcn_exp2f(s2 * A[k][v]);
            h[k][v] = fmaf(e, rs[k] ? 0.f : h[k][v], s * u[k] * Bv[k][v]);
            y = fmaf(Cv[k][v], h[k][v], y);
        }
        if constexpr (L > 1) y = add_dpp<0xB1>(y);
        if constexpr (L > 2) y = add_dpp<0x4E>(y);
        if constexpr (L > 4) y = add_dpp<0x141>(y);
        if constexpr (L > 8) y = add_dpp<0x140>(y);
        if constexpr (L > 16) y = add_swap16(y, y);
        if constexpr (L > 32) y = add_swap32(y, y);
        if (i >= total) continue;
        if constexpr (V == 4) *reinterpret_cast<float4*>(p.hT + i * N + n0) = make_float4(h[k][0], h[k][1], h[k][2], h[k][3]);
        else if (n0 < N) p.hT[i * N + n0] = h[k][0];
        if (lane == 0) {
            const long long b = (unsigned long long)i / (unsigned)D;
            y = fmaf(Dd[k], u[k], y);
            if (p.z) y *= z[k] * sigmoidf(z[k]);
            st((T*)p.y + b * p.y_b + (i - b * D), y);
        }
    }
}

// States a lane, of the four lanes a channel has. Up to 4 states one each: 120 x 64 x 1024 bf16 forward 29 us and both passes 98,
// with two each (half of them empty) 33 and 124.
static int ns_of(long long N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : N <= 48 ? 12 : 16; }

// Segments: one where the rows alone give the chip waves enough, else as many as bring it to 4 096, of at least 64 steps. A cut
// costs the carry pass (the recurrence without its read-out), which long sequences repay sooner. Both passes of T x B x D,
// 16 states, uncut and cut: 1000 x 25 x 512 (800 waves) 566 and 387 us, 300 x 18 x 1024 (1 152) 215 and 193, 1000 x 25 x 1024
// (1 600) 701 and 765, 120 x 11 x 1024 (704) 78 and 84, 200 x 10 x 1024 (640) 118 and 104.
struct Segs { int n, len; };
static Segs segments(long long T, long long B, long long D) {
    const long long waves = (D + 15) / 16 * B, chunks = (T + KC - 1) / KC;
    long long n = 1;
    if (waves < (chunks < 12 ? 512 : chunks < 16 ? 768 : 1400)) {
        n = (4096 + waves - 1) / waves;
        if (n > chunks / 4) n = chunks / 4;
        if (n < 1) n = 1;
    }
    const long long len = (chunks + n - 1) / n * KC;
    return {(int)((T + len - 1) / len), (int)len};
}

// floats of scratch that a forward (train = 0) or a forward and its backward (1) need
DRL_API int drl_ssm_ws(long long T, long long B, long long D, long long N, int train, long long* n) {
    if (T <= 0 || T > (1ll << 30) || B <= 0 || D <= 0 || D > (1ll << 22) || N <= 0 || N > 64 || B > 65535 || T * B > (1ll << 31)) return -1;
    const long long nblk = (D + 63) / 64, S = segments(T, B, D).n;
    *n = S > 1 ? S * B * D * (N + 1) : 0;
    if (train) *n += T * B * nblk * 8 * ns_of(N) + S * B * D * (N + 2);
    return 0;
}

// Offsets inside a chunk are 32-bit: 16 steps of any tensor lie under 2^31 bytes. The stride of a single step says nothing and
// may be anything; it becomes 0.
static bool steps_ok(SsmArgs& p) {
    for (long long* q : {&p.u_t, &p.dt_t, &p.z_t, &p.B_t, &p.C_t, &p.y_t, &p.dy_t, &p.du_t, &p.ddt_t, &p.dz_t}) {
        if (p.T == 1) *q = 0;
        else if (*q < 0 || *q >= (1ll << 25)) return false;
    }
    return true;
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
    const dim3 grid((unsigned)nblk, (unsigned)p.B, (unsigned)sg.n);
    if (p.reset) k_ssm_bwd<T, NS, true><<<grid, 256, 0, s>>>(p, sg.len, carry, part_bc, part_a);
    else k_ssm_bwd<T, NS, false><<<grid, 256, 0, s>>>(p, sg.len, carry, part_bc, part_a);
    const long long n = (p.T * p.B * 2 * p.N + 255) / 256;
    const unsigned n_bc = (unsigned)(n < (1 << 22) ? n : 1 << 22), n_a = (unsigned)((p.D * (p.N + 2) + 31) / 32);
    k_ssm_finish<T><<<n_bc + n_a, 256, 0, s>>>(p, part_bc, nblk, NP, n_bc, part_a, (int)rows);
}

#define SSM_NS(NAME, T)                       \
    switch (ns_of(p.N)) {                     \
        case 1: NAME<T, 1>(p, s); break;      \
        case 2: NAME<T, 2>(p, s); break;      \
        case 4: NAME<T, 4>(p, s); break;      \
        case 8: NAME<T, 8>(p, s); break;      \
        case 12: NAME<T, 12>(p, s); break;    \
        default: NAME<T, 16>(p, s); break;    \
    }

// [T, B, c] tensors of e bytes an element, and the fp32 ones
static View seq_view(const SsmArgs& p, const void* q, long long st, long long sb, long long c, long long e) { return {q, c * e, p.T, st * e, p.B, sb * e}; }
static View state_view(const SsmArgs& p, const void* q) { return {q, p.B * p.D * p.N * 4}; }
static View ckpt_view(const SsmArgs& p) { return {p.ckpt, (p.T + SAVE - 1) / SAVE * p.B * p.D * p.N * 4}; }

DRL_API int drl_ssm_fwd(const SsmArgs* a, int bf16, hipStream_t s) {
    SsmArgs p = *a;
    long long need;
    if (drl_ssm_ws(p.T, p.B, p.D, p.N, 0, &need) || !steps_ok(p)) return -1;
    if (p.ws_n < need) return -2;
    const long long e = bf16 ? 2 : 4, cols = p.D * 4;
    if (!apart({seq_view(p, p.y, p.y_t, p.y_b, p.D, e), state_view(p, p.hT), ckpt_view(p), {p.ws, need * 4}},
               {seq_view(p, p.u, p.u_t, p.u_b, p.D, e), seq_view(p, p.dt, p.dt_t, p.dt_b, p.D, e), seq_view(p, p.z, p.z_t, p.z_b, p.D, e),
                seq_view(p, p.Bm, p.B_t, p.B_b, p.N, e), seq_view(p, p.Cm, p.C_t, p.C_b, p.N, e), {p.A, cols * p.N}, {p.Dp, cols}, {p.bias, cols},
                state_view(p, p.h0), {p.reset, p.T * p.B}, {p.lengths, p.B * 4}})) return -3;
    if (bf16) { SSM_NS(launch_fwd, bf16_t) } else { SSM_NS(launch_fwd, float) }
    return (int)hipGetLastError();
}

DRL_API int drl_ssm_bwd(const SsmArgs* a, int bf16, hipStream_t s) {
    SsmArgs p = *a;
    long long need;
    if (drl_ssm_ws(p.T, p.B, p.D, p.N, 1, &need) || !p.ckpt || !steps_ok(p)) return -1;
    if (p.ws_n < need) return -2;
    const long long e = bf16 ? 2 : 4, cols = p.D * 4;
    if (!apart({seq_view(p, p.du, p.du_t, p.du_b, p.D, e), seq_view(p, p.ddt, p.ddt_t, p.ddt_b, p.D, e), seq_view(p, p.dz, p.dz_t, p.dz_b, p.D, e),
                seq_view(p, p.dBm, p.dB_t, p.dB_b, p.N, e), seq_view(p, p.dCm, p.dC_t, p.dC_b, p.N, e), {p.dA, cols * p.N}, {p.dD, cols}, {p.dbias, cols},
                state_view(p, p.dh0), {p.ws, need * 4}},
               {seq_view(p, p.u, p.u_t, p.u_b, p.D, e), seq_view(p, p.dt, p.dt_t, p.dt_b, p.D, e), seq_view(p, p.z, p.z_t, p.z_b, p.D, e),
                seq_view(p, p.Bm, p.B_t, p.B_b, p.N, e), seq_view(p, p.Cm, p.C_t, p.C_b, p.N, e), seq_view(p, p.dy, p.dy_t, p.dy_b, p.D, e),
                {p.A, cols * p.N}, {p.Dp, cols}, {p.bias, cols}, state_view(p, p.dhT), ckpt_view(p), {p.reset, p.T * p.B}, {p.lengths, p.B * 4}})) return -3;
    if (bf16) { SSM_NS(launch_bwd, bf16_t) } else { SSM_NS(launch_bwd, float) }
    return (int)hipGetLastError();
}

template <typename T, int V, int L>
static void launch_step(const SsmArgs& p, hipStream_t s) {
    const long long ch = p.B * p.D, nb = (ch + 256 / L - 1) / (256 / L), n4 = (nb + 3) / 4, x = n4 < (1 << 23) ? n4 : 1 << 23;
    if (nb >= 8192) k_ssm_step<T, V, L, 4><<<dim3((unsigned)x, (unsigned)((n4 + x - 1) / x)), 256, 0, s>>>(p);
    else k_ssm_step<T, V, L, 1><<<(unsigned)nb, 256, 0, s>>>(p);
}
template <typename T>
static void dispatch_step(const SsmArgs& p, hipStream_t s) {
    if (vec4(p.hT, p.N) && vec4(p.A, p.N) && (p.N & (p.N - 1)) == 0) {
        switch (p.N) {
            case 4: launch_step<T, 4, 1>(p, s); return;
            case 8: launch_step<T, 4, 2>(p, s); return;
            case 16: launch_step<T, 4, 4>(p, s); return;
            case 32: launch_step<T, 4, 8>(p, s); return;
            default: launch_step<T, 4, 16>(p, s); return;
        }
    }
    if (p.N <= 1) launch_step<T, 1, 1>(p, s);
    else if (p.N <= 2) launch_step<T, 1, 2>(p, s);
    else if (p.N <= 4) launch_step<T, 1, 4>(p, s);
    else if (p.N <= 8) launch_step<T, 1, 8>(p, s);
    else if (p.N <= 16) launch_step<T, 1, 16>(p, s);
    else if (p.N <= 32) launch_step<T, 1, 32>(p, s);
    else launch_step<T, 1, 64>(p, s);
}

DRL_API int drl_ssm_step(const SsmArgs* a, int bf16, hipStream_t s) {
    const SsmArgs p = *a;
    if (p.B <= 0 || p.D <= 0 || p.D >= (1ll << 31) || p.N <= 0 || p.N > 64 || p.B * p.D >= (1ll << 33)) return -1;
    const long long e = bf16 ? 2 : 4, cols = p.D * 4;
    if (!apart({{p.y, p.D * e, p.B, p.y_b * e}, state_view(p, p.hT)},
               {{p.u, p.D * e, p.B, p.u_b * e}, {p.dt, p.D * e, p.B, p.dt_b * e}, {p.z, p.D * e, p.B, p.z_b * e}, {p.Bm, p.N * e, p.B, p.B_b * e},
                {p.Cm, p.N * e, p.B, p.C_b * e}, {p.A, cols * p.N}, {p.Dp, cols}, {p.bias, cols}, {p.reset, p.B}})) return -3;
    if (bf16) dispatch_step<bf16_t>(p, s);
    else dispatch_step<float>(p, s);
    return (int)hipGetLastError();
}
