// SPDX-License-Identifier: Apache-2.0
// kda_tree.hip - a tree of drafted tokens through a KDA layer for gfx950: every node's output from one
// read of the state (k3hip_kda_tree_step), and the state moved along the accepted path
// (k3hip_kda_tree_commit).
//
// Node n of a tree continues the sequence from its parent p (the committed state where it has none):
//   S_n = (I - beta_n k_n k_n^T) Diag(a_n) S_p + beta_n k_n v_n^T,   o_n = S_n^T q_n,
// the recurrence of k3_kda_step (src/core/k3_ops.c:186-243) along each branch. Only S_0 is 64 KB a head;
// every other state differs from it by one rank a node, so the states are never formed. With
// E_nm = prod of a over the path from just below m down to n (E_n0: from the context), and
// w_m = beta_m (v_m - u_m) the value row that node m adds,
//   w_m = beta_m (v_m - (E_m0 k_m)^T S_0 - sum over m's ancestors j of (k_m . E_mj k_j) w_j)
//   o_n = (E_n0 q_n)^T S_0 + sum over n and its ancestors j of (q_n . E_nj k_j) w_j
// Decays are multiplied up the path, one product a step: no exponent of a sum, so no gate bound is
// needed and a decay of zero is just a zero.
#include "kda_internal.h"
#include "kda_prep_math.h"
#include "kda_tree.h"

namespace k3kda {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct TreeArgs {
    TreeSeqs t;
    int H, K;
    float lb, eps, q_scale;
    const void *qi, *ki, *vi;    // [B][N][P], in_dt
    int in_dt;
    const float *z, *bl;         // [B][N][P], [B][N][H]
    const void *gate;            // [B][N][P], g_dt
    int g_dt;
    const float *q_conv, *k_conv, *v_conv, *A_log, *dt_bias, *o_norm;
    float *hist;                 // [3][P][K-1] a sequence, h_stride floats apart
    long h_stride;
    float *S;                    // [H][D][D] a sequence, s_stride floats apart
    long s_stride;
    void *y;
    int y_dt;
    const int *accept;
    bool vec, vec_y;             // inputs and y may be accessed four elements at a time
};

__device__ __forceinline__ float load_any(const void *p, int dt, size_t i)
{
    return dt == K3HIP_BF16 ? load_act<K3HIP_BF16>(p, i) : load_act<K3HIP_F32>(p, i);
}

// Four adjacent elements i .. i + 3 of an activation, 16-byte (fp32) or 8-byte (bf16) aligned where vec.
__device__ __forceinline__ f4 load_four(const void *p, int dt, size_t i, bool vec)
{
    if (!vec) return f4{load_any(p, dt, i), load_any(p, dt, i + 1), load_any(p, dt, i + 2), load_any(p, dt, i + 3)};
    if (dt == K3HIP_F32) return *reinterpret_cast<const f4 *>(reinterpret_cast<const float *>(p) + i);
    const uint2 v = *reinterpret_cast<const uint2 *>(reinterpret_cast<const uint16_t *>(p) + i);
    return f4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
              __uint_as_float(v.y & 0xffff0000u)};
}

// The decay e^g of logit z (without its bias dt), ea = e^A_log.
__device__ __forceinline__ float decay_of(float lb, float ea, float z, float dt)
{
    return fast_exp(lb != 0.0f ? gate_bounded(lb, gate_a2(ea), z, dt) : -ea * softplus_ref(z + dt));
}

// CPL adjacent floats between registers and LDS, 16 bytes at a time where there are four.
template <int CPL>
__device__ __forceinline__ void lds_get(float (&x)[CPL], const float *p)
{
    if constexpr (CPL == 4) {
        const f4 v = *reinterpret_cast<const f4 *>(p);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
        for (int e = 0; e < CPL; e++) x[e] = p[e];
    }
}
template <int CPL>
__device__ __forceinline__ void lds_put(float *p, const float (&x)[CPL])
{
    if constexpr (CPL == 4) *reinterpret_cast<f4 *>(p) = f4{x[0], x[1], x[2], x[3]};
    else {
#pragma unroll
        for (int e = 0; e < CPL; e++) p[e] = x[e];
    }
}

template <int D, int TILES>
struct alignas(16) TreeLds {
    static constexpr int R = 16 * TILES;   // node rows, zero past the tree
    static constexpr int DP = D + 4;       // pitch: 16 rows x 4 adjacent floats on distinct banks
    static constexpr int AP = R + 4;
    float q[R * DP], k[R * DP], v[R * DP], a[R * DP];
    union {
        float A[R * AP];   // [j][m] above the diagonal: k_m . E_mj k_j; [n][j] on and below: q_n . E_nj k_j
        struct {
            float w[3][4][D], h[3][3][D];   // before it: the head's conv taps and history, tap and slot major
        } c;
    };
    float beta[R];
    uint64_t anc[R];   // the node and its ancestors, a bit each
    uint64_t bad[D];   // [value column] the nodes whose w is not finite there
    uint32_t up[R];    // the node, its parent, the parent's and the one after, a byte each; 0x80 + i: i back in the history
};

// One workgroup per (head, sequence), a wave per 16 value columns (value columns never meet before the
// norm). Everything is asked for at the start, in the order in which it is needed: the raw inputs (vectors of
// four channels), the conv's taps and history, the wave's columns of S as B fragments of
// v_mfma_f32_16x16x4_f32, the output gate. (K1 with loads of its own for each tap, 2 and 4 bytes a lane, held a
// workgroup for 42 us at 64 sequences x 16 nodes: 200 us a launch.) TILES: 16-row node tiles.
// Measured at 32 heads x 128: 64 sequences x 16 nodes 62 us (3.2 TB/s; three workgroups a CU in 80 registers, 2.7 rounds
// of 18 us: loads 5, conv 5, walk 2, products 3, solve 3), one sequence x 8 nodes 10 us, a chain of memory waits
// and barriers. Larger trees leave less beside each other: up to 32 nodes 127 registers and 78 KB, two workgroups a CU
// (16 sequences x 32 nodes 38 us, 32 x 32 69); up to 64 nodes 221 and 151 KB, one, whose chain nothing covers (16 x 64
// 119 us, one x 64 55).
template <int D, int TILES>
__global__ __launch_bounds__(4 * D, D == 128 && TILES == 1 ? 6 : 1) void kda_tree_kernel(const TreeArgs a)
{
    constexpr int NT = 4 * D;
    using L = TreeLds<D, TILES>;
    constexpr int R = L::R, DP = L::DP, AP = L::AP;
    constexpr int CPL = D >= 32 ? D / 32 : 1;
    constexpr int C4 = D / 4, HWS = NT / 32;
    extern __shared__ __attribute__((aligned(16))) char tree_smem[];
    L &s = *reinterpret_cast<L *>(tree_smem);
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int N = tree_count(a.t, b), K = a.K;
    const size_t P = (size_t)a.H * D, row0 = (size_t)b * a.t.N, c0 = (size_t)h * D;
    const float *hist = a.hist + (size_t)b * a.h_stride;
    const float *S = a.S + (size_t)b * a.s_stride + (size_t)h * D * D;

    // raw inputs: thread tid takes channels 4 (tid % C4) .. + 3 of rows tid / C4 + 16 i
    const int rch = 4 * (tid % C4), rrow = tid / C4;
    f4 raw[TILES][4];
#pragma unroll
    for (int i = 0; i < TILES; i++) {
        const int n = rrow + 16 * i;
        const size_t at = (row0 + (n < a.t.N ? n : 0)) * P + c0 + rch;   // also of rows that are no nodes: no wait for the count
        raw[i][0] = load_four(a.qi, a.in_dt, at, a.vec);
        raw[i][1] = load_four(a.ki, a.in_dt, at, a.vec);
        raw[i][2] = load_four(a.vi, a.in_dt, at, a.vec);
        raw[i][3] = load_four(a.z, K3HIP_F32, at, a.vec);
    }
    const f4 dtb = load_four(a.dt_bias, K3HIP_F32, c0 + rch, a.vec);
    const float A_log = a.A_log[h];
    const int par0 = tid < a.t.N ? tree_parent(a.t, b, tid) : -1;
    float s_bl[R / HWS];   // of this half-wave's rows
#pragma unroll
    for (int r = 0; r < R / HWS; r++) {
        const int n = (tid >> 5) + HWS * r;
        s_bl[r] = a.bl[(row0 + (n < a.t.N ? n : 0)) * a.H + h];
    }
    // taps and history of the head's channels, one (matrix, channel) a thread
    float tap[4], old[3];
    const int cm = tid / D, cc = tid % D;   // the fourth part of the threads has none
    if (cm < 3) {
        const float *w = (cm == 0 ? a.q_conv : cm == 1 ? a.k_conv : a.v_conv) + (c0 + cc) * K;
        const float *hs = hist + ((size_t)cm * P + c0 + cc) * (K - 1);
#pragma unroll
        for (int j = 0; j < 4; j++) tap[j] = j < K ? w[j] : 0.0f;
#pragma unroll
        for (int j = 0; j < 3; j++) old[j] = j < K - 1 ? hs[j] : 0.0f;
    }
    const int c16 = lane & 15, kq = lane >> 4, l32 = tid & 31, hw = tid >> 5;
    const bool active = l32 * CPL < D;
    const int cl = active ? l32 * CPL : 0;

    if (N == 0) return;
    constexpr int TPR = R / HWS;   // rows a half-wave, hw + HWS r
    // inputs to LDS (decays at once; zeros past the tree)
    {
        const float ea = expf(A_log);
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const int n = rrow + 16 * i, at = n * DP + rch;
            const bool ok = n < N;
            f4 d;
#pragma unroll
            for (int e = 0; e < 4; e++) d[e] = decay_of(a.lb, ea, raw[i][3][e], dtb[e]);
            *reinterpret_cast<f4 *>(s.q + at) = ok ? raw[i][0] : f4(0.0f);
            *reinterpret_cast<f4 *>(s.k + at) = ok ? raw[i][1] : f4(0.0f);
            *reinterpret_cast<f4 *>(s.v + at) = ok ? raw[i][2] : f4(0.0f);
            *reinterpret_cast<f4 *>(s.a + at) = ok ? d : f4(0.0f);
        }
    }
    if (tid < 64) {   // lane = node
        const uint64_t anc = tree_ancestors(par0);
        uint32_t up = lane & 0x7f;
        int m = lane, past = 0;
#pragma unroll
        for (int j = 1; j < 4; j++) {
            const int p = __shfl(par0, m < 0 ? 0 : m, 64);
            m = m < 0 ? -1 : p;
            past += m < 0;
            up |= (uint32_t)(m < 0 ? 0x80 + past : m) << (8 * j);
        }
        if (lane < R) {
            s.anc[lane] = anc;
            s.up[lane] = up;
        }
    }
    if (cm < 3) {
#pragma unroll
        for (int j = 0; j < 4; j++) s.c.w[cm][j][cc] = tap[j];
#pragma unroll
        for (int j = 0; j < 3; j++) s.c.h[cm][j][cc] = old[j];
    }
    __syncthreads();

    // K1: short conv over the node and its ancestors, then the history (kda_prep_math.h's arithmetic, taps oldest
    // first), L2 norm of q and k; a (matrix, node) a half-wave, results held until all inputs were read
    constexpr int KPT = 3 * R / HWS;
    float kx[KPT][CPL];
#pragma unroll
    for (int i = 0; i < KPT; i++) {
        const int task = hw + HWS * i, which = task % 3, n = task / 3;
        if (n >= N) continue;
        const float *x = which == 0 ? s.q : (which == 1 ? s.k : s.v);
        const uint32_t up = s.up[n];
        float in[4][CPL];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int m = up >> (8 * j) & 0xff;
            lds_get<CPL>(in[j], (m < 0x80 ? x + m * DP : s.c.h[which][max(K - 1 - (m - 0x80), 0)]) + cl);
        }
        float w[4][CPL];   // tap j tokens back
#pragma unroll
        for (int j = 0; j < 4; j++) lds_get<CPL>(w[j], s.c.w[which][max(K - 1 - j, 0)] + cl);
#pragma unroll
        for (int e = 0; e < CPL; e++) {
            float acc = w[0][e] * in[0][e];
#pragma unroll
            for (int j = 3; j >= 1; j--) acc = j < K ? __builtin_fmaf(w[j][e], in[j][e], acc) : acc;
            kx[i][e] = active ? acc * fast_sigmoid(acc) : 0.0f;
        }
        if (which < 2) l2norm_half<CPL>(kx[i]);
    }
    // S fragments: lane l holds rows 4 t + l / 16, column 16 wv + l % 16
    float sf[D / 4];
#pragma unroll
    for (int t = 0; t < D / 4; t++) sf[t] = S[(size_t)(4 * t + kq) * D + 16 * wv + c16];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KPT; i++) {
        const int task = hw + HWS * i, which = task % 3, n = task / 3;
        if (n >= N || !active) continue;
#pragma unroll
        for (int e = 0; e < CPL; e++) kx[i][e] = which == 0 ? kx[i][e] * a.q_scale : kx[i][e];
        lds_put<CPL>((which == 0 ? s.q : which == 1 ? s.k : s.v) + n * DP + cl, kx[i]);
    }
    for (int i = tid; i < R * AP; i += NT) s.A[i] = 0.0f;
    __syncthreads();

    // pair products: a half-wave walks from node m up its path (its ancestors from the highest number down),
    // the next ancestor's row asked for before the current one's products, and ends with E_m0
    float kt[TPR][CPL], qt[TPR][CPL];
#pragma unroll
    for (int r = 0; r < TPR; r++) {
        const int m = hw + HWS * r;
        if (m < N) {
            const float beta = fast_sigmoid(s_bl[r]);
            uint64_t left = s.anc[m];
            float E[CPL], kj[CPL], aj[CPL];
            lds_get<CPL>(kt[r], s.k + m * DP + cl);
            lds_get<CPL>(qt[r], s.q + m * DP + cl);
            lds_get<CPL>(aj, s.a + m * DP + cl);
#pragma unroll
            for (int e = 0; e < CPL; e++) {
                E[e] = active ? 1.0f : 0.0f;
                kj[e] = kt[r][e];
            }
            for (int j = m; j >= 0;) {
                left &= (1ull << j) - 1;
                const int up = left ? 63 - __builtin_clzll(left) : -1, ld = max(up, 0);
                float kn[CPL], an[CPL], kk = 0.0f, qk = 0.0f;
                lds_get<CPL>(kn, s.k + ld * DP + cl);
                lds_get<CPL>(an, s.a + ld * DP + cl);
#pragma unroll
                for (int e = 0; e < CPL; e++) {
                    const float x = E[e] * kj[e];
                    kk = __builtin_fmaf(kt[r][e], x, kk);
                    qk = __builtin_fmaf(qt[r][e], x, qk);
                    E[e] *= aj[e];
                    kj[e] = kn[e];
                    aj[e] = an[e];
                }
                kk = half_wave_sum(kk);
                qk = half_wave_sum(qk);
                if (l32 == 0) {
                    if (j != m) s.A[j * AP + m] = beta * kk;
                    s.A[m * AP + j] = qk;
                }
                j = up;
            }
#pragma unroll
            for (int e = 0; e < CPL; e++) {
                kt[r][e] *= E[e];
                qt[r][e] *= E[e];
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < TPR; r++) {
        const int m = hw + HWS * r;
        if (l32 == 0) s.beta[m] = m < N ? fast_sigmoid(s_bl[r]) : 0.0f;
        if (m < N && active) {
            lds_put<CPL>(s.k + m * DP + cl, kt[r]);
            lds_put<CPL>(s.q + m * DP + cl, qt[r]);
        }
    }
    __syncthreads();

    // (E k)^T S_0 and (E q)^T S_0; the right sides of the system into s.a (the decays are used up).
    // C layout: lane holds rows 4 kq + i, column c16
    f32x4 oq[TILES];
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        f32x4 u = {0.0f, 0.0f, 0.0f, 0.0f};
        oq[t] = u;
        const float *kr = s.k + (16 * t + c16) * DP + kq, *qr = s.q + (16 * t + c16) * DP + kq;
#pragma unroll
        for (int x = 0; x < D / 4; x++) {
            u = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[4 * x], sf[x], u, 0, 0, 0);
            oq[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(qr[4 * x], sf[x], oq[t], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int m = 16 * t + 4 * kq + i, at = m * DP + 16 * wv + c16;
            s.a[at] = s.beta[m] * (s.v[at] - u[i]);
        }
    }
    __syncthreads();

    // output gate and norm: half-wave hw takes nodes hw, hw + HWS, ...
    constexpr int GPT = R / HWS;   // its nodes
    float gate[GPT][CPL], on[CPL];
#pragma unroll
    for (int i = 0; i < GPT; i++) {
        const int n = hw + HWS * i;
#pragma unroll
        for (int e = 0; e < CPL; e++) gate[i][e] = load_any(a.gate, a.g_dt, (row0 + (n < a.t.N ? n : 0)) * P + c0 + cl + e);
    }
#pragma unroll
    for (int e = 0; e < CPL; e++) on[e] = a.o_norm[cl + e];

    // forward substitution, a thread per value column, 16 rows at a time in registers: w_m = rhs_m - sum_j
    // beta_m A_mj w_j. A w that is not finite is noted and taken as zero: zeros of A would spread it to nodes
    // that do not follow it, and those that do are set below.
    if (tid < D) {
        uint64_t bad = 0;
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            float w[16];
#pragma unroll
            for (int i = 0; i < 16; i++) w[i] = s.a[(16 * t + i) * DP + tid];
            for (int j = 0; j < 16 * t; j++) {
                const float x = s.a[j * DP + tid];
                const float *Aj = s.A + j * AP + 16 * t;
#pragma unroll
                for (int i = 0; i < 16; i++) w[i] = __builtin_fmaf(-Aj[i], x, w[i]);
            }
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const bool inf = !(fabsf(w[i]) < INFINITY);
                bad |= (uint64_t)inf << (16 * t + i);
                w[i] = inf ? 0.0f : w[i];
                const float *Ai = s.A + (16 * t + i) * AP + 16 * t;
#pragma unroll
                for (int q = (i + 1) / 4; q < 4; q++) {
                    const f4 c = *reinterpret_cast<const f4 *>(Ai + 4 * q);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (4 * q + e > i) w[4 * q + e] = __builtin_fmaf(-c[e], w[i], w[4 * q + e]);
                }
            }
#pragma unroll
            for (int i = 0; i < 16; i++) s.a[(16 * t + i) * DP + tid] = w[i];
        }
        s.bad[tid] = bad;
    }
    __syncthreads();

    // o = (E q)^T S_0 + A_qk w, into s.v
    const uint64_t bad = s.bad[16 * wv + c16];
#pragma unroll
    for (int t = 0; t < TILES; t++) {
#pragma unroll
        for (int x = 0; x < 4 * (t + 1); x++) {
            const int n = 16 * t + c16, j = 4 * x + kq;
            const float f = j <= n ? s.A[n * AP + j] : 0.0f;
            oq[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(f, s.a[j * DP + 16 * wv + c16], oq[t], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int n = 16 * t + 4 * kq + i;
            s.v[n * DP + 16 * wv + c16] = s.anc[n] & bad ? NAN : oq[t][i];
        }
    }
    __syncthreads();

    // K4, a node per half-wave
#pragma unroll
    for (int i = 0; i < GPT; i++) {
        const int n = hw + HWS * i;
        if (n >= N) continue;
        float x[CPL], part = 0.0f;
        lds_get<CPL>(x, s.v + n * DP + cl);
#pragma unroll
        for (int e = 0; e < CPL; e++) {
            part += active ? x[e] * x[e] : 0.0f;
        }
        const float inv = __builtin_amdgcn_rsqf(half_wave_sum(part) / (float)D + a.eps);
        if (!active) continue;
        const size_t at = (row0 + n) * P + c0 + cl;
#pragma unroll
        for (int e = 0; e < CPL; e++) x[e] = on[e] * x[e] * inv * fast_sigmoid(gate[i][e]);
        if (CPL == 4 && a.vec_y) {
            if (a.y_dt == K3HIP_BF16)
                *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(a.y) + at) =
                    uint2{(uint32_t)f2bf(x[0]) | ((uint32_t)f2bf(x[CPL > 1 ? 1 : 0]) << 16),
                          (uint32_t)f2bf(x[CPL > 2 ? 2 : 0]) | ((uint32_t)f2bf(x[CPL > 3 ? 3 : 0]) << 16)};
            else *reinterpret_cast<f4 *>(reinterpret_cast<float *>(a.y) + at) = f4{x[0], x[CPL > 1 ? 1 : 0], x[CPL > 2 ? 2 : 0], x[CPL > 3 ? 3 : 0]};
        } else {
#pragma unroll
            for (int e = 0; e < CPL; e++) {
                if (a.y_dt == K3HIP_BF16) reinterpret_cast<uint16_t *>(a.y)[at + e] = f2bf(x[e]);
                else reinterpret_cast<float *>(a.y)[at + e] = x[e];
            }
        }
    }
}

// S := S of the accepted node, one workgroup per (head, sequence): the path's nodes one after the other
// on a state held in registers (kda_decode_kernel's tile), so S is read once and written once whatever
// the path's length. K1 of up to TREE_CK nodes at a time runs before them, from their inputs and the three before
// them in LDS. The conv history of the head's channels becomes the last K - 1 inputs of history and path.
// Measured at 32 heads x 128: 64 sequences x 16 nodes 59 us (4.4 TB/s, reading and writing the state; a plain copy
// reaches 4.9, kda_decode_kernel 5.8 on the same states in place, with a store that no cache keeps), one sequence 9.3 us. Loading taps, inputs and history where they were used: 88 us.
constexpr int TREE_CK = 16;

template <int D>
__global__ __launch_bounds__(4 * D) void kda_tree_commit_kernel(const TreeArgs a)
{
    constexpr int NT = 4 * D, CPR = D / 4, RPP = NT / CPR, NPASS = D / RPP;
    constexpr int CPL = D >= 32 ? D / 32 : 1, HWS = NT / 32, KPT = 2 * TREE_CK / HWS;
    static_assert(RPP == TREE_CK, "a pass of the workgroup covers the rows of a chunk");
    // inputs of k and v: row 3 + i is path node i0 + i, rows 0 .. 2 the three before; then, from row 0, k and v
    __shared__ __attribute__((aligned(16))) float s_x[2][3 + TREE_CK][D], s_a[TREE_CK][D], s_w[2][4][D];
    __shared__ float s_b[TREE_CK];
    __shared__ f4 s_red[2][RPP][CPR];
    __shared__ int s_node[TREE_MAX], s_n;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int cg = tid % CPR, rs = tid / CPR;
    const int N = tree_count(a.t, b), node = a.accept[b], K = a.K, K1 = K - 1;
    if (node < 0 || node >= N) return;
    const size_t P = (size_t)a.H * D, row0 = (size_t)b * a.t.N, c0 = (size_t)h * D;
    float *hist = a.hist + (size_t)b * a.h_stride;
    const int par0 = tid < 64 && lane < N ? tree_parent(a.t, b, lane) : -1;
    float tap[4];   // of one (matrix, channel) a thread, half the threads
    const int cm = tid / D, cc = tid % D;
    if (cm < 2) {
        const float *w = (cm == 0 ? a.k_conv : a.v_conv) + (c0 + cc) * K;
#pragma unroll
        for (int j = 0; j < 4; j++) tap[j] = j < K ? w[j] : 0.0f;
    }
    const f4 dtb = load_four(a.dt_bias, K3HIP_F32, c0 + 4 * cg, a.vec);
    const float A_log = a.A_log[h];
    f4 *Sp = reinterpret_cast<f4 *>(a.S + (size_t)b * a.s_stride + (size_t)h * D * D);
    f4 s[NPASS];
#pragma unroll
    for (int m = 0; m < NPASS; m++) s[m] = __builtin_nontemporal_load(&Sp[(rs + m * RPP) * CPR + cg]);
    if (tid < 64) {
        const uint64_t m = tree_ancestors(par0);
        const uint64_t path = ((uint64_t)__shfl((uint32_t)(m >> 32), node, 64) << 32) | __shfl((uint32_t)m, node, 64);
        if (path >> lane & 1) s_node[__popcll(path & ((1ull << lane) - 1))] = lane;
        if (lane == 0) s_n = __popcll(path);
    }
    if (cm < 2)
#pragma unroll
        for (int j = 0; j < 4; j++) s_w[cm][j][cc] = tap[j];
    __syncthreads();
    const int n = s_n;
    const int l32 = tid & 31, hw = tid >> 5;
    const bool active = l32 * CPL < D;
    const int cl = active ? l32 * CPL : 0;
    // inputs 4 cg .. + 3 of path position i: a node's, or the history's
    auto input = [&](int which, int i) -> f4 {
        if (i >= 0) return load_four(which ? a.vi : a.ki, a.in_dt, (row0 + s_node[i]) * P + c0 + 4 * cg, a.vec);
        f4 x = 0.0f;
        if (K1 + i >= 0)
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = hist[((size_t)(1 + which) * P + c0 + 4 * cg + e) * K1 + K1 + i];
        return x;
    };
    for (int i0 = 0; i0 < n; i0 += TREE_CK) {
        const int ni = min(TREE_CK, n - i0);
        if (rs < ni) {
            const f4 k = input(0, i0 + rs), v = input(1, i0 + rs);
            const f4 z = load_four(a.z, K3HIP_F32, (row0 + s_node[i0 + rs]) * P + c0 + 4 * cg, a.vec);
            const float ea = expf(A_log);
            f4 d;
#pragma unroll
            for (int e = 0; e < 4; e++) d[e] = decay_of(a.lb, ea, z[e], dtb[e]);
            *reinterpret_cast<f4 *>(&s_x[0][3 + rs][4 * cg]) = k;
            *reinterpret_cast<f4 *>(&s_x[1][3 + rs][4 * cg]) = v;
            *reinterpret_cast<f4 *>(&s_a[rs][4 * cg]) = d;
        }
        if (rs >= RPP - 3)
#pragma unroll
            for (int which = 0; which < 2; which++)
                *reinterpret_cast<f4 *>(&s_x[which][rs - (RPP - 3)][4 * cg]) = input(which, i0 - 3 + rs - (RPP - 3));
        if (tid < ni) s_b[tid] = fast_sigmoid(a.bl[(row0 + s_node[i0 + tid]) * a.H + h]);
        __syncthreads();
        float kx[KPT][CPL];
#pragma unroll
        for (int t = 0; t < KPT; t++) {
            const int task = hw + HWS * t, which = task & 1, i = task >> 1;
            if (i >= ni) continue;
            float acc[CPL];
#pragma unroll
            for (int j = 0; j < 4; j++) {   // tap 0 now, then the oldest first (kda_prep_math.h)
                const int back = j == 0 ? 0 : 4 - j;
                float x[CPL], w[CPL];
                lds_get<CPL>(x, &s_x[which][3 + i - back][cl]);
                lds_get<CPL>(w, &s_w[which][max(K1 - back, 0)][cl]);
#pragma unroll
                for (int e = 0; e < CPL; e++) acc[e] = j == 0 ? w[e] * x[e] : (back < K ? __builtin_fmaf(w[e], x[e], acc[e]) : acc[e]);
            }
#pragma unroll
            for (int e = 0; e < CPL; e++) kx[t][e] = active ? acc[e] * fast_sigmoid(acc[e]) : 0.0f;
            if (which == 0) l2norm_half<CPL>(kx[t]);
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < KPT; t++) {
            const int task = hw + HWS * t, which = task & 1, i = task >> 1;
            if (i < ni && active) lds_put<CPL>(&s_x[which][i][cl], kx[t]);
        }
        __syncthreads();
        for (int i = 0; i < ni; i++) {
            f4 u = 0.0f;
#pragma unroll
            for (int m = 0; m < NPASS; m++) {
                const int r = rs + m * RPP;
                s[m] = s[m] * s_a[i][r];
                u = u + s_x[0][i][r] * s[m];
            }
            s_red[i & 1][rs][cg] = u;
            __syncthreads();   // the other half was last read before this barrier's predecessor
            f4 ut = s_red[i & 1][0][cg];
#pragma unroll
            for (int r = 1; r < RPP; r++) ut = ut + s_red[i & 1][r][cg];
            const f4 d = (*reinterpret_cast<const f4 *>(&s_x[1][i][4 * cg]) - ut) * s_b[i];
#pragma unroll
            for (int m = 0; m < NPASS; m++) s[m] = s[m] + s_x[0][i][rs + m * RPP] * d;
        }
        __syncthreads();   // the chunk's arrays are free; the history's last reader is done
    }
#pragma unroll
    for (int m = 0; m < NPASS; m++) __builtin_nontemporal_store(s[m], &Sp[(rs + m * RPP) * CPR + cg]);
    // history: slot j of the new one is entry n + j of (the old K - 1, then the path's inputs); ascending
    // order, so a slot is read before the one that replaces it is written
    for (int c = tid; c < 3 * D; c += NT) {
        const int which = c / D;
        const size_t ch = c0 + c % D;
        const void *src = which == 0 ? a.qi : (which == 1 ? a.ki : a.vi);
        float *hs = hist + ((size_t)which * P + ch) * K1;
        for (int j = 0; j < K1; j++) {
            const int at = n + j;
            hs[j] = at < K1 ? hs[at] : load_any(src, a.in_dt, (row0 + s_node[at - K1]) * P + ch);
        }
    }
}

template <int D, int TILES>
int launch_tree(int B, const TreeArgs &a, hipStream_t st)
{
    using L = TreeLds<D, TILES>;
    static_assert(sizeof(L) <= 160 * 1024, "LDS");
    const void *kern = (const void *)kda_tree_kernel<D, TILES>;
    if (sizeof(L) > 64 * 1024) K3_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(L)));
    hipLaunchKernelGGL((kda_tree_kernel<D, TILES>), dim3(a.H, B), dim3(4 * D), sizeof(L), st, a);
    K3_LAUNCHED();
    return K3HIP_OK;
}

template <int D>
int launch_tree_d(int B, const TreeArgs &a, hipStream_t st)
{
    switch ((a.t.N + 15) / 16) {
    case 1: return launch_tree<D, 1>(B, a, st);
    case 2: return launch_tree<D, 2>(B, a, st);
    case 3: return launch_tree<D, 3>(B, a, st);
    default: return launch_tree<D, 4>(B, a, st);
    }
}

// What both entry points check alike.
int tree_args(const char *who, TreeArgs &a, int B, int N, int H, int D, int K, float gate_lb, int in_dtype,
              const void *q_in, const void *k_in, const void *v_in, const float *z, const float *b_logit,
              const float *q_conv, const float *k_conv, const float *v_conv, const float *A_log, const float *dt_bias,
              const float *conv_state, long conv_stride, const float *S, long s_stride)
{
    if (B < 0 || N < 0 || H <= 0) K3_FAIL(K3HIP_EINVAL, "%s: B=%d N=%d H=%d", who, B, N, H);
    if (!is_pow2_head(D)) K3_FAIL(K3HIP_EUNSUPPORTED, "%s: D=%d not in {16,32,64,128}", who, D);
    if (K < 1 || K > 4) K3_FAIL(K3HIP_EUNSUPPORTED, "%s: conv_k=%d not in 1..4", who, K);
    if (N > TREE_MAX) K3_FAIL(K3HIP_EUNSUPPORTED, "%s: a tree of %d nodes (at most %d)", who, N, TREE_MAX);
    if (B > 65535) K3_FAIL(K3HIP_EINVAL, "%s: B=%d (at most 65535)", who, B);
    if (!(gate_lb <= 0.0f)) K3_FAIL(K3HIP_EINVAL, "%s: gate_lb=%g (a bound <= 0; 0 selects the softplus gate)", who, gate_lb);
    if (in_dtype != K3HIP_F32 && in_dtype != K3HIP_BF16) K3_FAIL(K3HIP_EINVAL, "%s: in_dtype=%d", who, in_dtype);
    const long P = (long)H * D;
    if (s_stride < P * D || (s_stride & 3) || (K > 1 && conv_stride < 3 * P * (K - 1)))
        K3_FAIL(K3HIP_EINVAL, "%s: strides of S %ld (at least H D D, a multiple of 4) and conv_state %ld", who, s_stride, conv_stride);
    if (B == 0 || N == 0) return K3HIP_OK;
    if (!q_in || !k_in || !v_in || !z || !b_logit || !q_conv || !k_conv || !v_conv || !A_log || !dt_bias || !S ||
        (K > 1 && !conv_state))
        K3_FAIL(K3HIP_EINVAL, "%s: NULL argument (conv_state is needed for conv_k > 1)", who);
    if ((uintptr_t)S & 15) K3_FAIL(K3HIP_EINVAL, "%s: S needs 16-byte alignment", who);
    a.H = H; a.K = K; a.lb = gate_lb;
    a.qi = q_in; a.ki = k_in; a.vi = v_in; a.in_dt = in_dtype;
    a.z = z; a.bl = b_logit;
    a.q_conv = q_conv; a.k_conv = k_conv; a.v_conv = v_conv; a.A_log = A_log; a.dt_bias = dt_bias;
    a.hist = const_cast<float *>(conv_state); a.h_stride = conv_stride;
    a.S = const_cast<float *>(S); a.s_stride = s_stride;
    a.vec = (((uintptr_t)q_in | (uintptr_t)k_in | (uintptr_t)v_in) & (in_dtype == K3HIP_F32 ? 15 : 7)) == 0 &&
            (((uintptr_t)z | (uintptr_t)dt_bias) & 15) == 0;
    return K3HIP_OK;
}

}  // namespace

}  // namespace k3kda

using namespace k3kda;

extern "C" int k3hip_kda_tree_step(int B, int N, int H, int D, int K, float gate_lb, float rms_eps, int in_dtype,
                                   const void *q_in, const void *k_in, const void *v_in, const float *z,
                                   const float *b_logit, const void *gate, int gate_dtype, const float *q_conv,
                                   const float *k_conv, const float *v_conv, const float *A_log, const float *dt_bias,
                                   const float *o_norm, const float *conv_state, long conv_stride, float q_scale,
                                   const float *S, long s_stride, const int *counts, const int *parents, void *y,
                                   int y_dtype, void *stream)
{
    clear_error();
    static const char *who = "k3hip_kda_tree_step";
    TreeArgs a{};
    if (int rc = tree_args(who, a, B, N, H, D, K, gate_lb, in_dtype, q_in, k_in, v_in, z, b_logit, q_conv, k_conv, v_conv,
                           A_log, dt_bias, conv_state, conv_stride, S, s_stride))
        return rc;
    if ((gate_dtype != K3HIP_F32 && gate_dtype != K3HIP_BF16) || (y_dtype != K3HIP_F32 && y_dtype != K3HIP_BF16))
        K3_FAIL(K3HIP_EINVAL, "%s: dtypes gate=%d y=%d", who, gate_dtype, y_dtype);
    if (B == 0 || N == 0) return K3HIP_OK;
    if (!gate || !o_norm || !y) K3_FAIL(K3HIP_EINVAL, "%s: NULL gate, o_norm or y", who);
    a.t = TreeSeqs{N, nullptr, counts, parents};
    a.eps = rms_eps; a.q_scale = q_scale;
    a.gate = gate; a.g_dt = gate_dtype; a.o_norm = o_norm;
    a.y = y; a.y_dt = y_dtype;
    a.vec_y = ((uintptr_t)y & (y_dtype == K3HIP_F32 ? 15 : 7)) == 0;
    switch (D) {
    case 16: return launch_tree_d<16>(B, a, as_stream(stream));
    case 32: return launch_tree_d<32>(B, a, as_stream(stream));
    case 64: return launch_tree_d<64>(B, a, as_stream(stream));
    default: return launch_tree_d<128>(B, a, as_stream(stream));
    }
}

extern "C" int k3hip_kda_tree_commit(int B, int N, int H, int D, int K, float gate_lb, int in_dtype, const void *q_in,
                                     const void *k_in, const void *v_in, const float *z, const float *b_logit,
                                     const float *q_conv, const float *k_conv, const float *v_conv, const float *A_log,
                                     const float *dt_bias, float *conv_state, long conv_stride, float *S,
                                     long s_stride, const int *counts, const int *parents, const int *accept,
                                     void *stream)
{
    clear_error();
    static const char *who = "k3hip_kda_tree_commit";
    TreeArgs a{};
    if (int rc = tree_args(who, a, B, N, H, D, K, gate_lb, in_dtype, q_in, k_in, v_in, z, b_logit, q_conv, k_conv, v_conv,
                           A_log, dt_bias, conv_state, conv_stride, S, s_stride))
        return rc;
    if (B == 0 || N == 0) return K3HIP_OK;
    if (!accept) K3_FAIL(K3HIP_EINVAL, "%s: NULL accept", who);
    a.t = TreeSeqs{N, nullptr, counts, parents};
    a.accept = accept;
#define K3_TC(DD) hipLaunchKernelGGL((kda_tree_commit_kernel<DD>), dim3(H, B), dim3(4 * DD), 0, as_stream(stream), a)
    switch (D) {
    case 16: K3_TC(16); break;
    case 32: K3_TC(32); break;
    case 64: K3_TC(64); break;
    default: K3_TC(128); break;
    }
#undef K3_TC
    K3_LAUNCHED();
    return K3HIP_OK;
}
