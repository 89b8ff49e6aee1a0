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
};

__device__ __forceinline__ float load_any(const void *p, int dt, size_t i)
{
    return dt == K3HIP_BF16 ? load_act<K3HIP_BF16>(p, i) : load_act<K3HIP_F32>(p, i);
}

// K1 of one node by one half-wave, CPL adjacent channels a lane from channel c0 of the layer (cl of the
// head): which = 0, 1, 2 the short conv of q, k, v over the node and its ancestors, then the history
// (the arithmetic of kda_prep_math.h, taps oldest first), L2-normalised for q and k. par: the sequence's
// parents in LDS; row0: its first row.
template <int CPL>
__device__ __forceinline__ void tree_conv(float (&x)[CPL], const TreeArgs &a, int which, int n, const int *par, size_t row0,
                                          size_t P, size_t c0, bool active, const float *hist)
{
    const float *cw = which == 0 ? a.q_conv : (which == 1 ? a.k_conv : a.v_conv);
    const void *src = which == 0 ? a.qi : (which == 1 ? a.ki : a.vi);
    const int K = a.K;
    float in[4][CPL];   // inputs 0 .. 3 tokens back
    int m = n, past = 0;   // past: tokens back into the history (1 = its newest)
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int hs = (K - 1) - past;
#pragma unroll
        for (int e = 0; e < CPL; e++) {
            in[j][e] = 0.0f;
            if (j < K) {
                if (m >= 0) in[j][e] = load_any(src, a.in_dt, (row0 + m) * P + c0 + e);
                else in[j][e] = hist[((size_t)which * P + c0 + e) * (K - 1) + hs];
            }
        }
        if (m >= 0) m = par[m];
        if (m < 0) past++;
    }
#pragma unroll
    for (int e = 0; e < CPL; e++) {
        const float *w = cw + (c0 + e) * K;
        float acc = w[K - 1] * in[0][e];
#pragma unroll
        for (int j = 3; j >= 1; j--)
            if (j < K) acc = __builtin_fmaf(w[K - 1 - j], in[j][e], acc);
        x[e] = active ? acc * fast_sigmoid(acc) : 0.0f;
    }
    if (which < 2) l2norm_half<CPL>(x);
}

// The decay of one node, as above.
template <int CPL>
__device__ __forceinline__ void tree_decay(float (&x)[CPL], const TreeArgs &a, size_t row, int h, size_t P, size_t c0)
{
    const float ea = expf(a.A_log[h]);
#pragma unroll
    for (int e = 0; e < CPL; e++) {
        const float z = a.z[row * P + c0 + e], dt = a.dt_bias[c0 + e];
        const float g = a.lb != 0.0f ? gate_bounded(a.lb, gate_a2(ea), z, dt) : -ea * softplus_ref(z + dt);
        x[e] = fast_exp(g);
    }
}

// Sum over the 16 lanes of a row, in every lane.
__device__ __forceinline__ float row_sum(float x)
{
    x = x + dpp_f<0xB1>(x);    // lane ^ 1
    x = x + dpp_f<0x4E>(x);    // lane ^ 2
    x = x + dpp_f<0x141>(x);   // mirror in 8
    return x + dpp_f<0x140>(x);   // mirror in 16
}

template <int D, int TILES>
struct TreeLds {
    static constexpr int R = 16 * TILES;   // node rows, zero past the tree
    static constexpr int DP = D + 4;       // pitch: 16 rows x 4 adjacent floats on distinct banks
    static constexpr int AP = R + 4;
    float q[R * DP], k[R * DP], v[R * DP], a[R * DP];
    float A[R * AP];   // [j][m] above the diagonal: k_m . E_mj k_j; [n][j] on and below: q_n . E_nj k_j
    float beta[R];
    int par[R];
};

// One workgroup per (head, sequence), a wave per 16 value columns (value columns never meet before the
// norm): the wave's columns of S are asked for first, as the B fragments of v_mfma_f32_16x16x4_f32, and
// arrive while K1 and the pair products run. TILES: 16-row node tiles.
template <int D, int TILES>
__global__ __launch_bounds__(4 * D) void kda_tree_kernel(const TreeArgs a)
{
    constexpr int NT = 4 * D;
    using L = TreeLds<D, TILES>;
    constexpr int R = L::R, DP = L::DP, AP = L::AP;
    constexpr int CPL = D >= 32 ? D / 32 : 1;
    extern __shared__ __attribute__((aligned(16))) char tree_smem[];
    L &s = *reinterpret_cast<L *>(tree_smem);
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int N = tree_count(a.t, b);
    if (N == 0) return;
    const size_t P = (size_t)a.H * D, row0 = (size_t)b * a.t.N;
    const float *hist = a.hist + (size_t)b * a.h_stride;
    const float *S = a.S + (size_t)b * a.s_stride + (size_t)h * D * D;

    // S fragments: lane l holds rows 4 t + l / 16, column 16 wv + l % 16
    const int c16 = lane & 15, kq = lane >> 4;
    float sf[D / 4];
#pragma unroll
    for (int t = 0; t < D / 4; t++) sf[t] = S[(size_t)(4 * t + kq) * D + 16 * wv + c16];

    for (int i = tid; i < R * AP; i += NT) s.A[i] = 0.0f;
    if (tid < R) {
        s.par[tid] = tid < N ? tree_parent(a.t, b, tid) : -1;
        s.beta[tid] = tid < N ? fast_sigmoid(a.bl[(row0 + tid) * a.H + h]) : 0.0f;
    }
    for (int i = tid; i < (R - N) * DP; i += NT) {
        const int at = N * DP + i;
        s.q[at] = s.k[at] = s.v[at] = s.a[at] = 0.0f;
    }
    __syncthreads();

    // K1, a task of a node per half-wave
    {
        const int l32 = tid & 31;
        const bool active = l32 * CPL < D;
        const int cl = active ? l32 * CPL : 0;
        const size_t c0 = (size_t)h * D + cl;
        for (int task = tid >> 5; task < 4 * N; task += NT / 32) {
            const int which = task & 3, n = task >> 2;
            float x[CPL];
            if (which < 3) tree_conv<CPL>(x, a, which, n, s.par, row0, P, c0, active, hist);
            else tree_decay<CPL>(x, a, row0 + n, h, P, c0);
            float *dst = (which == 0 ? s.q : which == 1 ? s.k : which == 2 ? s.v : s.a) + n * DP + cl;
            if (active)
#pragma unroll
                for (int e = 0; e < CPL; e++) dst[e] = which == 0 ? x[e] * a.q_scale : x[e];
        }
    }
    __syncthreads();

    // pair products: 16 lanes walk from node m up its path, D / 16 channels a lane, and end with E_m0
    constexpr int CH = D / 16, GR = NT / 16;
    constexpr int RPG = (R + GR - 1) / GR;   // rows a group of lanes
    float kt[RPG][CH], qt[RPG][CH];
#pragma unroll
    for (int r = 0; r < RPG; r++) {
        const int m = (tid >> 4) + r * GR;
        if (m < N) {
            float E[CH];
#pragma unroll
            for (int e = 0; e < CH; e++) {
                E[e] = 1.0f;
                kt[r][e] = s.k[m * DP + CH * c16 + e];
                qt[r][e] = s.q[m * DP + CH * c16 + e];
            }
            for (int j = m; j >= 0; j = s.par[j]) {
                float kk = 0.0f, qk = 0.0f;
#pragma unroll
                for (int e = 0; e < CH; e++) {
                    const float x = E[e] * s.k[j * DP + CH * c16 + e];
                    kk = __builtin_fmaf(kt[r][e], x, kk);
                    qk = __builtin_fmaf(qt[r][e], x, qk);
                    E[e] *= s.a[j * DP + CH * c16 + e];
                }
                kk = row_sum(kk);
                qk = row_sum(qk);
                if (c16 == 0) {
                    if (j != m) s.A[j * AP + m] = kk;
                    s.A[m * AP + j] = qk;
                }
            }
#pragma unroll
            for (int e = 0; e < CH; e++) {
                kt[r][e] *= E[e];
                qt[r][e] *= E[e];
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RPG; r++) {
        const int m = (tid >> 4) + r * GR;
        if (m < N)
#pragma unroll
            for (int e = 0; e < CH; e++) {
                s.k[m * DP + CH * c16 + e] = kt[r][e];
                s.q[m * DP + CH * c16 + e] = qt[r][e];
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

    // forward substitution, a thread per value column: w_m = rhs_m - beta_m sum_j A_mj w_j, 16 rows at a
    // time in registers
    if (tid < D) {
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            float w[16];
#pragma unroll
            for (int i = 0; i < 16; i++) w[i] = 0.0f;
            for (int j = 0; j < 16 * t; j++) {
                const float x = s.a[j * DP + tid];
                const float *Aj = s.A + j * AP + 16 * t;
#pragma unroll
                for (int i = 0; i < 16; i++) w[i] = __builtin_fmaf(Aj[i], x, w[i]);
            }
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int m = 16 * t + i;
                w[i] = __builtin_fmaf(-s.beta[m], w[i], s.a[m * DP + tid]);
                s.a[m * DP + tid] = w[i];
                const float *Ai = s.A + m * AP + 16 * t;
#pragma unroll
                for (int i2 = i + 1; i2 < 16; i2++) w[i2] = __builtin_fmaf(Ai[i2], w[i], w[i2]);
            }
        }
    }
    __syncthreads();

    // o = (E q)^T S_0 + A_qk w, into s.v
#pragma unroll
    for (int t = 0; t < TILES; t++) {
#pragma unroll
        for (int x = 0; x < 4 * (t + 1); x++) {
            const int n = 16 * t + c16, j = 4 * x + kq;
            const float f = j <= n ? s.A[n * AP + j] : 0.0f;
            oq[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(f, s.a[j * DP + 16 * wv + c16], oq[t], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s.v[(16 * t + 4 * kq + i) * DP + 16 * wv + c16] = oq[t][i];
    }
    __syncthreads();

    // K4, a node per half-wave
    {
        const int l32 = tid & 31;
        const bool active = l32 * CPL < D;
        const int cl = active ? l32 * CPL : 0;
        for (int n = tid >> 5; n < N; n += NT / 32) {
            float x[CPL], part = 0.0f;
#pragma unroll
            for (int e = 0; e < CPL; e++) {
                x[e] = s.v[n * DP + cl + e];
                part += active ? x[e] * x[e] : 0.0f;
            }
            const float inv = __builtin_amdgcn_rsqf(half_wave_sum(part) / (float)D + a.eps);
            if (!active) continue;
            const size_t at = (row0 + n) * P + (size_t)h * D + cl;
#pragma unroll
            for (int e = 0; e < CPL; e++) {
                const float y = a.o_norm[cl + e] * x[e] * inv * fast_sigmoid(load_any(a.gate, a.g_dt, at + e));
                if (a.y_dt == K3HIP_BF16) reinterpret_cast<uint16_t *>(a.y)[at + e] = f2bf(y);
                else reinterpret_cast<float *>(a.y)[at + e] = y;
            }
        }
    }
}

// S := S of the accepted node, one workgroup per (head, sequence): the path's nodes one after the other
// on a state held in registers (kda_decode_kernel's tile), so S is read once and written once whatever
// the path's length. K1 of up to CK nodes at a time runs in parallel before them. The conv history of
// the head's channels becomes the last K - 1 inputs of history and path.
constexpr int TREE_CK = 16;

template <int D>
__global__ __launch_bounds__(4 * D) void kda_tree_commit_kernel(const TreeArgs a)
{
    constexpr int NT = 4 * D, CPR = D / 4, RPP = NT / CPR, NPASS = D / RPP;
    constexpr int CPL = D >= 32 ? D / 32 : 1;
    __shared__ float s_k[TREE_CK][D], s_v[TREE_CK][D], s_a[TREE_CK][D], s_b[TREE_CK];
    __shared__ f4 s_red[2][RPP][CPR];
    __shared__ int s_par[TREE_MAX], s_node[TREE_MAX], s_n;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int cg = tid % CPR, rs = tid / CPR;
    const int N = tree_count(a.t, b), node = a.accept[b];
    if (node < 0 || node >= N) return;
    const size_t P = (size_t)a.H * D, row0 = (size_t)b * a.t.N;
    float *hist = a.hist + (size_t)b * a.h_stride;
    f4 *Sp = reinterpret_cast<f4 *>(a.S + (size_t)b * a.s_stride + (size_t)h * D * D);
    f4 s[NPASS];
#pragma unroll
    for (int m = 0; m < NPASS; m++) s[m] = Sp[(rs + m * RPP) * CPR + cg];
    if (tid < 64) {
        const int p = lane < N ? tree_parent(a.t, b, lane) : -1;
        const uint64_t m = tree_ancestors(p);
        const uint64_t path = ((uint64_t)__shfl((uint32_t)(m >> 32), node, 64) << 32) | __shfl((uint32_t)m, node, 64);
        s_par[lane] = p;
        if (path >> lane & 1) s_node[__popcll(path & ((1ull << lane) - 1))] = lane;
        if (lane == 0) s_n = __popcll(path);
    }
    __syncthreads();
    const int n = s_n;
    const int l32 = tid & 31;
    const bool active = l32 * CPL < D;
    const int cl = active ? l32 * CPL : 0;
    const size_t c0 = (size_t)h * D + cl;
    for (int i0 = 0; i0 < n; i0 += TREE_CK) {
        const int ni = min(TREE_CK, n - i0);
        for (int task = tid >> 5; task < 3 * ni; task += NT / 32) {
            const int which = task % 3 + 1, i = task / 3, m = s_node[i0 + i];
            float x[CPL];
            if (which < 3) tree_conv<CPL>(x, a, which, m, s_par, row0, P, c0, active, hist);
            else tree_decay<CPL>(x, a, row0 + m, h, P, c0);
            float *dst = (which == 1 ? s_k[i] : which == 2 ? s_v[i] : s_a[i]) + cl;
            if (active)
#pragma unroll
                for (int e = 0; e < CPL; e++) dst[e] = x[e];
        }
        if (tid < ni) s_b[tid] = fast_sigmoid(a.bl[(row0 + s_node[i0 + tid]) * a.H + h]);
        __syncthreads();
        for (int i = 0; i < ni; i++) {
            f4 u = 0.0f;
#pragma unroll
            for (int m = 0; m < NPASS; m++) {
                const int r = rs + m * RPP;
                s[m] = s[m] * s_a[i][r];
                u = u + s_k[i][r] * s[m];
            }
            s_red[i & 1][rs][cg] = u;
            __syncthreads();   // the other half was last read before this barrier's predecessor
            f4 ut = s_red[i & 1][0][cg];
#pragma unroll
            for (int r = 1; r < RPP; r++) ut = ut + s_red[i & 1][r][cg];
            const f4 d = (reinterpret_cast<const f4 *>(s_v[i])[cg] - ut) * s_b[i];
#pragma unroll
            for (int m = 0; m < NPASS; m++) s[m] = s[m] + s_k[i][rs + m * RPP] * d;
        }
        __syncthreads();   // s_k .. s_b are free; the history's last reader is done
    }
#pragma unroll
    for (int m = 0; m < NPASS; m++) Sp[(rs + m * RPP) * CPR + cg] = s[m];
    // history: slot j of the new one is entry n + j of (the old K - 1, then the path's inputs); ascending
    // order, so a slot is read before the one that replaces it is written
    const int K1 = a.K - 1;
    for (int c = tid; c < 3 * D; c += NT) {
        const int which = c / D;
        const size_t ch = (size_t)h * D + c % D;
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
