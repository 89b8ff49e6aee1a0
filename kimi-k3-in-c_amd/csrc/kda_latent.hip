// SPDX-License-Identifier: Apache-2.0
// kda_latent.hip - a paged cache of MLA latents for gfx950: new rows normalised, rotated and written
// to their pages (k3hip_latent_append), and an accepted path's rows moved together
// (k3hip_latent_commit).
//
// A cache row is what kda_mla.hip caches per position, the rmsnorm'd compressed latent (KL wide) and
// the shared rope slot (QR wide), in fp32 or bf16. Slot s of sequence b is row s % page of page
// table[b][s / page]. Node n of a drafted tree takes slot lens[b] + n; its place in the text, which
// the rotation goes by, is lens[b] + (its ancestors), the same for every alternative at one depth.
#include "kda_internal.h"
#include "kda_tree.h"

namespace k3kda {

namespace {

struct AppendArgs {
    TreeSeqs t;
    PagedRows c;
    int KL, QR;
    void *pages;
    int dtype;
    const void *rows;
    int rows_dt;
    long rows_ld;
    const float *norm_w;
    float eps;
    const float *inv_freq;
    int halves;
    int H;
    const void *q;
    int q_dt;
    long q_ld, q_hd;
    void *qo;
    int qo_dt;
    long qo_ld, qo_hd;
};

// V adjacent elements to or from fp32 registers (V = 8 or 4: 16-byte accesses, p aligned to them;
// V = 1 or 2: element by element).
template <int V>
__device__ __forceinline__ void ld(float (&x)[V], const void *p, int dt, size_t i)
{
    if (dt == K3HIP_F32) {
        const float *f = reinterpret_cast<const float *>(p) + i;
        if constexpr (V >= 4) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const f4 v = *reinterpret_cast<const f4 *>(f + e);
                x[e] = v.x; x[e + 1] = v.y; x[e + 2] = v.z; x[e + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) x[e] = f[e];
        }
    } else {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p) + i;
        if constexpr (V >= 4) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const uint2 v = *reinterpret_cast<const uint2 *>(h + e);
                x[e] = __uint_as_float(v.x << 16); x[e + 1] = __uint_as_float(v.x & 0xffff0000u);
                x[e + 2] = __uint_as_float(v.y << 16); x[e + 3] = __uint_as_float(v.y & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) x[e] = bf2f(h[e]);
        }
    }
}

template <int V>
__device__ __forceinline__ void st(const float (&x)[V], void *p, int dt, size_t i)
{
    if (dt == K3HIP_F32) {
        float *f = reinterpret_cast<float *>(p) + i;
        if constexpr (V >= 4) {
#pragma unroll
            for (int e = 0; e < V; e += 4) *reinterpret_cast<f4 *>(f + e) = f4{x[e], x[e + 1], x[e + 2], x[e + 3]};
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) f[e] = x[e];
        }
    } else {
        uint16_t *h = reinterpret_cast<uint16_t *>(p) + i;
        if constexpr (V >= 4) {
#pragma unroll
            for (int e = 0; e < V; e += 4)
                *reinterpret_cast<uint2 *>(h + e) = uint2{(uint32_t)f2bf(x[e]) | ((uint32_t)f2bf(x[e + 1]) << 16),
                                                          (uint32_t)f2bf(x[e + 2]) | ((uint32_t)f2bf(x[e + 3]) << 16)};
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) h[e] = f2bf(x[e]);
        }
    }
}

// Pairs i .. i + U - 1 of one rope slot turned by their angles: pair i is elements (2 i, 2 i + 1), or
// (i, QR / 2 + i) with `halves`. cs: cosine and sine of pair i at cs[i], nullptr: copied.
template <int U>
__device__ __forceinline__ void turn(const void *src, int sdt, size_t s0, void *dst, int ddt, size_t d0, int i, int QR,
                                     bool halves, const f2 *cs)
{
    float a[U], b[U];
    if (halves) {
        ld<U>(a, src, sdt, s0 + i);
        ld<U>(b, src, sdt, s0 + QR / 2 + i);
    } else {
        float x[2 * U];
        ld<2 * U>(x, src, sdt, s0 + 2 * i);
#pragma unroll
        for (int e = 0; e < U; e++) {
            a[e] = x[2 * e];
            b[e] = x[2 * e + 1];
        }
    }
    if (cs) {
#pragma unroll
        for (int e = 0; e < U; e++) {
            const f2 t = cs[i + e];
            const float u = a[e] * t.x - b[e] * t.y, v = a[e] * t.y + b[e] * t.x;
            a[e] = u;
            b[e] = v;
        }
    }
    if (halves) {
        st<U>(a, dst, ddt, d0 + i);
        st<U>(b, dst, ddt, d0 + QR / 2 + i);
    } else {
        float x[2 * U];
#pragma unroll
        for (int e = 0; e < U; e++) {
            x[2 * e] = a[e];
            x[2 * e + 1] = b[e];
        }
        st<2 * U>(x, dst, ddt, d0 + 2 * i);
    }
}

constexpr int AP_NT = 256;
constexpr int AP_MAXR = 256;   // rope width

// One workgroup per row. The cosines and sines of the row's position are made once, in LDS: the angle
// position * inv_freq in double and taken to one turn there (at a position of 130,000 an fp32 product is
// already 0.004 off), then in fp32. Wave 0 takes the latent (its mean of squares in fp32 lanes, then
// across the wave) and the rope slot, all waves the queries' slots. Bound: bytes for prompts (8.7k rows with the
// slots of 64 queries, bf16: 29 us in cache, 40 us among other work, 3.9 TB/s), latency for trees (128 rows: 6.7 us).
// VEC: units of 8 elements.
template <bool VEC>
__global__ __launch_bounds__(AP_NT) void latent_append_kernel(const AppendArgs a)
{
    __shared__ f2 cs[AP_MAXR / 2];
    __shared__ int s_depth;
    const int n = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    if (n >= tree_count(a.t, b)) return;
    const int len = paged_len(a.c, a.t.lens, b);
    const bool turns = a.inv_freq != nullptr;
    if (turns) {
        if (a.t.parents) {
            if (tid < 64) {
                const uint64_t m = tree_ancestors(lane < a.t.N ? tree_parent(a.t, b, lane) : -1);
                if (lane == n) s_depth = __popcll(m) - 1;
            }
            __syncthreads();
        }
        const int depth = a.t.parents ? s_depth : n;
        for (int i = tid; i < a.QR / 2; i += AP_NT) {
            double r = ((double)len + depth) * (double)a.inv_freq[i] * 0.15915494309189535;   // in turns
            r -= rint(r);
            float s, c;
            sincospif((float)(2.0 * r), &s, &c);
            cs[i] = f2{c, s};
        }
        __syncthreads();
    }
    const size_t row = (size_t)b * a.t.N + n;
    const int UP = VEC ? 4 : 1;   // pairs a unit
    const f2 *t = turns ? cs : nullptr;
    if (tid < 64) {
        const long at = paged_row(a.c, b, len + n);
        if (at >= 0) {
            const size_t dst = (size_t)at * (a.KL + a.QR), src = row * a.rows_ld;
            constexpr int V = VEC ? 8 : 1;
            float inv = 1.0f;
            if (a.norm_w) {
                float ss = 0.0f;
                for (int c = lane * V; c < a.KL; c += 64 * V) {
                    float x[V];
                    ld<V>(x, a.rows, a.rows_dt, src + c);
#pragma unroll
                    for (int e = 0; e < V; e++) ss += x[e] * x[e];
                }
#pragma unroll
                for (int m = 32; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, 64);
                inv = 1.0f / sqrtf(ss / (float)a.KL + a.eps);
            }
            for (int c = lane * V; c < a.KL; c += 64 * V) {
                float x[V];
                ld<V>(x, a.rows, a.rows_dt, src + c);
                if (a.norm_w) {
                    float w[V];
                    ld<V>(w, a.norm_w, K3HIP_F32, c);
#pragma unroll
                    for (int e = 0; e < V; e++) x[e] = w[e] * x[e] * inv;
                }
                st<V>(x, a.pages, a.dtype, dst + c);
            }
            for (int i = lane * UP; i < a.QR / 2; i += 64 * UP)
                turn<VEC ? 4 : 1>(a.rows, a.rows_dt, src + a.KL, a.pages, a.dtype, dst + a.KL, i, a.QR, a.halves, t);
        }
    }
    if (a.q) {
        const int per = a.QR / 2 / UP;   // units a head
        for (int u = tid; u < a.H * per; u += AP_NT) {
            const int h = u / per, i = (u - h * per) * UP;
            turn<VEC ? 4 : 1>(a.q, a.q_dt, row * a.q_ld + h * a.q_hd, a.qo, a.qo_dt, row * a.qo_ld + h * a.qo_hd, i, a.QR,
                              a.halves, t);
        }
    }
}

// The accepted path's rows of one sequence to slots len, len + 1, ...: one workgroup, the i-th node of
// the path (its nodes in order of their numbers: a parent stands before its children) to slot len + i.
// A destination may be another node's source, so a workgroup holds what it moves in registers, UM units
// of U a thread, and stores after a barrier; wider paths go in blocks of columns, whose units never
// meet. A row whose source or destination has no page stays. Latency bound (one table
// lookup, one load, one store): 3.9 us for 64 sequences of 16 nodes, 3.4 for one of 64 (4.3 with units of the
// runtime's vector type, which went through scratch memory).
constexpr int CM_NT = 512, CM_UM = 8;
template <typename U>
__global__ __launch_bounds__(CM_NT) void latent_commit_kernel(TreeSeqs t, PagedRows c, U *pages, int units,
                                                              const int *accept, int *lens_out)
{
    __shared__ long s_src[TREE_MAX], s_dst[TREE_MAX];
    __shared__ int s_n, s_path;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    if (tid < 64) {
        const int cnt = tree_count(t, b), len = paged_len(c, t.lens, b), node = accept[b];
        uint64_t path = tree_ancestors(lane < t.N ? tree_parent(t, b, lane) : -1);
        const bool took = node >= 0 && node < cnt;
        const int from = took ? node : 0;
        const uint32_t lo = __shfl((uint32_t)path, from, 64), hi = __shfl((uint32_t)(path >> 32), from, 64);
        path = took ? ((uint64_t)hi << 32) | lo : 0;
        const int place = __popcll(path & ((1ull << lane) - 1));
        long src = -1, dst = -1;
        if ((path >> lane & 1) && place != lane) {
            src = paged_row(c, b, len + lane);
            dst = paged_row(c, b, len + place);
        }
        const bool moves = src >= 0 && dst >= 0;
        const uint64_t mv = __ballot(moves);
        if (moves) {
            const int at = __popcll(mv & ((1ull << lane) - 1));
            s_src[at] = src;
            s_dst[at] = dst;
        }
        if (lane == 0) {
            s_n = __popcll(mv);
            s_path = min(len + __popcll(path), paged_cap(c));
        }
    }
    __syncthreads();
    if (lens_out && tid == 0) lens_out[b] = s_path;
    const int n = s_n;
    if (n == 0) return;
    const int cols = min(units, CM_NT * CM_UM / n);   // >= 64: n <= 63
    for (int c0 = 0; c0 < units; c0 += cols) {
        const int w = min(cols, units - c0);
        U v[CM_UM];
#pragma unroll
        for (int k = 0; k < CM_UM; k++) {
            const int i = tid + CM_NT * k;
            if (i < n * w) v[k] = pages[(size_t)s_src[i / w] * units + c0 + i % w];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < CM_UM; k++) {
            const int i = tid + CM_NT * k;
            if (i < n * w) pages[(size_t)s_dst[i / w] * units + c0 + i % w] = v[k];
        }
    }
}

// rows x H pieces of `width` elements, rows `ld` apart and heads `head` apart (each at least width): no two meet.
// Row i and head j meet where j heads and i rows are less than a width apart.
bool apart(long rows, long H, long ld, long head, long width)
{
    if (rows <= 1 || H <= 1 || (H - 1) * head + width <= ld || (rows - 1) * ld + width <= head) return true;
    for (long j = 1; j < H; j++) {
        const long i = j * head / ld, over = j * head - i * ld;
        if ((i >= 1 && i < rows && over < width) || (i + 1 < rows && ld - over < width)) return false;
    }
    return true;
}

bool act_dtype(int dt) { return dt == K3HIP_F32 || dt == K3HIP_BF16; }

}  // namespace

}  // namespace k3kda

using namespace k3kda;

extern "C" int k3hip_latent_append(int B, int N, int kv_lora, int rope, void *pages, int dtype, int n_pages, int page,
                                   const int *table, int max_pages, const int *lens, const int *counts,
                                   const int *parents, const void *rows, int rows_dtype, long rows_ld,
                                   const float *norm_w, float eps, const float *inv_freq, int rope_style, int H,
                                   const void *q, int q_dtype, long q_ld, long q_head, void *q_out, int q_out_dtype,
                                   long q_out_ld, long q_out_head, void *stream)
{
    clear_error();
    static const char *who = "k3hip_latent_append";
    if (int rc = paged_check(who, B, N, n_pages, page, max_pages, pages, table, lens)) return rc;
    if (kv_lora <= 0 || rope < 0 || rope > AP_MAXR || (rope & 1))
        K3_FAIL(K3HIP_EINVAL, "%s: kv_lora=%d rope=%d (rope even, at most %d)", who, kv_lora, rope, AP_MAXR);
    if (!act_dtype(dtype) || !act_dtype(rows_dtype)) K3_FAIL(K3HIP_EINVAL, "%s: dtypes cache=%d rows=%d", who, dtype, rows_dtype);
    if (rope_style != K3HIP_ROPE_PAIRS && rope_style != K3HIP_ROPE_HALVES)
        K3_FAIL(K3HIP_EINVAL, "%s: rope_style=%d", who, rope_style);
    if (parents && N > TREE_MAX) K3_FAIL(K3HIP_EUNSUPPORTED, "%s: a tree of %d nodes (at most %d)", who, N, TREE_MAX);
    if (B > 65535) K3_FAIL(K3HIP_EINVAL, "%s: B=%d", who, B);
    if (q && (H <= 0 || !q_out || !act_dtype(q_dtype) || !act_dtype(q_out_dtype) || q_ld < 0 || q_out_ld < 0 ||
              q_head < rope || q_out_head < rope || rope == 0 || (long)H * rope > 0x7fffff00L))
        K3_FAIL(K3HIP_EINVAL, "%s: queries H=%d dtypes %d -> %d, head strides %ld -> %ld, rope=%d", who, H, q_dtype,
                q_out_dtype, q_head, q_out_head, rope);
    if (q && (long)B * N > 1 && q_out_ld < rope)
        K3_FAIL(K3HIP_EINVAL, "%s: rows of rotated queries %ld elements apart", who, q_out_ld);
    if (B == 0 || N == 0) return K3HIP_OK;
    if (q && !apart((long)B * N, H, q_out_ld, q_out_head, rope))
        K3_FAIL(K3HIP_EINVAL, "%s: rotated queries overlap: rows %ld, heads %ld elements apart", who, q_out_ld, q_out_head);
    if (q && q == q_out && (q_dtype != q_out_dtype || ((long)B * N > 1 && q_ld != q_out_ld) || (H > 1 && q_head != q_out_head)))
        K3_FAIL(K3HIP_EINVAL, "%s: queries rotated in place: dtypes %d -> %d, strides %ld, %ld -> %ld, %ld", who, q_dtype, q_out_dtype,
                q_ld, q_head, q_out_ld, q_out_head);
    if (!rows || rows_ld < kv_lora + rope) K3_FAIL(K3HIP_EINVAL, "%s: rows NULL or stride %ld", who, rows_ld);
    AppendArgs a{};
    a.t = TreeSeqs{N, lens, counts, parents};
    a.c = PagedRows{table, n_pages, page, max_pages};
    a.KL = kv_lora; a.QR = rope; a.pages = pages; a.dtype = dtype;
    a.rows = rows; a.rows_dt = rows_dtype; a.rows_ld = rows_ld;
    a.norm_w = norm_w; a.eps = eps;
    a.inv_freq = rope ? inv_freq : nullptr;
    a.halves = rope_style == K3HIP_ROPE_HALVES;
    a.H = H; a.q = q; a.q_dt = q_dtype; a.q_ld = q_ld; a.q_hd = q_head;
    a.qo = q_out; a.qo_dt = q_out_dtype; a.qo_ld = q_out_ld; a.qo_hd = q_out_head;
    // units of 8 elements (4 pairs) where every one of them starts on 16 bytes
    bool vec = kv_lora % 8 == 0 && rope % 8 == 0 && rows_ld % 8 == 0 &&
               !(((uintptr_t)pages | (uintptr_t)rows | (uintptr_t)norm_w) & 15);
    if (q)
        vec = vec && q_ld % 8 == 0 && q_head % 8 == 0 && q_out_ld % 8 == 0 && q_out_head % 8 == 0 &&
              !(((uintptr_t)q | (uintptr_t)q_out) & 15);
    const dim3 grid((unsigned)N, (unsigned)B);
    if (vec) hipLaunchKernelGGL((latent_append_kernel<true>), grid, dim3(AP_NT), 0, as_stream(stream), a);
    else hipLaunchKernelGGL((latent_append_kernel<false>), grid, dim3(AP_NT), 0, as_stream(stream), a);
    K3_LAUNCHED();
    return K3HIP_OK;
}

extern "C" int k3hip_latent_commit(int B, int N, int width, void *pages, int dtype, int n_pages, int page,
                                   const int *table, int max_pages, const int *lens, const int *counts,
                                   const int *parents, const int *accept, int *lens_out, void *stream)
{
    clear_error();
    static const char *who = "k3hip_latent_commit";
    if (int rc = paged_check(who, B, N, n_pages, page, max_pages, pages, table, lens)) return rc;
    if (width <= 0 || !act_dtype(dtype)) K3_FAIL(K3HIP_EINVAL, "%s: width=%d dtype=%d", who, width, dtype);
    if (N > TREE_MAX) K3_FAIL(K3HIP_EUNSUPPORTED, "%s: a tree of %d nodes (at most %d)", who, N, TREE_MAX);
    if (B == 0) return K3HIP_OK;
    if (!accept) K3_FAIL(K3HIP_EINVAL, "%s: NULL accept", who);
    const size_t bytes = (size_t)width * (dtype == K3HIP_F32 ? 4 : 2);
    const TreeSeqs t{N, lens, counts, parents};
    const PagedRows c{table, n_pages, page, max_pages};
#define K3_CM(U) hipLaunchKernelGGL((latent_commit_kernel<U>), dim3(B), dim3(CM_NT), 0, as_stream(stream), t, c, \
                                    reinterpret_cast<U *>(pages), (int)(bytes / sizeof(U)), accept, lens_out)
    if (bytes % 16 == 0 && !((uintptr_t)pages & 15)) K3_CM(f4);
    else if (dtype == K3HIP_F32) K3_CM(uint32_t);
    else K3_CM(uint16_t);
#undef K3_CM
    K3_LAUNCHED();
    return K3HIP_OK;
}
