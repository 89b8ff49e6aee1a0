// SPDX-License-Identifier: Apache-2.0
// kda_tree_attn.hip - attention of drafted token trees over a paged cache of MLA latents, in one pass
// over the cache, for gfx950 (k3hip_mla_tree_attention).
//
// Query row (n, h) of sequence b, in absorbed form (qcat = [W_UK_h^T q_nope, q_rope], CW wide), sees the
// lens[b] committed rows c_t of the cache and the rows of node n and its ancestors:
//   p_t = softmax_t(scale qcat . c_t),   o = sum_t p_t c_t[0 .. KL).
// Every head of every node reads the same rows, so a sequence is one product of (nodes x heads) rows with
// its cache: bytes bind for one node, the matrix cores from a few nodes on.
//
//  * A workgroup owns a tile of query rows and a range of steps of 32 positions, which it walks once; all
//    sequences' steps stand on one axis that is cut into ranges, one for as many workgroups as the largest
//    sequence has row tiles (find_slot). A range that ends inside a sequence leaves unnormalised sums with (M, l); a
//    second launch merges them in order, so results do not depend on timing.
//  * Scores^T (positions x query rows), the softmax in base 2 and o^T (latent channels x query rows) += latents^T . p.
//    With the query row in the column, a softmax row is a lane: its max, its sum, its rescale and its mask are
//    per-lane values, and p goes from the score product's output layout into the second product's operand
//    without leaving the lane.
//  * The 16 rows of a block stand in the score product in the order 4 (m % 4) + m / 4, so that the four
//    positions a lane quarter ends up with are four rows apart, which is what the transposed reads of the second
//    product (ds_read_b64_tr_b16) hand out. A step is staged as column groups [32 rows][8 units of 16 bytes] with
//    unit u of row r at u ^ ((r / 2) & 6): free of bank conflicts for these and for the 16-byte reads of the
//    score product (of the 64 lanes, 0-3, 12-15, 20-27 go together, and so on).
//  * The reference max of a row moves only when a score passes it by TA_LAZY, so sums are rescaled rarely.
//
// What a row does not see cannot reach it: masked scores are selected away, and a node's row that holds an
// infinity or a NaN is staged as zeros and noted; the query rows that see it become NaN.
#include <math.h>

#include <algorithm>

#include "kda_internal.h"
#include "kda_tree.h"

namespace k3kda {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef s16x4 __attribute__((address_space(3))) *lds_s16x4_ptr;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void glb_void;
typedef __attribute__((address_space(1))) const char glb_cchar;
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) const char lds_cchar;

constexpr int TA_NT = 256;
constexpr int TA_KL = 512, TA_CW = 576;        // widest latent and cache row
constexpr float TA_LOG2E = 1.4426950408889634f, TA_LN2 = 0.6931471805599453f;
constexpr float TA_LAZY = 8.0f;                // log2 of the largest weight before a rescale

// What rows without a page and channels past CW are staged from: eight rows of bf16.
__device__ const uint4 ta_zeros[8 * TA_CW * 2 / 16] = {};

struct AttnArgs {
    TreeSeqs t;
    PagedRows c;
    int H, CW, KL;
    const void *pages, *q;
    void *o;
    int o_dt;
    float *lse;
    float scale2;     // scale log2(e)
    int B;
    uint32_t page_bytes;
    int tcol, trow;        // a step in table columns and rows
    float *po, *pm, *pl;   // parts, two a workgroup [rows of a tile] ( x KL): their sums, M and l
    float *pr;             // fp32 caches: what l is taken against (bf16: M)
    int4 *plan;            // [B] first and last slot, workgroups a slot
};

// The 16x16x32 MFMAs of the bf16 kernel. With 32 query rows a wave the second product's 256 accumulators fill
// the accumulation registers: with the builtin the compiler moves them between the register files and
// spills hundreds (with 16 rows it moves a hundred a step), so the instruction is issued by itself, acc tied to its
// registers, everything else in ordinary ones. The compiler then knows no MFMA; wait() stands where it would
// have put wait states.
__device__ __forceinline__ void mfma_acc(const bf16x8 &a, const bf16x8 &b, f32x4 &c)
{
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

// In ordinary registers; both operands come from memory (of a vector instruction's result it would have to wait).
__device__ __forceinline__ void mfma_vec(const bf16x8 &a, const bf16x8 &b, f32x4 &c, bool first)
{
    if (first) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
    else asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}

// c += column sums of b; b, c and the ones may have been written just before, b is ready for others after it.
__device__ __forceinline__ void mfma_sum(bf16x8 &b, f32x4 &c)
{
    const bf16x8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
    asm volatile("s_nop 3\n\tv_mfma_f32_16x16x32_bf16 %0, %2, %1, %0" : "+v"(c), "+v"(b) : "v"(ones));
}

// Ten wait states, between MFMAs and other instructions on their results (eight are needed for this one) or
// between other instructions' results and MFMAs on them; nothing is scheduled across.
__device__ __forceinline__ void wait()
{
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 9");
    __builtin_amdgcn_sched_barrier(0);
}

// c *= m, a register at a time through one ordinary register (left to the compiler, all of them are brought
// over at once and spill).
__device__ __forceinline__ void acc_scale(f32x4 &c, float m)
{
    float t;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        float v = c[e];
        asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
                     : "+a"(v), "=&v"(t) : "v"(m));
        c[e] = v;
    }
}

// Eight lanes a row that agree: a bit a row.
__device__ __forceinline__ uint32_t gather_rows(uint64_t ballot)
{
    return (uint32_t)(((ballot & 0x0101010101010101ull) * 0x0102040810204080ull) >> 56);
}

// Sixteen lanes a row that agree: a bit a row.
__device__ __forceinline__ uint32_t gather_rows16(uint64_t ballot)
{
    return (uint32_t)(ballot & 1) | (uint32_t)(ballot >> 15 & 2) | (uint32_t)(ballot >> 30 & 4) | (uint32_t)(ballot >> 45 & 8);
}

// The larger of x and another lane's, by a DPP control (a NaN is passed over).
template <int C>
__device__ __forceinline__ float dpp_max(float x)
{
    return fmaxf(x, __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), C, 0xf, 0xf, true)));
}

// The largest of m and the magnitudes of x and y (NaNs are passed over), two values an instruction: left to
// the compiler, values from memory are each made canonical first.
__device__ __forceinline__ float max_abs(float m, const f4 &x, const f4 &y)
{
    asm("v_max3_f32 %0, %0, |%1|, |%2|\n\tv_max3_f32 %0, %0, |%3|, |%4|\n\tv_max3_f32 %0, %0, |%5|, |%6|\n\tv_max3_f32 %0, %0, |%7|, |%8|"
        : "+v"(m) : "v"(x.x), "v"(x.y), "v"(x.z), "v"(x.w), "v"(y.x), "v"(y.y), "v"(y.z), "v"(y.w));
    return m;
}

// Either of two bf16 is an infinity or a NaN.
__device__ __forceinline__ bool not_finite16(uint32_t w)
{
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// Four fp32 to bf16, to nearest even.
__device__ __forceinline__ uint2 pack4(const f32x4 &v)
{
    const bf16x2 x = __builtin_convertvector(f2{v[0], v[1]}, bf16x2), y = __builtin_convertvector(f2{v[2], v[3]}, bf16x2);
    return uint2{__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y)};
}

// Which workgroup takes what. All sequences' steps stand on one axis, cut into slots; a slot takes the n
// workgroups that the most row tiles of a sequence need, one each, so the workgroups of a slot walk the same
// positions (and stand on one XCD, where they share its L2), and sequences of different lengths cost no
// one a wait. A slot that ends inside a sequence leaves that sequence's sums as a part, merged after.
//
// The slots end where sequences end, each of at most L steps, if that takes no more slots than there are and
// L is at most `over` steps over the average: a slot that goes on into a second sequence reads its queries and fills its
// pipeline anew, and leaves two parts. Otherwise the axis is cut into equal slots. (Equal slots, and this, bf16: 16
// sequences of one token over up to 1024 positions 37.5 and 31.5 us, of 8 tokens 66 and 52, 64 of one over up to
// 8192 118 and 113; fp32: 4 of 8 tokens over up to 2000 70 and 58. With a step of fp32 at 3.7 us, four more than
// the average cost more than they save: 7 of 13 tokens 144 and 152. Both values of `over` come from these sizes.)
// Slots that end where sequences end are worked out a sequence a lane, so for up to 64 sequences: one more and
// the slots are equal (one token each over up to 2048 positions: 64 sequences 43 us, 65 50, 96 61). Two costs stay: there are
// as many slots as workgroups allow whatever a part costs to write and merge (one sequence of 4000 positions is 125
// slots of a step, 27 us), and every slot takes as many workgroups as the largest sequence has row tiles, so one tree
// of 64 nodes among single tokens leaves 31 of 32 workgroups of the others' slots without work.
constexpr int TB_OVER = 6, TS_OVER = 2;
struct Slots {
    int n;          // workgroups a slot
    int from, to;   // the slot's steps on the axis
};

// Sequence b's row tiles (of `rows` rows) and steps (of `tp` positions).
__device__ __forceinline__ void seq_size(const AttnArgs &a, int b, int rows, int tp, int &nrt, int &steps)
{
    const int cnt = tree_count(a.t, b);
    nrt = (cnt * a.H + rows - 1) / rows;
    steps = cnt ? (paged_len(a.c, a.t.lens, b) + cnt + tp - 1) / tp : 0;
}

// Workgroup id's slot, and the sequence b that it begins in, with the step of the axis that
// sequence begins at; every wave works it out for itself, a sequence a lane. Workgroup 0 writes down for the
// merge which slots each sequence begins and ends in.
__device__ __forceinline__ bool find_slot(const AttnArgs &a, int rows, int tp, int over, int id, int most, Slots &s, int &b, int &begin)
{
    const int lane = threadIdx.x & 63;
    int n = 0, steps0 = 0, T = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        int nrt = 0, steps = 0;
        if (b0 + lane < a.B) seq_size(a, b0 + lane, rows, tp, nrt, steps);
        n = max(n, nrt);
        T += steps;
        if (b0 == 0) steps0 = steps;
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        n = max(n, __shfl_xor(n, m, 64));
        T += __shfl_xor(T, m, 64);
    }
    n = __builtin_amdgcn_readfirstlane(n);
    if (n == 0) return false;
    s.n = n;
    T = __builtin_amdgcn_readfirstlane(T);   // the host checks that two of them fit an int
    int count = min(max(1, most / n), T), L = 0;   // slots; their most steps, 0: equal slots
    if (a.B > 1 && a.B <= 64 && count < 0x8000) {
        const int avg = (T + count - 1) / count;
        const int l[4] = {avg, avg + 1, avg + over / 2, avg + over};
        uint32_t sum[2];   // of the slots that each needs: at most T / l + 64, two a register
#pragma unroll
        for (int i = 0; i < 2; i++) {
            sum[i] = (uint32_t)((steps0 + l[2 * i] - 1) / l[2 * i]) | (uint32_t)((steps0 + l[2 * i + 1] - 1) / l[2 * i + 1]) << 16;
#pragma unroll
            for (int m = 32; m >= 1; m >>= 1) sum[i] += (uint32_t)__shfl_xor((int)sum[i], m, 64);
        }
#pragma unroll
        for (int i = 3; i >= 0; i--) L = (int)(sum[i >> 1] >> (16 * (i & 1)) & 0xffff) <= count ? l[i] : L;
        L = __builtin_amdgcn_readfirstlane(L);
    }
    const int k = id / n;
    if (k >= count) return false;
    s.from = (int)((uint64_t)T * (uint32_t)k / (uint32_t)count);
    s.to = (int)((uint64_t)T * (uint32_t)(k + 1) / (uint32_t)count);
    auto slot_of = [&](int step) { return (int)(((uint64_t)(step + 1) * (uint32_t)count - 1) / (uint32_t)T); };
    int base = 0, base_slot = 0;   // steps and slots of the sequences before
    bool found = false;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        int nrt = 0, steps = steps0;
        if (b0 > 0) {
            steps = 0;
            if (b0 + lane < a.B) seq_size(a, b0 + lane, rows, tp, nrt, steps);
        }
        const int mine = L ? (steps + L - 1) / L : 0;
        int end = steps, end_slot = mine;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int x = __shfl_up(end, m, 64), y = __shfl_up(end_slot, m, 64);
            if (lane >= m) {
                end += x;
                end_slot += y;
            }
        }
        const int first = base + end - steps, first_slot = base_slot + end_slot - mine;
        if (id == 0 && threadIdx.x < 64 && b0 + lane < a.B && steps)
            a.plan[b0 + lane] = L ? int4{first_slot, first_slot + mine - 1, n, 0} : int4{slot_of(first), slot_of(first + steps - 1), n, 0};
        const uint64_t in = L ? __ballot(k >= first_slot && k < first_slot + mine) : __ballot(s.from >= first && s.from < first + steps);
        if (in && !found) {
            const int at = __builtin_ctzll(in);
            b = b0 + at;
            begin = __builtin_amdgcn_readlane(first, at);
            if (L) {
                const int all = __builtin_amdgcn_readlane(steps, at), of = __builtin_amdgcn_readlane(mine, at);
                const int place = k - __builtin_amdgcn_readlane(first_slot, at);
                s.from = begin + (int)((uint64_t)all * (uint32_t)place / (uint32_t)of);
                s.to = begin + (int)((uint64_t)all * (uint32_t)(place + 1) / (uint32_t)of);
            }
            found = true;
            if (id != 0) break;
        }
        base += __builtin_amdgcn_readlane(end, 63);
        base_slot += __builtin_amdgcn_readlane(end_slot, 63);
    }
    return found;   // with L there can be slots to spare
}

// x, worked out anew from here on: what the compiler would else keep in registers over the whole loop.
__device__ __forceinline__ int opaque(int x)
{
    asm volatile("" : "+v"(x));
    return x;
}

// The larger of x and the values of lanes l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float quarter_max(float x)
{
    const auto u = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(u[0]), __uint_as_float(u[1]));
    const auto v = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
}

// The largest score M that a part is merged by, l its sum of weights. Maxima pass over NaNs, so a part that
// saw a NaN can have any M, -inf if it saw nothing else: it gets +inf, which makes its weight in the merge,
// 2^(inf - inf), and with it the row NaN whatever the other parts hold.
__device__ __forceinline__ float part_max(float M, float l) { return l != l ? INFINITY : M; }

// bf16 caches. A step is 32 positions, staged as nine column groups [32 rows][8 units of 16 bytes] so that one
// load of 64 lanes fills 8 rows of a group and a lane's row, unit and swizzle are the same in all of
// them: one row address a lane and step, the groups by immediate offset. Four buffers: while step s is
// summed and s + 1 scored, s + 2 and s + 3 are on their way.
//
// One wave a SIMD has to keep its matrix pipe busy by itself, so the steps overlap: the products of step
// s + 1's scores are followed by the products of step s's sum with step s + 1's softmax spread between
// them, two or three vector instructions to a product; the barrier of a step stands before the sum's last
// eight products, behind which the next scores' first fragments arrive.
//
// Measured: 4 sequences x 64 nodes x 64 heads over up to 32,768 positions 798 us, 1.24 PFLOP/s (a large library product
// reaches 1.36), bound by the matrix cores; 64 tokens over up to 8192 positions 113 us, of which the loop 76 (6 TB/s of
// cache), first loads 9, 33 MB of parts written and merged most of the rest. The form of 128 rows spills 52 registers, none
// of them in the loop.
constexpr int TB_TP = 32, TB_GRP = TB_TP * 128, TB_BUF = 9 * TB_GRP, TB_NB = 4;
constexpr int TB_LDS = TB_NB * TB_BUF + 64 + TREE_MAX * 8;
static_assert(TB_LDS <= 160 * 1024, "LDS");

template <bool FAST, int NR>
__global__ __launch_bounds__(TA_NT) __attribute__((amdgpu_waves_per_eu(1, 1))) void tree_attn16_kernel(const AttnArgs a)
{
    constexpr int ROWS = 64 * NR, DT = TA_KL / 16, KS = TA_CW / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    uint8_t *s_ok = reinterpret_cast<uint8_t *>(smem + TB_NB * TB_BUF);   // [buffer][wave] a bit a row; [16 + wave]: not finite
    uint64_t *s_anc = reinterpret_cast<uint64_t *>(smem + TB_NB * TB_BUF + 64);   // [node] its ancestors

    const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, kq = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int per = gridDim.x / 8, id = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);   // the grid is a multiple of 8
    const int H = a.H, CW = FAST ? TA_CW : a.CW, KL = a.KL;
    Slots sl;
    int seq = 0, begin = 0;
    if (!find_slot(a, ROWS, TB_TP, TB_OVER, id, gridDim.x, sl, seq, begin)) return;
    const int rt = id % sl.n;   // its row tile
    const int to = sl.to;
    int from = sl.from;
    for (int b = seq; from < to; b++) {
        const int cnt = tree_count(a.t, b), rows = cnt * H, r0 = rt * ROWS;
        const int len = paged_len(a.c, a.t.lens, b), end = len + cnt;
        const int nstep = cnt ? (end + TB_TP - 1) / TB_TP : 0;
        const int s0 = from - begin, s1 = min(nstep, to - begin);
        const bool split = s0 > 0 || s1 < nstep;
        begin += nstep;
        from = min(begin, to);
        if (s0 >= s1 || r0 >= rows) continue;
        __syncthreads();   // the staged steps of the sequence before

        const int par = tid < 64 && lane < cnt ? tree_parent(a.t, b, lane) : -1;
        // this lane's query rows: column c16 of each of the wave's NR row tiles
        auto row_of = [&](int r) __attribute__((always_inline)) { return r0 + 16 * (NR * wv + r) + (opaque(tid) & 15); };

        // staging: wave wv brings rows 8 wv .. + 7 of a step
        const int lrow = lane >> 3, prow = 8 * wv + lrow, lu = (lane & 7) ^ ((prow >> 1) & 6);
        // The page number `pgn` (-1: none) and row in it of the step loaded next; (ncol, nrow) the table column and
        // row of the one after it, which end at (ecol, erow). A step is tcol columns, trow rows. FAST: of the
        // wave's first row, its eight lie in one page; else of each lane's.
        const int stop = min(end, s1 * TB_TP);   // what lies behind is not brought in
        const int ecol = min(stop / a.c.page, a.c.max_pages), erow = ecol < a.c.max_pages ? stop - ecol * a.c.page : 0;
        const int frow = s0 * TB_TP + (FAST ? 8 * wv : prow);
        int pgn = -1, pgo = 0, ncol = frow / a.c.page, nrow = frow - ncol * a.c.page;
        const int *table = a.c.table + (size_t)b * a.c.max_pages;
        auto find_rows = [&]() __attribute__((always_inline)) {   // no branch: it stands between products
            const bool in = (ncol < ecol) | ((ncol == ecol) & (nrow < erow));
            int at = in ? ncol : 0;
            if constexpr (FAST) asm volatile("" : "+v"(at));   // a vector load: a scalar one shares the counter of the LDS reads
            const int n = table[at];
            pgn = in ? n : -1;
            pgo = nrow;
            nrow += a.trow;
            ncol += a.tcol + (nrow >= a.c.page);
            nrow -= nrow >= a.c.page ? a.c.page : 0;
        };
        // Loads of a step into LDS. FAST: buffer loads from the page's start (of zeros, where there is none; rows
        // behind the last node are zeroed where they are used). The others go by global loads, a lane's row where
        // it is, which the compiler takes for LDS accesses too: it then waits for all LDS reads after each.
        const int fast_off = lrow * (TA_CW * 2) + 16 * lu;
        int ldo = 0, ldn = 0;
        const char *ldp = nullptr;
        auto load_row = [&](int buf) __attribute__((always_inline)) {
            uint32_t okb;
            if constexpr (FAST) {
                const int page = __builtin_amdgcn_readfirstlane(pgn);
                const bool ok = page >= 0 && page < a.c.n_pages;
                const char *p = reinterpret_cast<const char *>(a.pages) + (uint64_t)(uint32_t)page * a.page_bytes;
                ldp = ok ? p : reinterpret_cast<const char *>(ta_zeros);
                ldn = ok ? (int)a.page_bytes : 8 * TA_CW * 2;
                ldo = ok ? pgo * (TA_CW * 2) : 0;
                okb = ok ? 0xff : 0;
            } else {
                const bool ok = pgn >= 0 && pgn < a.c.n_pages;
                const char *p = reinterpret_cast<const char *>(a.pages) + (uint64_t)(uint32_t)pgn * a.page_bytes + (uint32_t)pgo * (uint32_t)(CW * 2);
                ldp = (ok ? p : reinterpret_cast<const char *>(ta_zeros)) + 16 * lu;
                okb = gather_rows(__ballot(ok));
            }
            s_ok[4 * buf + wv] = (uint8_t)okb;   // every lane the same
        };
        auto load_group = [&](lds_char *dst, int g) __attribute__((always_inline)) {
            lds_void *to = (lds_void *)(dst + TB_GRP * g + 1024 * wv);
            if constexpr (FAST) {
                __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void *)ldp, (short)0, ldn, 0x00020000), to, 16, fast_off, ldo + 128 * g, 0, 0);
            } else {
                const char *src = ldp + 128 * g;
                if (8 * g + lu >= CW / 8) src = reinterpret_cast<const char *>(ta_zeros);
                __builtin_amdgcn_global_load_lds((glb_void *)src, to, 16, 0, 0);
            }
        };
        auto load_step = [&](lds_char *dst, int buf) __attribute__((always_inline)) {
            load_row(buf);
#pragma unroll
            for (int g = 0; g < 9; g++) load_group(dst, g);
        };
        auto buf_of = [](int s) { return s & (TB_NB - 1); };
        lds_char *lds = (lds_char *)smem;

        // steps s0 .. s0 + 2 on their way, the page of s0 + 3 looked up; all lookups first
        const int sm = min(s1, max(s0, len / TB_TP));   // whole steps of committed positions end here
        {
            int n[4], o[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                find_rows();
                n[i] = pgn;
                o[i] = pgo;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                pgn = n[i];
                pgo = o[i];
                if (i < 3) load_step(lds + buf_of(s0 + i) * TB_BUF, buf_of(s0 + i));
            }
        }
        // Queries; rows behind the last one read the first, their sums are not written.
        bf16x8 qb[KS][NR];
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const int row = row_of(r);
            glb_cchar *src = (glb_cchar *)a.q + (((size_t)b * a.t.N * H + (row < rows ? row : 0)) * CW + 8 * kq) * 2;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                glb_cchar *at = src + 64 * ks;
                if (!FAST && 4 * ks + kq >= CW / 8) at = (glb_cchar *)ta_zeros;
                qb[ks][r] = *(const __attribute__((address_space(1))) bf16x8 *)at;
            }
        }
        f32x4 acc[DT][NR], lacc[NR];
        float M[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) {
            M[r] = -INFINITY;
            lacc[r] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; d++) {
                acc[d][r] = 0.0f;
                asm volatile("" : "+a"(acc[d][r]));   // there from here on, not constants
            }
        }
        wait();
        if (tid < 64) s_anc[lane] = tree_ancestors(par);
        // LDS addresses in a block of 16 rows. Score product: row pi, units 4 (ks & 1) + kq of group ks / 2.
        // Second product: rows 4 ((lane / 4) % 4) + kq, units 2 (d % 4) + (lane / 2) % 2 of group d / 4. Unit u
        // of row r stands at u ^ ((r / 2) & 6), so the other units are the first ones with a bit or two turned. The
        // fragments go in an order that changes the unit seldom, and each address is worked out when it does.
        const int pi = 4 * (c16 & 3) + (c16 >> 2), vr = 4 * ((lane >> 2) & 3) + kq;
        const int ka = 128 * pi + 16 * (kq ^ ((pi >> 1) & 6));
        const int va = 128 * vr + 16 * (((lane >> 1) & 1) ^ ((vr >> 1) & 6)) + 8 * (lane & 1);

        // fragments read ahead, and score fragments of a step (fragment 2 ks + block)
        constexpr int AH = 8, NF = 2 * KS;
        // fragment f of the scores: block f % 2 of K-step ks_of(f); of the sum: latent tile d_of(i)
        auto ks_of = [](int f) { return f < KS ? 2 * (f >> 1) : 2 * ((f - KS) >> 1) + 1; };
        auto d_of = [](int i) { return 4 * (i & 7) + (i >> 3); };
        static_assert(KS % 2 == 0 && DT == 32, "fragment orders");
        int kat = 0, vat = 0;
        auto kread = [&](lds_cchar *buf, int f) __attribute__((always_inline)) {
            if (f == 0 || f == KS) kat = opaque(ka) ^ (f == KS ? 64 : 0);
            return *(const __attribute__((address_space(3))) bf16x8 *)(buf + kat + TB_GRP * (ks_of(f) >> 1) + 2048 * (f & 1));
        };
        auto vread = [&](lds_cchar *buf, int i) __attribute__((always_inline)) {
            if (i % 8 == 0) vat = opaque(va) ^ (4 * i);
            lds_cchar *at = buf + vat + TB_GRP * (d_of(i) >> 2);
            const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)at);
            const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(at + 2048));
            const uint2 y0 = __builtin_bit_cast(uint2, x0), y1 = __builtin_bit_cast(uint2, x1);
            return __builtin_bit_cast(bf16x8, uint4{y0.x, y0.y, y1.x, y1.y});
        };
        // Scores of a step, its first AH fragments already read; the last AH products read the first fragments of
        // the sum from `sum`. between(f): work that goes between the products.
        auto scores = [&](lds_cchar *buf, lds_cchar *sum, bf16x8 (&kf)[AH], bf16x8 (&vf)[AH], f32x4 (&S)[2][NR], auto between)
                          __attribute__((always_inline)) {
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const bf16x8 x = kf[f % AH];
#pragma unroll
                for (int r = 0; r < NR; r++) mfma_vec(x, qb[ks_of(f)][r], S[f & 1][r], f < 2);
                if (f + AH < NF) kf[f % AH] = kread(buf, f + AH);
                else vf[f + AH - NF] = vread(sum, f + AH - NF);
                between(f);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto nothing = [](int) __attribute__((always_inline)) {};
        // The sum of a step, its first AH fragments already read; between(d) before the next fragment but AH is read.
        auto values = [&](lds_cchar *buf, bf16x8 (&vf)[AH], const bf16x8 (&pf)[NR], auto between) __attribute__((always_inline)) {
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const bf16x8 v = vf[d % AH];
#pragma unroll
                for (int r = 0; r < NR; r++) mfma_acc(v, pf[r], acc[d_of(d)][r]);
                if (d + AH < DT) vf[d % AH] = vread(buf, d + AH);
                between(d);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // the softmax of a step in 28 pieces: S to weights in the second product's operand, M and the factor al
        // that the sums before it are to be scaled by
        struct Soft {
            float mt[NR], ref[NR], al[NR];
            bool moved;
        };
        auto soft_piece = [&](int i, f32x4 (&S)[2][NR], Soft &x, bf16x8 (&pf)[NR]) __attribute__((always_inline)) {
            if (i < NR) {
                const f32x4 u = S[0][i], v = S[1][i];
                x.mt[i] = fmaxf(fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3])), fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
            } else if (i == 2) {
#pragma unroll
                for (int r = 0; r < NR; r++) x.mt[r] = quarter_max(x.mt[r]) * a.scale2;
            } else if (i == 3) {
                x.moved = false;
#pragma unroll
                for (int r = 0; r < NR; r++) {
                    const bool up = x.mt[r] > M[r] + TA_LAZY;
                    const float mn = up ? x.mt[r] : M[r];
                    x.al[r] = up ? __builtin_amdgcn_exp2f(M[r] - mn) : 1.0f;
                    x.moved = x.moved || up;
                    M[r] = mn;
                    x.ref[r] = mn == -INFINITY ? 0.0f : mn;
                }
            } else if (i >= 4 && i < 4 + 8 * NR) {
                const int k = i - 4, r = k >> 3, e = k & 7;
                float p = __builtin_amdgcn_exp2f(__builtin_fmaf(S[e >> 2][r][e & 3], a.scale2, -x.ref[r]));
                asm volatile("" : "+v"(p));   // here, not where it is used
                S[e >> 2][r][e & 3] = p;
            } else if (i >= 20 && i < 20 + 4 * NR) {
                const int k = i - 20, r = k >> 2, w = k & 3;
                const bf16x2 y = __builtin_convertvector(f2{S[w >> 1][r][2 * (w & 1)], S[w >> 1][r][2 * (w & 1) + 1]}, bf16x2);
                pf[r][2 * w] = y[0];
                pf[r][2 * w + 1] = y[1];
            }
        };
        auto rescale = [&](const Soft &x) __attribute__((always_inline)) {
            if (!__ballot(x.moved)) return;
            wait();
#pragma unroll
            for (int r = 0; r < NR; r++) lacc[r] *= x.al[r];
#pragma unroll
            for (int r = 0; r < NR; r++)
#pragma unroll
                for (int d = 0; d < DT; d++) acc_scale(acc[d][r], x.al[r]);
            wait();
        };
        auto publish = [](int left) __attribute__((always_inline)) {   // this wave's loads but the last `left`, then every wave's
            if (left) asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        auto pages_of = [&](int s) __attribute__((always_inline)) { return reinterpret_cast<const uint32_t *>(s_ok)[buf_of(s)]; };
        auto mask_pages = [&](uint32_t held, f32x4 (&S)[2][NR]) __attribute__((always_inline)) {
            const uint32_t ok = __builtin_amdgcn_readfirstlane(held);
            if (ok == 0xffffffffu) return;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (!(ok >> (16 * i + 4 * e + kq) & 1))
#pragma unroll
                        for (int r = 0; r < NR; r++) S[i][r][e] = -INFINITY;
        };

        if (s0 < sm) {
            f32x4 S[2][NR];
            bf16x8 kf[AH], vf[AH], pf[NR];
            Soft x;
            publish(9);
            {
                lds_cchar *cur = lds + buf_of(s0) * TB_BUF;
#pragma unroll
                for (int f = 0; f < AH; f++) kf[f] = kread(cur, f);
                scores(cur, cur, kf, vf, S, nothing);
                wait();
                mask_pages(pages_of(s0), S);
#pragma unroll
                for (int i = 0; i < 28; i++) soft_piece(i, S, x, pf);
                cur = lds + buf_of(s0 + 1) * TB_BUF;
#pragma unroll
                for (int f = 0; f < AH; f++) kf[f] = kread(cur, f);
            }
            // the sums are zeros yet: nothing to rescale
            // Step s's sum and step s + 1's scores. The buffers as parameters that do not alias: else the compiler
            // has every transposed read wait for the loads in flight.
            auto step = [&](lds_cchar *__restrict__ cur, lds_cchar *__restrict__ nxt, lds_cchar *__restrict__ nx2,
                            lds_char *__restrict__ fill, int s) __attribute__((always_inline)) {
                uint32_t held = 0;
                scores(nxt, cur, kf, vf, S, [&](int f) __attribute__((always_inline)) {
                    if (f == 6) held = pages_of(s + 1);
                    if (f == 2) load_row(buf_of(s + 3));
                    if (f == 4) find_rows();
                    if (f >= 8 && f < 26 && f % 2 == 0) load_group(fill, (f - 8) / 2);
                });
                bf16x8 pn[NR];
#pragma unroll
                for (int r = 0; r < NR; r++) mfma_sum(pf[r], lacc[r]);   // with its wait states, S is there
                __builtin_amdgcn_sched_barrier(0);
                mask_pages(held, S);
                values(cur, vf, pf, [&](int d) __attribute__((always_inline)) {
                    if (d < 28) soft_piece(d, S, x, pn);
                    if (d == 28) {
                        // every fragment of step s is in registers: its buffer is free behind the barrier
                        publish(9);
#pragma unroll
                        for (int f = 0; f < 4; f++) kf[f] = kread(nx2, f);
                    }
                    if (d > 28) kf[d - 25] = kread(nx2, d - 25);
                    if (d == 31) kf[7] = kread(nx2, 7);
                });
                rescale(x);
#pragma unroll
                for (int r = 0; r < NR; r++) pf[r] = pn[r];
            };
            for (int s = s0; s + 1 < sm; s++)
                step(lds + buf_of(s) * TB_BUF, lds + buf_of(s + 1) * TB_BUF, lds + buf_of(s + 2) * TB_BUF, lds + buf_of(s + 3) * TB_BUF, s);
            wait();
            {
                lds_cchar *cur = lds + buf_of(sm - 1) * TB_BUF;
                publish(0);
                load_step(lds + buf_of(sm + 2) * TB_BUF, buf_of(sm + 2));
#pragma unroll
                for (int d = 0; d < AH; d++) vf[d] = vread(cur, d);
#pragma unroll
                for (int r = 0; r < NR; r++) mfma_sum(pf[r], lacc[r]);
                values(cur, vf, pf, nothing);
                wait();
            }
        }
        // the steps that hold nodes: at most three, on their way by now
        for (int s = sm; s < s1; s++) {
            publish(0);
            const int ln = opaque(tid) & 63, pr = 8 * wv + (ln >> 3), q4 = ln >> 4;
            char *at = smem + buf_of(s) * TB_BUF + 1024 * wv + 16 * ln;
            lds_cchar *cur = lds + buf_of(s) * TB_BUF;
            const uint32_t ok = reinterpret_cast<const uint32_t *>(s_ok)[buf_of(s)];
            const int n0 = len - s * TB_TP;   // place of the first node in the step
            // Zeros in the rows behind the last node, and in rows of nodes that hold an infinity or a NaN, which are
            // noted, so that the query rows that see them become NaN and no others
            bool inf = false;
            if (cnt > 1) {
#pragma unroll
                for (int g = 0; g < 9; g++) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(at + TB_GRP * g);
                    inf = inf || not_finite16(w.x) || not_finite16(w.y) || not_finite16(w.z) || not_finite16(w.w);
                }
            }
            const bool behind = s * TB_TP + pr >= end;
            const uint64_t m = __ballot(inf && pr >= n0);
            const bool mine = (m >> (ln & 56) & 0xff) != 0 && !behind;
            if (mine || behind)
#pragma unroll
                for (int g = 0; g < 9; g++) *reinterpret_cast<uint4 *>(at + TB_GRP * g) = uint4{0, 0, 0, 0};
            s_ok[16 + wv] = (uint8_t)gather_rows(__ballot(mine));
            __syncthreads();
            const uint32_t bad = reinterpret_cast<const uint32_t *>(s_ok)[4];
            f32x4 S[2][NR];
            bf16x8 kf[AH], vf[AH], pf[NR];
            Soft x;
#pragma unroll
            for (int f = 0; f < AH; f++) kf[f] = kread(cur, f);
            scores(cur, cur, kf, vf, S, nothing);
            wait();
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const int row = row_of(r);
                const uint64_t anc = s_anc[row < rows ? row / H : 0];
                uint32_t w = n0 >= 32 ? ~0u : n0 <= 0 ? 0u : (1u << n0) - 1;
                if (n0 >= 0 && n0 < 32) w |= (uint32_t)(anc << n0);
                else if (n0 < 0 && n0 > -64) w |= (uint32_t)(anc >> -n0);
                w &= ok;
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int bit = 16 * i + 4 * e + q4;
                        const float seen = bad >> bit & 1 ? NAN : 0.0f;
                        S[i][r][e] = w >> bit & 1 ? S[i][r][e] + seen : -INFINITY;
                    }
            }
#pragma unroll
            for (int i = 0; i < 28; i++) soft_piece(i, S, x, pf);
            rescale(x);
#pragma unroll
            for (int r = 0; r < NR; r++) mfma_sum(pf[r], lacc[r]);
            values(cur, vf, pf, nothing);
            wait();
        }

#pragma unroll
        for (int r = 0; r < NR; r++) {
            const int row = row_of(r);
            if (row >= rows) continue;
            const float l = lacc[r][0];
            const int q4 = (opaque(tid) & 63) >> 4;
            const size_t orow = (size_t)b * a.t.N * H + row, prow = ((size_t)2 * id + (s0 == 0)) * ROWS + (row - r0);
            if (split) {
                const float m = part_max(M[r], l);
                if (q4 == 0) {
                    a.pm[prow] = m;
                    a.pl[prow] = l;
                }
                if (m == -INFINITY) continue;   // nothing seen: the merge does not read its sums
                float *dst = a.po + prow * KL + 4 * q4;
#pragma unroll
                for (int d = 0; d < DT; d++)
                    if (16 * d + 4 * q4 < KL) *reinterpret_cast<f32x4 *>(dst + 16 * d) = acc[d][r];
            } else {
                if (q4 == 0 && a.lse) a.lse[orow] = l == 0.0f ? -INFINITY : (M[r] + __builtin_amdgcn_logf(l)) * TA_LN2;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                if (a.o_dt == K3HIP_F32) {
                    float *dst = reinterpret_cast<float *>(a.o) + orow * KL + 4 * q4;
#pragma unroll
                    for (int d = 0; d < DT; d++)
                        if (16 * d + 4 * q4 < KL) *reinterpret_cast<f32x4 *>(dst + 16 * d) = acc[d][r] * inv;
                } else {
                    uint16_t *dst = reinterpret_cast<uint16_t *>(a.o) + orow * KL + 4 * q4;
#pragma unroll
                    for (int d = 0; d < DT; d++)
                        if (16 * d + 4 * q4 < KL) *reinterpret_cast<uint2 *>(dst + 16 * d) = pack4(acc[d][r] * inv);
                }
            }
        }
    }
}

// fp32 caches. The products run on the fp16 matrix cores near fp32's accuracy: a row is scaled by a power of
// two that puts its largest value just under 2^15 and split into fp16 hi + 2^-11 lo, 22 bits together (down to
// 2^-29 of the row's largest value; what is left out is under 2^-51 of it), and hi hi + hi lo + lo hi are summed in
// fp32, three matrix instructions where six are needed on bf16 parts and sixteen times the rate of the fp32
// instruction. A cache row's scale 2^k goes with its weight: the reference that the second product's weights are taken
// against is the largest of (score - k), so the scaled weight 2^(score - k - M + TS_UP) is at most 2^(TS_UP + TA_LAZY)
// whatever the rows' sizes. The sum of the weights is that of 2^(score - R) with R the largest score itself: a sum of
// the scaled weights with their 2^k taken back out leaves fp32's range where rows are tiny, and loses the weights of
// rows that are tiny beside others. M and R are whole numbers, so that one weight is the other times 2^-k and
// 2^(R - M + TS_UP), exactly, and the output takes 2^(M - TS_UP - R) back out at the end.
//
// A step is 32 positions, staged as two planes of column groups as in the bf16 kernel, two buffers. Eight
// waves, two a SIMD: waves w and w + 4 own 16 query rows; each scores half of the cache row's channels (so it holds half
// of the query's hi + lo, 72 registers), they add their halves through LDS, both work out the softmax, and each sums half of
// the latent's channels (64 registers). A step has two barriers, behind the halves of the scores and behind the
// sum; a wave keeps 4 rows on their way to registers and converts and stages them, a column group at a time, between the
// products: groups 4 .. 8 beside the scores, where groups 0 .. 3 of the buffer carry the halves, those beside the sum.
// Measured (7 sequences of up to 3001 positions x 13 nodes x 64 heads): 146 us with the merge, 193 TFLOP/s of fp32 work
// (144 before the weights' sum had its own reference), 3.3k of a step's 8.7k cycles matrix instructions and 3.4k LDS
// accesses; what binds is the wait of two waves in step for LDS fragments (registers allow one K-step of look-ahead), the hand-over
// (800 cycles) and the softmax (about 800). 64 sequences of one token over up to 8192 positions: 265 us, 3.5 TB/s of
// cache. All 256 registers are taken and 25 spilled (27 where rows are narrower), one of them (three) in the loop. With
// four waves of whole rows, one a SIMD, 238 us: nothing stood beside their waits, and they spilled in it.
constexpr int TS_BUF = 2 * TB_BUF;
constexpr int TS_NT = 512;
constexpr int TS_LDS = 2 * TS_BUF + 2 * 32 * 8 + 64 + TREE_MAX * 8;
constexpr int TS_UP = 7;          // log2 of the weight of the reference
// The largest scale of a row: R - M + TS_UP is at most TS_KMAX + 1 + TA_LAZY + TS_UP, an exponent of fp32 (and at least
// -116: a scale is at least 2^-114). A row under 2^-96 stays further under 2^15, and its values are whole
// multiples of 2^-145 rather than 22 bits.
constexpr int TS_KMAX = 110;
constexpr float TS_LO = 2048.0f;  // what lo parts are scaled by
static_assert(TS_LDS <= 160 * 1024, "LDS");

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// x = hi + 2^-11 lo
__device__ __forceinline__ void split16(const float (&x)[8], f16x8 &hi, f16x8 &lo)
{
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const f16x2 h = __builtin_convertvector(f2{x[e], x[e + 1]}, f16x2);
        const f16x2 l = __builtin_convertvector(f2{(x[e] - (float)h[0]) * TS_LO, (x[e + 1] - (float)h[1]) * TS_LO}, f16x2);
        hi[e] = h[0];
        hi[e + 1] = h[1];
        lo[e] = l[0];
        lo[e + 1] = l[1];
    }
}

// The same of x times a power of two, a product and its rounding in one instruction. Between two that write halves of a
// register, or one that writes and one that reads it, stands another.
__device__ __forceinline__ void split4(const f4 &x, float scale, uint2 &hi, uint2 &lo)
{
    float t0, t1, t2, t3;
    asm("v_fma_mixlo_f16 %0, %8, %12, 0\n\t"
        "v_fma_mixlo_f16 %1, %10, %12, 0\n\t"
        "v_fma_mixhi_f16 %0, %9, %12, 0\n\t"
        "v_fma_mixhi_f16 %1, %11, %12, 0\n\t"
        "v_fma_mix_f32 %4, %8, %12, -%0 op_sel_hi:[0,0,1]\n\t"
        "v_fma_mix_f32 %6, %10, %12, -%1 op_sel_hi:[0,0,1]\n\t"
        "v_fma_mix_f32 %5, %9, %12, -%0 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mix_f32 %7, %11, %12, -%1 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixlo_f16 %2, %4, %13, 0\n\t"
        "v_fma_mixlo_f16 %3, %6, %13, 0\n\t"
        "v_fma_mixhi_f16 %2, %5, %13, 0\n\t"
        "v_fma_mixhi_f16 %3, %7, %13, 0\n\t"
        "s_nop 0"
        : "=&v"(hi.x), "=&v"(hi.y), "=&v"(lo.x), "=&v"(lo.y), "=&v"(t0), "=&v"(t1), "=&v"(t2), "=&v"(t3)
        : "v"(x.x), "v"(x.y), "v"(x.z), "v"(x.w), "v"(scale), "s"(TS_LO));
}

// 2^(x + add), x a whole number (of a row that has seen nothing, or an infinity: any).
__device__ __forceinline__ float exp2_int(float x, int add) { return __builtin_amdgcn_ldexpf(1.0f, (int)x + add); }

// The power of two that a row whose largest magnitude has these bits is scaled by. Zeros by the largest: they add
// nothing to the second product, and by a smaller one they would make the others' weights small in it (by 1, those of
// rows of 1e-4 some 2^-19, fp16 subnormals).
__device__ __forceinline__ int row_scale(uint32_t most)
{
    return min(14 - ((int)(most >> 23) - 127), TS_KMAX);
}

// Behind it every wave's LDS accesses before it; loads to registers stay on their way.
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <bool FULL>
__global__ __launch_bounds__(TS_NT) __attribute__((amdgpu_waves_per_eu(2, 2))) void tree_attn32_kernel(const AttnArgs a)
{
    constexpr int ROWS = 64, DT = TA_KL / 32, KS = TA_CW / 64;   // a wave's halves
    extern __shared__ __attribute__((aligned(16))) char smem[];
    f2 *s_k = reinterpret_cast<f2 *>(smem + 2 * TS_BUF);                 // [buffer][row] of its scale 2^k: 2^-k, k
    uint8_t *s_ok = reinterpret_cast<uint8_t *>(s_k + 64);               // [buffer][seen, not finite][wave] a bit a row
    uint64_t *s_anc = reinterpret_cast<uint64_t *>(s_ok + 64);           // [node] its ancestors

    const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, kq = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), half = wv >> 2;
    const int per = gridDim.x / 8, id = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    const int H = a.H, CW = FULL ? TA_CW : a.CW, KL = a.KL;
    Slots sl;
    int seq = 0, begin = 0;
    if (!find_slot(a, ROWS, TB_TP, TS_OVER, id, gridDim.x, sl, seq, begin)) return;
    const int rt = id % sl.n;   // its row tile
    const int to = sl.to;
    int from = sl.from;
    for (int b = seq; from < to; b++) {
        const int cnt = tree_count(a.t, b), rows = cnt * H, r0 = rt * ROWS;
        const int len = paged_len(a.c, a.t.lens, b), end = len + cnt;
        const int nstep = cnt ? (end + TB_TP - 1) / TB_TP : 0;
        const int s0 = from - begin, s1 = min(nstep, to - begin);
        const bool split = s0 > 0 || s1 < nstep;
        begin += nstep;
        from = min(begin, to);
        if (s0 >= s1 || r0 >= rows) continue;
        __syncthreads();   // the staged steps of the sequence before

        const int par = tid < 64 && lane < cnt ? tree_parent(a.t, b, lane) : -1;
        const int row = r0 + 16 * (wv & 3) + c16;   // this lane's query row

        // staging: rows 4 wv .. + 3 of a step, channels 4 (lane & 15) .. + 3 of each column group
        const int prow = 4 * wv + kq;
        const int stop = min(end, s1 * TB_TP);   // what lies behind is not brought in
        const int ecol = min(stop / a.c.page, a.c.max_pages), erow = ecol < a.c.max_pages ? stop - ecol * a.c.page : 0;
        int col = (s0 * TB_TP + prow) / a.c.page, prw = s0 * TB_TP + prow - col * a.c.page;   // of the row to load next
        const int *table = a.c.table + (size_t)b * a.c.max_pages;
        auto has_page = [&]() __attribute__((always_inline)) { return (col < ecol) | ((col == ecol) & (prw < erow)); };
        int page = table[has_page() ? col : 0];
        f4 R[9];                       // the row's values in flight
        bool rok = false, nok = false; // that row, and the one that next_row found, have a page
        glb_cchar *src = nullptr;
        auto next_row = [&]() __attribute__((always_inline)) {
            rok = nok;
            nok = has_page() & (page >= 0) & (page < a.c.n_pages);
            const uint64_t at = (uint64_t)(uint32_t)page * a.page_bytes + (uint32_t)prw * (uint32_t)(CW * 4);
            src = (nok ? (glb_cchar *)a.pages + at : (glb_cchar *)ta_zeros) + 16 * c16;
            prw += a.trow;
            col += a.tcol + (prw >= a.c.page);
            prw -= prw >= a.c.page ? a.c.page : 0;
            page = table[has_page() ? col : 0];
        };
        auto load = [&](int g) __attribute__((always_inline)) {
            glb_cchar *at = src + 256 * g;
            if (!FULL && 64 * g + 4 * c16 >= CW) at = (glb_cchar *)ta_zeros;
            R[g] = *(const __attribute__((address_space(1))) f4 *)at;
        };
        // the row's scale, from its largest value
        float scale = 0.0f;
        auto largest = [&](float &m, int i) __attribute__((always_inline)) {   // in three pieces
#pragma unroll
            for (int g = 4 * i; g < min(4 * i + 4, 9); g += 2) m = max_abs(m, R[g], R[min(g + 1, 8)]);
        };
        auto scale_row = [&](int s, float m) __attribute__((always_inline)) {
            const int buf = s & 1;
            asm volatile("s_nop 1" : "+v"(m));   // the compiler does not see that a vector instruction wrote what DPP reads
            m = dpp_max<0x121>(m);   // row_ror 1, 2, 4, 8: over the row's sixteen lanes
            m = dpp_max<0x122>(m);
            m = dpp_max<0x124>(m);
            m = dpp_max<0x128>(m);
            uint32_t bits = 0;
            // a node's row that holds an infinity or a NaN: zeros, and noted, so that the query rows that see
            // it become NaN and no others
            if ((s + 1) * TB_TP > len) {
                bool bad = false;
#pragma unroll
                for (int g = 0; g < 9; g++)
#pragma unroll
                    for (int e = 0; e < 4; e++) bad |= (__float_as_uint(R[g][e]) & 0x7f800000u) == 0x7f800000u;
                bad &= s * TB_TP + prow >= len;
                const uint64_t any = __ballot(bad);
#pragma unroll
                for (int r = 0; r < 4; r++) bits |= any >> (16 * r) & 0xffff ? 1u << r : 0u;
                if (bits >> kq & 1)
#pragma unroll
                    for (int g = 0; g < 9; g++) R[g] = 0.0f;
            }
            const int k = row_scale(__float_as_uint(m));
            scale = __uint_as_float((uint32_t)(127 + k) << 23);
            s_k[32 * buf + 4 * wv + (opaque(tid) >> 4 & 3)] = f2{__uint_as_float((uint32_t)(127 - k) << 23), (float)k};   // sixteen lanes the same
            s_ok[16 * buf + wv] = (uint8_t)gather_rows16(__ballot(rok));
            s_ok[16 * buf + 8 + wv] = (uint8_t)bits;
        };
        // a column group of it to LDS
        auto put = [&](int s, int g, int sa) __attribute__((always_inline)) {
            uint2 hi, lo;
            split4(R[g], scale, hi, lo);
            char *at = smem + (s & 1) * TS_BUF + TB_GRP * g + sa;
            *reinterpret_cast<uint2 *>(at) = hi;
            *reinterpret_cast<uint2 *>(at + TB_BUF) = lo;
        };
        next_row();
#pragma unroll
        for (int g = 0; g < 9; g++) load(g);
        next_row();

        // query fragments, scaled and split alike: channels 32 kstep(ks) + 8 kq .. + 7 of the row
        auto kstep = [&](int ks) __attribute__((always_inline)) { return ks < 8 ? 8 * half + ks : 16 + half; };
        f16x8 qh[KS], ql[KS];
        float qscale;   // of the scores of this half
        {
            glb_cchar *src = (glb_cchar *)a.q + (((size_t)b * a.t.N * H + (row < rows ? row : 0)) * CW + 8 * kq) * 4;
            f4 x[2 * KS];
#pragma unroll
            for (int i = 0; i < 2 * KS; i++) {
                glb_cchar *at = src + 128 * kstep(i >> 1) + 16 * (i & 1);
                if (!FULL && 32 * kstep(i >> 1) + 8 * kq >= CW) at = (glb_cchar *)ta_zeros;
                x[i] = *(const __attribute__((address_space(1))) f4 *)at;
            }
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * KS; i += 2) m = max_abs(m, x[i], x[i + 1]);
            m = quarter_max(m);
            const int k = row_scale(__float_as_uint(m));
            const float sc = __uint_as_float((uint32_t)(127 + k) << 23);
            qscale = ldexpf(a.scale2, -k);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const f4 u = x[2 * ks] * sc, v = x[2 * ks + 1] * sc;
                const float y[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
                split16(y, qh[ks], ql[ks]);
            }
        }

        // LDS places, worked out from the lane anew in every step: staged channels, fragments of the scores'
        // K-steps and of the half's last, of the sum
        auto put_at = [&](int t) __attribute__((always_inline)) {
            const int r = 4 * wv + (t >> 4 & 3), u = t >> 1 & 7;
            return 128 * r + 16 * (u ^ ((r >> 1) & 6)) + 8 * (t & 1);
        };
        auto key_at = [&](int t, int first) __attribute__((always_inline)) {
            const int r = 4 * (t & 3) + (t >> 2 & 3);
            return 128 * r + 16 * (((t >> 4 & 3) + first) ^ ((r >> 1) & 6));
        };
        auto sum_at = [&](int t) __attribute__((always_inline)) {
            const int r = 4 * (t >> 2 & 3) + (t >> 4 & 3);
            return 128 * r + 16 * ((t >> 1 & 1) ^ ((r >> 1) & 6)) + 8 * (t & 1) + 4 * half * TB_GRP;
        };
        auto kread = [&](lds_cchar *buf, int f, int ka, int kb) __attribute__((always_inline)) {   // block f % 2 of K-step f / 2
            lds_cchar *at = f < 16 ? buf + (ka ^ (f & 2 ? 64 : 0)) + 4 * half * TB_GRP + TB_GRP * (f >> 2) : buf + kb + 8 * TB_GRP;
            return *(const __attribute__((address_space(3))) f16x8 *)(at + 2048 * (f & 1));
        };
        auto vread = [&](lds_cchar *buf, int d, int va) __attribute__((always_inline)) {
            lds_cchar *at = buf + (va ^ (32 * (d & 3))) + TB_GRP * (d >> 2);
            const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)at);
            const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(at + 2048));
            const uint2 y0 = __builtin_bit_cast(uint2, x0), y1 = __builtin_bit_cast(uint2, x1);
            return __builtin_bit_cast(f16x8, uint4{y0.x, y0.y, y1.x, y1.y});
        };
        // A wave hands its half of the scores over where its partner will stage rows of the next step: nothing
        // is read there any more, and the partner, which reads them, is the only one to write there next.
        auto half_at = [&](int s, int w, int i, int t) __attribute__((always_inline)) {
            return reinterpret_cast<f4 *>(smem + ((s + 1) & 1) * TS_BUF + TB_GRP * 2 * i + (t >> 5 & 1) * TB_GRP + 512 * w + 16 * (t & 31));
        };
        f32x4 acc[DT];
        float M = -INFINITY, Rf = -INFINITY, lsum = 0.0f;   // references of the sums and of the weights
#pragma unroll
        for (int d = 0; d < DT; d++) acc[d] = 0.0f;
        if (tid < 64) s_anc[lane] = tree_ancestors(par);
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 3; i++) largest(most, i);
        scale_row(s0, most);
#pragma unroll
        for (int g = 0; g < 9; g++) {
            put(s0, g, put_at(tid));
            load(g);
        }
        next_row();
        lds_barrier();

        for (int s = s0; s < s1; s++) {
            lds_cchar *cur = (lds_cchar *)smem + (s & 1) * TS_BUF;
            const int st = opaque(tid), ka = key_at(st, 0), kb = key_at(st, 4 * half), sa = put_at(st);
            constexpr int AK = 2, AV = 2;   // fragment pairs read ahead
            f16x8 kh[AK], kl[AK];
            f32x4 S[2], Sl[2];
#pragma unroll
            for (int i = 0; i < 2; i++) S[i] = Sl[i] = 0.0f;
#pragma unroll
            for (int f = 0; f < AK; f++) {
                kh[f] = kread(cur, f, ka, kb);
                kl[f] = kread(cur + TB_BUF, f, ka, kb);
            }
            most = 0.0f;
#pragma unroll
            for (int f = 0; f < 2 * KS; f += 2) {   // both blocks of a K-step
                f16x8 h[2], l[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    h[i] = kh[(f + i) % AK];
                    l[i] = kl[(f + i) % AK];
                }
#pragma unroll
                for (int i = 0; i < 2; i++) S[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h[i], qh[f >> 1], S[i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 2; i++) Sl[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h[i], ql[f >> 1], Sl[i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 2; i++) Sl[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[i], qh[f >> 1], Sl[i], 0, 0, 0);
                if (f + AK < 2 * KS)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        kh[(f + i) % AK] = kread(cur, f + i + AK, ka, kb);
                        kl[(f + i) % AK] = kread(cur + TB_BUF, f + i + AK, ka, kb);
                    }
                // step s + 1 (past the end: rows of zeros), and the loads of step s + 2
                if (f < 6) largest(most, f / 2);
                if (f == 6) scale_row(s + 1, most);
                if (f >= 8) {
                    put(s + 1, f / 2, sa);
                    load(f / 2);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            const int ht = opaque(tid);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                S[i] = (S[i] + Sl[i] * (1.0f / TS_LO)) * qscale;
                asm volatile("" : "+v"(S[i]));   // rounded here, as its partner gets it: both have to come to the same bits
                *half_at(s, wv ^ 4, i, ht) = f4{S[i][0], S[i][1], S[i][2], S[i][3]};
            }
            const int va = sum_at(ht);
            f16x8 vh[AV], vl[AV];
#pragma unroll
            for (int d = 0; d < AV; d++) {
                vh[d] = vread(cur, d, va);
                vl[d] = vread(cur + TB_BUF, d, va);
            }
            f2 k[8];
            const f2 *ks = s_k + 32 * (s & 1) + (ht >> 4 & 3);
#pragma unroll
            for (int x = 0; x < 8; x++) k[x] = ks[16 * (x >> 2) + 4 * (x & 3)];
            const uint64_t *okw = reinterpret_cast<const uint64_t *>(s_ok) + 2 * (s & 1);
            const uint64_t ok = okw[0], bad = okw[1];
            lds_barrier();
            float y[8];   // scores in base 2
            f4 other[2];
#pragma unroll
            for (int i = 0; i < 2; i++) other[i] = *half_at(s, wv, i, ht);
            // scores with their rows' scales, masks, softmax
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) y[4 * i + e] = (S[i][e] + other[i][e]) * k[4 * i + e].x;
            if (ok != 0x0f0f0f0f0f0f0f0full || (s + 1) * TB_TP > len) {
                const int n0 = len - s * TB_TP;   // place of the first node in the step
                const int q4 = opaque(tid) >> 4 & 3, row = r0 + 16 * (wv & 3) + (opaque(tid) & 15);
                const uint64_t anc = s_anc[row < rows ? row / H : 0];
                uint32_t w = n0 >= 32 ? ~0u : n0 <= 0 ? 0u : (1u << n0) - 1;
                if (n0 >= 0 && n0 < 32) w |= (uint32_t)(anc << n0);
                else if (n0 < 0 && n0 > -64) w |= (uint32_t)(anc >> -n0);
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const int bit = 16 * (x >> 2) + 4 * (x & 3) + q4, byte = 8 * (4 * (x >> 2) + (x & 3)) + q4;
                    const float seen = bad >> byte & 1 ? NAN : 0.0f;
                    y[x] = (w >> bit & 1) && (ok >> byte & 1) ? y[x] + seen : -INFINITY;
                }
            }
            float mt = -INFINITY, rt = -INFINITY;
#pragma unroll
            for (int x = 0; x < 8; x++) {
                mt = fmaxf(mt, y[x] - k[x].y);
                rt = fmaxf(rt, y[x]);
            }
            mt = quarter_max(mt);
            rt = quarter_max(rt);
            if (__ballot(mt > M + TA_LAZY || rt > Rf + TA_LAZY)) {
                const float mn = mt > M + TA_LAZY ? ceilf(mt) : M, rn = rt > Rf + TA_LAZY ? ceilf(rt) : Rf;
                const float al = mn == M ? 1.0f : __builtin_amdgcn_exp2f(M - mn);
                lsum *= rn == Rf ? 1.0f : __builtin_amdgcn_exp2f(Rf - rn);
                M = mn;
                Rf = rn;
#pragma unroll
                for (int d = 0; d < DT; d++) acc[d] *= al;
            }
            const float ref = Rf == -INFINITY ? 0.0f : Rf, up = exp2_int(Rf - M, TS_UP);
            f16x8 ph, pl;
            float pw[8];
#pragma unroll
            for (int x = 0; x < 8; x++) {
                const float p = __builtin_amdgcn_exp2f(y[x] - ref);
                lsum += p;
                pw[x] = p * k[x].x * up;   // the second factor first: p 2^-k is at most 2^122
            }
            f16x8 pd;   // for the rows' lo parts
#pragma unroll
            for (int x = 0; x < 8; x += 2) {
                const f16x2 h = __builtin_convertvector(f2{pw[x], pw[x + 1]}, f16x2);
                const f16x2 l = __builtin_convertvector(f2{pw[x] - (float)h[0], pw[x + 1] - (float)h[1]}, f16x2);
                const f16x2 d = __builtin_convertvector(f2{pw[x] * (1.0f / TS_LO), pw[x + 1] * (1.0f / TS_LO)}, f16x2);
                ph[x] = h[0];
                ph[x + 1] = h[1];
                pl[x] = l[0];
                pl[x + 1] = l[1];
                pd[x] = d[0];
                pd[x + 1] = d[1];
            }
#pragma unroll
            for (int d = 0; d < DT; d += 2) {
#pragma unroll
                for (int i = 0; i < 2; i++) acc[d + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl[(d + i) % AV], pd, acc[d + i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 2; i++) acc[d + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[(d + i) % AV], pl, acc[d + i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 2; i++) acc[d + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[(d + i) % AV], ph, acc[d + i], 0, 0, 0);
                if (d + AV < DT)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        vh[(d + i) % AV] = vread(cur, d + i + AV, va);
                        vl[(d + i) % AV] = vread(cur + TB_BUF, d + i + AV, va);
                    }
                if (d < 8) {
                    put(s + 1, d / 2, sa);
                    load(d / 2);
                }
                if (d == 8) next_row();
                __builtin_amdgcn_sched_barrier(0);
            }
            lds_barrier();
        }
        lsum += __shfl_xor(lsum, 16, 64);
        lsum += __shfl_xor(lsum, 32, 64);

        if (row >= rows) continue;
        const size_t orow = (size_t)b * a.t.N * H + row, part = ((size_t)2 * id + (s0 == 0)) * ROWS + (row - r0);
        const int ch = 16 * DT * half + 4 * kq;   // this lane's first channels
        if (split) {
            const float m = part_max(M, lsum);
            if (kq == 0 && half == 0) {
                a.pm[part] = m;
                a.pr[part] = part_max(Rf, lsum);
                a.pl[part] = lsum;
            }
            if (m == -INFINITY) continue;   // nothing seen: the merge does not read its sums
            float *dst = a.po + part * KL + ch;
#pragma unroll
            for (int d = 0; d < DT; d++)
                if (16 * d + ch < KL) *reinterpret_cast<f32x4 *>(dst + 16 * d) = acc[d];
        } else {
            if (kq == 0 && half == 0 && a.lse) a.lse[orow] = lsum == 0.0f ? -INFINITY : (Rf + __builtin_amdgcn_logf(lsum)) * TA_LN2;
            const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum, down = exp2_int(M - Rf, -TS_UP);
            if (a.o_dt == K3HIP_F32) {
                float *dst = reinterpret_cast<float *>(a.o) + orow * KL + ch;
#pragma unroll
                for (int d = 0; d < DT; d++)
                    if (16 * d + ch < KL) *reinterpret_cast<f32x4 *>(dst + 16 * d) = acc[d] * inv * down;
            } else {
                uint16_t *dst = reinterpret_cast<uint16_t *>(a.o) + orow * KL + ch;
#pragma unroll
                for (int d = 0; d < DT; d++)
                    if (16 * d + ch < KL) *reinterpret_cast<uint2 *>(dst + 16 * d) = pack4(acc[d] * inv * down);
            }
        }
    }
}

// The parts of a row merged, by W waves: o = sum 2^(M_s - M) o_s / sum 2^(M_s - M) l_s, wave w the parts
// w, w + W, ..., the waves' sums in order. Of fp32 caches l_s is taken against R_s, not M_s, and o takes
// 2^(M - TS_UP - R). Eight waves a row up to 512 rows, where long sequences have many parts each (with the first launch, 64 rows of 125 parts: 28 us, 31 with four waves; of 256 parts: 34, 40), one beyond (1024 rows
// of 17 parts: 38, 40 with eight; 16,384 rows of 3: 40 us for the merge with four waves, 21 with one). The sums are
// asked for four parts at a time, the next four before these are added, and
// at the start every part's (M_s, l_s), a part a lane, before they are needed: one after the other their latencies
// made a merge of 16 parts 27 us. A part that saw nothing (M_s = -inf) left no sums: its memory is read, its
// weight not used. One that saw a NaN (M_s = inf) makes the row NaN.
constexpr int TM_PER = 4;
template <int W, bool F32>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void tree_attn_merge_kernel(const AttnArgs a, int tile_rows)
{
    __shared__ float s_m[W], s_r[W], s_l[W];
    __shared__ f32x4 s_v[W == 1 ? 1 : W][TA_KL / 4];
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = W == 1 ? 0 : tid >> 6;
    const int row = W == 1 ? blockIdx.x * 4 + (tid >> 6) : blockIdx.x;
    if (row >= tree_count(a.t, b) * a.H) return;
    const int rt = row / tile_rows, in = row % tile_rows;
    const int4 p = a.plan[b];
    const int n = p.y - p.x + 1;
    if (n <= 1) return;   // written by its only workgroup
    // part s: the first slot's second part, then the others' first
    auto at = [&](int s) -> size_t { return (2 * ((size_t)(p.x + s) * p.z + rt) + (s == 0)) * tile_rows + in; };
    const int mine = n > wv ? (n - wv + W - 1) / W : 0;   // this wave's parts
    f32x4 x[TM_PER][2];
    auto ask = [&](int i) {   // for parts i .. i + TM_PER - 1 of this wave's
#pragma unroll
        for (int k = 0; k < TM_PER; k++) {
            const float *src = a.po + at(wv + W * max(min(i + k, mine - 1), 0)) * a.KL;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int ch = 256 * c + 4 * lane;
                x[k][c] = ch < a.KL ? *reinterpret_cast<const f32x4 *>(src + ch) : f32x4(0.0f);
            }
        }
    };
    float M = -INFINITY, R = -INFINITY, l = 0.0f;
    f32x4 v[2] = {f32x4(0.0f), f32x4(0.0f)};
    if (mine > 0) ask(0);
    for (int i0 = 0; i0 < mine; i0 += 64) {
        const bool has = i0 + lane < mine;
        const size_t pa = at(wv + W * (has ? i0 + lane : 0));
        const float m = has ? a.pm[pa] : -INFINITY, pl = a.pl[pa];
        float mx = m;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        const float mn = fmaxf(M, mx), old = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - mn);
        const float w = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        float wl = w, oldl = old;
        if constexpr (F32) {
            const float r = has ? a.pr[pa] : -INFINITY;
            float rx = r;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) rx = fmaxf(rx, __shfl_xor(rx, o, 64));
            const float rn = fmaxf(R, rx);
            oldl = R == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(R - rn);
            wl = r == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(r - rn);
            R = rn;
        }
        float ls = wl == 0.0f ? 0.0f : wl * pl;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) ls += __shfl_xor(ls, o, 64);
        l = l * oldl + ls;
        v[0] *= old;
        v[1] *= old;
        M = mn;
        for (int i = 0; i < min(64, mine - i0); i += TM_PER) {
            f32x4 y[TM_PER][2];
#pragma unroll
            for (int k = 0; k < TM_PER; k++)
#pragma unroll
                for (int c = 0; c < 2; c++) y[k][c] = x[k][c];
            if (i0 + i + TM_PER < mine) ask(i0 + i + TM_PER);
#pragma unroll
            for (int k = 0; k < TM_PER; k++) {
                const float ws = __shfl(w, i + k, 64);   // zero past the last
                if (ws != 0.0f) {
                    v[0] += ws * y[k][0];
                    v[1] += ws * y[k][1];
                }
            }
        }
    }
    float Mx = M, Rx = F32 ? R : M;
    if constexpr (W > 1) {
        if (lane == 0) {
            s_m[wv] = M;
            s_r[wv] = Rx;
            s_l[wv] = l;
        }
        s_v[wv][lane] = v[0];
        s_v[wv][64 + lane] = v[1];
        __syncthreads();
        if (wv > 1) return;   // wave c takes channels 256 c .. + 255
        Mx = Rx = -INFINITY;
#pragma unroll
        for (int k = 0; k < W; k++) {
            Mx = fmaxf(Mx, s_m[k]);
            Rx = fmaxf(Rx, s_r[k]);
        }
        l = 0.0f;
        v[0] = v[1] = f32x4(0.0f);
#pragma unroll
        for (int k = 0; k < W; k++) {
            if (s_m[k] == -INFINITY) continue;
            const float w = __builtin_amdgcn_exp2f(s_m[k] - Mx);
            l += (F32 ? __builtin_amdgcn_exp2f(s_r[k] - Rx) : w) * s_l[k];
            v[0] += w * s_v[k][64 * wv + lane];
        }
        v[1] = v[0];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l, down = F32 ? exp2_int(Mx - Rx, -TS_UP) : 1.0f;
    const size_t orow = (size_t)b * a.t.N * a.H + row;
#pragma unroll
    for (int c = 0; c < 2; c++) {
        const int ch = 256 * c + 4 * lane;
        if (ch >= a.KL || (W > 1 && c != wv)) continue;
        if (a.o_dt == K3HIP_F32) *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(a.o) + orow * a.KL + ch) = v[c] * inv * down;
        else *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(a.o) + orow * a.KL + ch) = pack4(v[c] * inv * down);
    }
    if (a.lse && lane == 0 && wv == 0) a.lse[orow] = l == 0.0f ? -INFINITY : (Rx + __builtin_amdgcn_logf(l)) * TA_LN2;
}

// Query rows a workgroup takes: 128 on bf16 where a sequence has more (64 and 128 measured: 64 sequences of 128 rows
// 150 and 157 us, of 256 rows 270 and 240, 4 of 4096 rows 997 and 798): half the LDS reads a product, but larger
// parts.
int ta_rows(bool f32, long rows) { return f32 || rows <= 128 ? 64 : 128; }

// The workgroups of a launch, the least multiple of the CUs whose slots of n leave no more than a
// tenth of them without work.
long ta_grid(int n)
{
    int ncu = 256;
    (void)cu_count(ncu);
    long best = 0;
    double most = 0.0;
    for (long k = (n + ncu - 1) / ncu, k0 = k; k < k0 + 4; k++) {
        const double used = (double)(ncu * k / n * n) / (double)(ncu * k);
        if (used > most + 0.01) {
            most = used;
            best = ncu * k;
        }
        if (used >= 0.9) break;
    }
    return (best + 7) & ~7L;   // a multiple of the XCDs
}

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// Sequences and query rows that the launches hold.
bool ta_fits(int B, int N, int H) { return B <= 65535 && (long)N * H <= 65535L * 16; }

// `parts` partial sums of `rows` rows, and the plan of B sequences.
size_t ta_ws_bytes(long parts, int rows, int KL, int B)
{
    const size_t r = (size_t)parts * rows;
    return up256(r * KL * 4) + 3 * up256(r * 4) + up256((size_t)B * sizeof(int4));
}

}  // namespace

}  // namespace k3kda

using namespace k3kda;

extern "C" size_t k3hip_mla_tree_workspace(int B, int N, int H, int kv_lora)
{
    if (B <= 0 || N <= 0 || N > TREE_MAX || H <= 0 || kv_lora <= 0 || kv_lora > TA_KL || !ta_fits(B, N, H)) return 0;
    size_t most = 0;
    for (bool f32 : {false, true}) {
        const int rows = ta_rows(f32, (long)N * H);
        most = std::max(most, ta_ws_bytes(2 * ta_grid((int)(((long)N * H + rows - 1) / rows)), rows, kv_lora, B));
    }
    return most;
}

extern "C" int k3hip_mla_tree_attention(int B, int N, int H, int kv_lora, int rope, float scale, const void *q,
                                        const void *pages, int dtype, int n_pages, int page, const int *table,
                                        int max_pages, const int *lens, const int *counts, const int *parents, void *o,
                                        int o_dtype, float *lse, void *workspace, size_t workspace_bytes, void *stream)
{
    clear_error();
    static const char *who = "k3hip_mla_tree_attention";
    if (int rc = paged_check(who, B, N, n_pages, page, max_pages, pages, table, lens)) return rc;
    if (H <= 0) K3_FAIL(K3HIP_EINVAL, "%s: H=%d", who, H);
    if (N > TREE_MAX) K3_FAIL(K3HIP_EUNSUPPORTED, "%s: a tree of %d nodes (at most %d)", who, N, TREE_MAX);
    if (dtype != K3HIP_F32 && dtype != K3HIP_BF16) K3_FAIL(K3HIP_EINVAL, "%s: cache dtype=%d", who, dtype);
    if (o_dtype != K3HIP_F32 && o_dtype != K3HIP_BF16) K3_FAIL(K3HIP_EINVAL, "%s: o_dtype=%d", who, o_dtype);
    const int CW = kv_lora + rope;
    if (kv_lora <= 0 || rope < 0 || kv_lora > TA_KL || CW > TA_CW || kv_lora % 8 || rope % 8)
        K3_FAIL(K3HIP_EUNSUPPORTED, "%s: kv_lora=%d rope=%d (multiples of 8, at most %d and %d together)", who, kv_lora,
                rope, TA_KL, TA_CW);
    if (!(scale > 0.0f)) K3_FAIL(K3HIP_EINVAL, "%s: scale=%g (positive)", who, scale);
    if (B * (((long)max_pages * page + N) / TB_TP + 1) > 0x3fffff00L)   // steps: sums of two counts fit an int
        K3_FAIL(K3HIP_EINVAL, "%s: %d sequences of up to %ld positions", who, B, (long)max_pages * page);
    if ((long)page * CW * 4 > 0x7fffffffL) K3_FAIL(K3HIP_EINVAL, "%s: pages of %d rows", who, page);
    if (!ta_fits(B, N, H)) K3_FAIL(K3HIP_EINVAL, "%s: B=%d N=%d H=%d", who, B, N, H);
    if (B == 0 || N == 0) return K3HIP_OK;
    if (!q || !o) K3_FAIL(K3HIP_EINVAL, "%s: NULL q or o", who);
    if (((uintptr_t)q | (uintptr_t)pages | (uintptr_t)o) & 15)
        K3_FAIL(K3HIP_EINVAL, "%s: q, pages and o need 16-byte alignment", who);
    hipStream_t st = as_stream(stream);
    const bool f32 = dtype == K3HIP_F32;
    AttnArgs a{};
    a.t = TreeSeqs{N, lens, counts, parents};
    a.c = PagedRows{table, n_pages, page, max_pages};
    a.H = H; a.CW = CW; a.KL = kv_lora;
    a.pages = pages; a.q = q; a.o = o; a.o_dt = o_dtype; a.lse = lse;
    a.scale2 = scale * TA_LOG2E;
    const int rows = ta_rows(f32, (long)N * H);
    const long grid = ta_grid((int)(((long)N * H + rows - 1) / rows));
    a.B = B;
    a.tcol = TB_TP / page;
    a.trow = TB_TP % page;
    a.page_bytes = (uint32_t)page * (uint32_t)CW * (f32 ? 4 : 2);
    const size_t need = ta_ws_bytes(2 * grid, rows, kv_lora, B);
    StreamBuf buf;
    if (!workspace) {
        if (int rc = stream_alloc(buf, need, st)) return rc;
        workspace = buf.p;
    } else if (workspace_bytes < need || ((uintptr_t)workspace & 15)) {
        K3_FAIL(K3HIP_EINVAL, "%s: workspace of %zu bytes, %zu needed, 16-byte aligned", who, workspace_bytes, need);
    }
    const size_t r = (size_t)2 * grid * rows;
    a.po = (float *)workspace;
    a.pm = (float *)((char *)workspace + up256(r * kv_lora * 4));
    a.pl = (float *)((char *)a.pm + up256(r * 4));
    a.pr = (float *)((char *)a.pl + up256(r * 4));
    a.plan = (int4 *)((char *)a.pr + up256(r * 4));
    // bf16: eight rows of full width in one page go by buffer loads from one address (otherwise an address a lane, by
    // global loads: 830 us for 798 at 4 sequences of 64 nodes over 32,768 positions, 4% more at 64 tokens over 8192)
    const void *kern;
    const size_t lds = f32 ? TS_LDS : TB_LDS;
    if (f32) kern = CW == TA_CW ? (const void *)tree_attn32_kernel<true> : (const void *)tree_attn32_kernel<false>;
    else if (CW == TA_CW && page % 8 == 0)
        kern = rows == 64 ? (const void *)tree_attn16_kernel<true, 1> : (const void *)tree_attn16_kernel<true, 2>;
    else kern = rows == 64 ? (const void *)tree_attn16_kernel<false, 1> : (const void *)tree_attn16_kernel<false, 2>;
    K3_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    void *args[] = {&a};
    K3_HIP(hipLaunchKernel(kern, dim3((unsigned)grid), dim3(f32 ? TS_NT : TA_NT), args, lds, st));
    K3_LAUNCHED();
    const bool few = (long)B * N * H <= 512;
    const dim3 mg(few ? (unsigned)(N * H) : (unsigned)((N * H + 3) / 4), (unsigned)B);
    if (few && f32) hipLaunchKernelGGL((tree_attn_merge_kernel<8, true>), mg, dim3(512), 0, st, a, rows);
    else if (few) hipLaunchKernelGGL((tree_attn_merge_kernel<8, false>), mg, dim3(512), 0, st, a, rows);
    else if (f32) hipLaunchKernelGGL((tree_attn_merge_kernel<1, true>), mg, dim3(256), 0, st, a, rows);
    else hipLaunchKernelGGL((tree_attn_merge_kernel<1, false>), mg, dim3(256), 0, st, a, rows);
    K3_LAUNCHED();
    return K3HIP_OK;
}
