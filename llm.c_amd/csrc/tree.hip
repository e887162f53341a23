// tree.hip — attention for a tree of drafted tokens per sequence over its KV
// cache, gfx950.  Nodes i < N <= 64 of sequence b, anc(i) = i's ancestors in
// the tree and i itself:
//   q, k, v = rms_norm(x) . [W_Q | W_K | W_V], RoPE at pos[b] + |anc(i)| - 1
//   s(i, t) = q_i . K_t / sqrt(hd), t over cached rows 0 .. pos[b] - 1 and
//             over the nodes anc(i)
//   y_i = x_i + W_O . (sum_t e^s(i, t) V_t / sum_t e^s(i, t))
// The decode step's mathematics (attention.hip) for N rows that share one
// pass over the cache; N = 1 is that step.
//
// Launches: QKV (which also finds the rows' positions), attention, the merge
// of the splits (if any), W_O.
//
// Attention: the N G query rows of one (sequence, kv head), G query heads
// per kv head, are cut into blocks of 16 QT; a wave takes such a block over
// a range of 16-position tiles.  Products on the fp32 matrix cores
// (v_mfma_f32_16x16x4_f32), transposed so that no operand passes through
// LDS:
//   S^T = K Q^T    M = 16 positions, N = 16 query rows, k = head dimension.
//                  Lane l holds K[l % 16][g HD/4 ..] with g = l / 16 straight
//                  from memory (k step s of lane group g is dimension g HD/4 +
//                  s), Q the same way, kept for the whole range.
//   softmax        lane l's four sums of a tile are positions 4 g + r of query
//                  row l % 16.
//   O^T = V^T P^T  k step r takes positions 4 g + r: the probabilities are
//                  the B operand as they lie, and V's rows 4 g + r, DT dimensions
//                  per lane, the A operand as they come from memory.
// The running maximum m of a query row moves only when a score passes it by
// more than kSlack (in log2 units): a shuffle-free check for most tiles; sums stay exact
// to fp32 because e^(s - m) <= 2^kSlack is a float like any other.
#include "attn_proj.h"
#include "gemm_split.h"
#include "moe_internal.h"
#include "moe_math.h"
#include <algorithm>

namespace moe {
namespace {

using split::fx4;
using split::fx16;
using split::ux4;
using split::Frag;
using split::kPairA;
using split::kPairB;
using split::kPairs;

constexpr float kSlack = 16.0f;
// The split kernel: m is kSplitLift below the maximum it was set from, and
// moves when a score passes it by kSplitSlack.
constexpr float kSplitLift = 12.0f, kSplitSlack = 15.0f;
// Outputs whose dimensions are this much smaller (root mean square) than the
// largest values there are left to float products.
constexpr float kLeastOut = 0x1p-12f;
// Keys and queries from here on are left to float products.
constexpr float kMostKey = 4096.0f;
// And scores (log2 units) that the split could move by more than this: 2.6e-6 of
// a probability.
constexpr float kMostError = 0x1p-18f;
constexpr float kLow = -3.0e38f;   // running maximum before the first score
constexpr int kWaves = 4;
constexpr int kMaxSplits = 128;
constexpr long long kLittle = 1LL << 22;   // query rows times positions

// ---------------------------------------------------------------------------
// The tree of one sequence by a wave, lane base + i = node i.
struct Node {
    unsigned long long anc;   // ancestors and itself
    bool chain;               // the chain of parents ends at the context
};
// par: node i's parent (anything for lanes without a node).  By pointer
// doubling: after step s `up` holds the nearest 2^s members of the chain and
// `jump` the next.
__device__ inline Node tree_node(int par, int i, int base, bool node) {
    int jump = node && par >= -1 && par < i ? par : -2;
    unsigned long long up = 1ull << i;
#pragma unroll
    for (int s = 0; s < 6; ++s) {
        const int src = base + max(jump, 0);
        const unsigned lo = __shfl((unsigned)up, src), hi = __shfl((unsigned)(up >> 32), src);
        const int jj = __shfl(jump, src);
        if (jump >= 0) {
            up |= (unsigned long long)hi << 32 | lo;
            jump = jj;
        }
    }
    return Node{up, jump == -1};
}
// RoPE position of a node, or -1 if it is no token of the call.
__device__ inline int node_pos(const Node &n, int pos, int max_seq) {
    const int depth = __popcll(n.anc) - 1;
    return n.chain && pos >= 0 && pos < max_seq && depth < max_seq - pos ? pos + depth : -1;
}

}  // namespace

// p[r - r0] = the position of rows r0 .. r0 + n - 1 (those below B): a wave
// takes 64 / N whole sequences at a time.
__device__ inline void TreeArgs::find_rows(int r0, int n, int wave, int waves, int lane, int *p) const {
    const int per = 64 / N, last = (min(r0 + n, B) - 1) / N;
    const int i = lane % N, base = lane - i;
    for (int s = r0 / N + wave * per; s <= last; s += waves * per) {
        const int b = s + lane / N;
        const bool node = lane < per * N && b < seqs;
        const size_t r = node ? (size_t)b * N + i : 0;
        const int at = pos[node ? b : 0];
        const Node t = tree_node(parent[r], i, base, node);
        if (node && r >= (size_t)r0 && r < (size_t)r0 + n) p[r - r0] = node_pos(t, at, max_seq);
    }
}

namespace {

// ---------------------------------------------------------------------------
// Projections of many rows on the bf16 matrix cores, operands as sums of
// three bf16 terms (gemm_split.h): Y = X . W for 32 MB rows and 32 NT columns per
// workgroup, the reduction cut over its four waves, so that a few hundred rows
// already fill the card.  Nothing is shared inside the loop: lane l holds
// row l % 32 of X, k 8 (l / 32) .. + 7 of each 16 straight from memory and splits it;
// the weights are kept split, in operand order (launch_pack_split): a KB
// per 32 columns, 16 k and term.  The waves' sums meet in LDS; then, as in
// proj16_kernel: QKV rows are scaled by 1/rms, q and k turned by RoPE; W_O's
// are added to x.
// Number range: the split holds an operand to 2^-134 at worst (its last
// term is a bfloat16 subnormal), 24 bits from 2^-109 on.  Weights with a
// nonzero value below that, or one of 2^127 and more, are not used in this form
// at all (TreeArgs::wqkv_s null; loaded under a captured launch, every sum is
// computed again), so a sum over K products of weights up to w is
// off by at most K w 2^-134 from it: a sum below max(2^-80, K w
// 2^-110), and one that is not finite, is computed again as float products.
// Measured (d = 512, 8/2 heads of 64): QKV of 4096 rows 32 us (100 TFLOP/s of float
// products), W_O 22; of 1024 rows 13 and 8.4.  Bound by what each wave does for
// its tile, in turn: splitting X (a third of the VALU's 10 us), the products (8 us
// of the matrix cores), the epilogue (5 us), the start (4 us).  X through LDS,
// split once for 64 columns with a barrier a step: 42 and 27, 18 and 14.
template <bool QKV, int MB, int NT>
__global__ __launch_bounds__(256, NT > 2 ? 1 : 2) void proj_mma_kernel(TreeArgs a, int ntiles) {
    constexpr int LD = 32 * NT + 4;
    __shared__ __align__(16) float red[4][32][LD];
    __shared__ float ssq[4][32 * MB];
    __shared__ int rowp[32 * MB];
    const int M = QKV ? a.d : a.qd, NC = QKV ? a.qd + 2 * a.kd : a.d;
    const float *X = QKV ? a.x : a.o;
    const int nsteps = (M + 15) / 16;
    const unsigned short *W = QKV ? a.wqkv_s : a.wo_s;
    // Every eighth workgroup runs on one XCD: the column tiles of a row block
    // go to the same one, one after the other, and share its L2.
    const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
    const int nt = slot % ntiles, r0 = ((slot / ntiles) * 8 + xcd) * 32 * MB, c0 = nt * 32 * NT;
    if (r0 >= a.B) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5;

    const float *xp[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m)
        xp[m] = X + (size_t)min(r0 + 32 * m + li, a.B - 1) * M;
    // 32-column tile j of this workgroup (the last may be past the end: that
    // one again, left out below).
    const int tiles32 = (NC + 31) / 32;
    const unsigned short *wp[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
        wp[j] = W + (size_t)min(NT * nt + j, tiles32 - 1) * nsteps * 1536 + lane * 8;

    // Two sets of registers: loads run two steps ahead.  Every load is
    // unconditional (past the wave's range: its last step again, times zeros
    // of X) and what it brings is touched only when its step comes, so that a
    // step waits for its own.
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    const int s0 = nsteps * wave / 4, s1 = nsteps * (wave + 1) / 4;
    fx4 ra[2][MB][2], rw[2][2];
    ux4 rb[2][NT][3];
    auto load = [&](auto set, int step) {
        constexpr int S = decltype(set)::value;
        const int s = max(min(step, s1 - 1), 0), k = 16 * s + 8 * lh;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int kk = k + 4 * i < M ? k + 4 * i : 0;
#pragma unroll
            for (int m = 0; m < MB; ++m) ra[S][m][i] = *reinterpret_cast<const fx4 *>(xp[m] + kk);
            if (QKV) rw[S][i] = *reinterpret_cast<const fx4 *>(a.rms_w + kk);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int p = 0; p < 3; ++p)
                rb[S][j][p] = *reinterpret_cast<const ux4 *>(wp[j] + (size_t)s * 1536 + p * 512);
    };
    fx16 acc[MB][NT];
    float ss[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        ss[m] = 0.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[m][j][r] = 0.0f;
    }
    load(S0{}, s0);
    load(S1{}, s0 + 1);
    if (QKV) a.find_rows(r0, 32 * MB, wave, 4, lane, rowp);
    else if (tid < 32 * MB) rowp[tid] = r0 + tid < a.B ? a.row_pos(r0 + tid) : -1;
    auto step = [&](auto set, int s) {
        constexpr int S = decltype(set)::value;
        Frag fa[MB];
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            fx4 v[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool in = s < s1 && 16 * s + 8 * lh + 4 * i < M;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = in ? ra[S][m][i][e] : 0.0f;
                    if (QKV) {
                        ss[m] = fmaf(x, x, ss[m]);
                        x *= rw[S][i][e];
                    }
                    v[i][e] = x;
                }
            }
            fa[m] = split::split8(v[0], v[1]);
        }
#pragma unroll
        for (int q = 0; q < kPairs; ++q)
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[m][j] = split::mma(fa[m].t[kPairA[q]], rb[S][j][kPairB[q]], acc[m][j]);
        load(set, s + 2);
        __builtin_amdgcn_sched_barrier(0);   // (the loads stay here)
    };
    for (int s = s0; s < s1; s += 2) {
        step(S0{}, s);
        step(S1{}, s + 1);
    }
    if (QKV)
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const float t = ss[m] + __shfl_xor(ss[m], 32);
            if (lh == 0) ssq[wave][32 * m + li] = t;
        }
    // Thread: row tid / 8, columns 8 (tid % 8) .. + 7 of each 64 (all q, all k or all v).
    const int row = tid >> 3;
    const unsigned *range = a.range + (QKV ? 0 : 2);
    const bool unfit = range[1] != 0;
    const float small = fmaxf(0x1p-80f, (float)M * 0x1p-110f * __uint_as_float(range[0]));
    auto doubtful = [&](float y) {
        return unfit || (!(fabsf(y) >= small && fabsf(y) <= 3.4028235e38f) && y != 0.0f);
    };
#pragma unroll
    for (int m = 0; m < MB; ++m) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                red[wave][8 * (r >> 2) + 4 * lh + (r & 3)][32 * j + li] = acc[m][j][r];
        __syncthreads();
        const int orow = r0 + 32 * m + row;
#pragma unroll 1
        for (int c8 = 8 * (tid & 7); c8 < 32 * NT; c8 += 64) {
            const int col = c0 + c8;
            const int p = orow < a.B && col < NC ? rowp[32 * m + row] : -1;
            if (QKV && col == 0 && orow < a.B) a.keep_row(orow, p);
            if (p < 0) continue;
            float y[8];
            bool again = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y[e] = ((red[0][row][c8 + e] + red[1][row][c8 + e]) +
                        red[2][row][c8 + e]) + red[3][row][c8 + e];
                again |= col + e < NC && doubtful(y[e]);
            }
            if (again)
                for (int e = 0; e < 8 && col + e < NC; ++e) {
                    if (!doubtful(y[e])) continue;
                    const int c = col + e;
                    const float *w = !QKV ? a.wo + c : c < a.qd ? a.wq + c : c < a.qd + a.kd ? a.wk + (c - a.qd) : a.wv + (c - a.qd - a.kd);
                    const int ld = !QKV ? a.d : c < a.qd ? a.qd : a.kd;
                    float t = 0.0f;
                    for (int k = 0; k < M; ++k) {
                        const float x = X[(size_t)orow * M + k];
                        t = fmaf(QKV ? x * a.rms_w[k] : x, w[(size_t)k * ld], t);
                    }
                    y[e] = t;
                }
            if (QKV) {
                const float sq = (ssq[0][32 * m + row] + ssq[1][32 * m + row]) + (ssq[2][32 * m + row] + ssq[3][32 * m + row]);
                const float inv = 1.0f / sqrtf(sq / (float)M + a.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] *= inv;
                const int hc = col < a.qd ? col : col < a.qd + a.kd ? col - a.qd : col - a.qd - a.kd;
                if (col < a.qd + a.kd) {
                    const size_t t0 = (size_t)p * (a.hd / 2) + (hc % a.hd) / 2;
#pragma unroll
                    for (int e = 0; e < 4; ++e) rope_pair(y[2 * e], y[2 * e + 1], a.cos_t[t0 + e], a.sin_t[t0 + e]);
                }
                float *dst = (col < a.qd ? a.q + (size_t)orow * a.qd : a.kv_row(orow, p, col < a.qd + a.kd)) + hc;
                *reinterpret_cast<float4 *>(dst) = make_float4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<float4 *>(dst + 4) = make_float4(y[4], y[5], y[6], y[7]);
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (col + 4 * h >= NC) break;   // (d is a multiple of 4)
                    const float4 xo = *reinterpret_cast<const float4 *>(a.x + (size_t)orow * a.d + col + 4 * h);
                    *reinterpret_cast<float4 *>(a.out_row(orow) + col + 4 * h) =
                        add4(xo, make_float4(y[4 * h], y[4 * h + 1], y[4 * h + 2], y[4 * h + 3]));
                }
            }
        }
        if (m + 1 < MB) __syncthreads();
    }
}

// src [K x N] (fp32, row-major) as columns col0 .. of the split weights:
// dst[tile][k step][term][lane][8], lane l of tile t: column 32 t + l % 32,
// k 16 step + 8 (l / 32) .. + 7.  Thread (column, group of 8 k).
// range[0] = the bits of the largest |value|, range[1] = 1 where one cannot be
// held (both grow only).
__global__ __launch_bounds__(256) void pack_split_kernel(const float *src, unsigned short *dst, int K,
                                                         int N, int col0, unsigned *range) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int groups = (K + 7) / 8;
    if (i >= (size_t)groups * N) return;
    const int n = (int)(i % N), kg = (int)(i / N), c = col0 + n;
    float v[8];
    unsigned most = 0, bad = 0;
    for (int e = 0; e < 8; ++e) {
        v[e] = 8 * kg + e < K ? src[(size_t)(8 * kg + e) * N + n] : 0.0f;
        const unsigned u = __float_as_uint(v[e]) & 0x7fffffffu;
        most = max(most, u);
        bad |= (u != 0 && u < __float_as_uint(0x1p-109f)) || u >= __float_as_uint(0x1p127f);
    }
    // (most threads find the maximum taken already)
    if (most > __hip_atomic_load(&range[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))
        atomicMax(&range[0], most);
    if (bad) atomicOr(&range[1], 1u);
    const Frag f = split::split8(fx4{v[0], v[1], v[2], v[3]}, fx4{v[4], v[5], v[6], v[7]});
    unsigned short *d = dst + ((size_t)(c / 32) * ((K + 15) / 16) + kg / 2) * 1536 +
                        ((c & 31) + 32 * (kg & 1)) * 8;
    for (int p = 0; p < 3; ++p) *reinterpret_cast<ux4 *>(d + p * 512) = f.t[p];
}

// ---------------------------------------------------------------------------
template <int CNT, int VEC> __device__ inline void load_vec(const float *p, float *v) {
    static_assert(CNT % VEC == 0, "whole vectors");
    typedef float vec __attribute__((ext_vector_type(VEC)));
#pragma unroll
    for (int i = 0; i < CNT / VEC; ++i) {
        const vec t = *reinterpret_cast<const vec *>(p + VEC * i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[VEC * i + j] = t[j];
    }
}

template <int HD> struct Shape {
    static constexpr int KS = HD / 4;                      // k steps of a score tile
    static constexpr int KV = HD % 16 == 0 ? 4 : 2;        // floats per load of a K row
    static constexpr int DT = (HD + 15) / 16;              // output tiles
    static constexpr int LDO = 16 * DT + 4;                // row of the merge buffer
};

// Partial results of some positions are kept as (m, l, o): l = sum e^(s - m),
// o the normalised output, which never passes the largest |V| (0 where no
// position counts); joined by the weights l e^(m - M) / L.
__device__ inline float part_inv(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// One workgroup: block rb of 16 QT query rows of (sequence b, kv head kvh),
// split sp of the positions; its four waves take a quarter of the split each
// and merge through LDS.  Bound by the reads where rows are few: 64 single
// tokens over 1024 positions (8/2 heads of 64) 14.7 us, 59 MB at 4.0 TB/s; one
// tree of 8 6.3 us, a round trip of loads and the merge.
template <int HD, int QT>
__global__ __launch_bounds__(256, 2) void tree_attn_kernel(TreeArgs a, int blocks) {
    constexpr int KS = Shape<HD>::KS, KV = Shape<HD>::KV, DT = Shape<HD>::DT, LDO = Shape<HD>::LDO;
    constexpr int ROWS = 16 * QT, NS = 3;
    __shared__ float sm_o[kWaves][ROWS][LDO];
    __shared__ float sm_m[kWaves][ROWS], sm_l[kWaves][ROWS];
    int id = blockIdx.x;
    const int sp = id % a.splits; id /= a.splits;
    const int rb = id % blocks; id /= blocks;
    const int kvh = id % a.nkv, b = id / a.nkv;
    const int N = a.N, G = a.nh / a.nkv, rows = N * G;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, g = lane >> 4;

    const int pos = __builtin_amdgcn_readfirstlane(a.pos[b]);
    if (pos < 0 || pos >= a.max_seq) return;   // (no live node)
    const int par = lane < N ? a.parent[(size_t)b * N + lane] : -2;

    // Tiles 0 .. nct - 1 are cached positions, the others nodes.  The loads of
    // NS tiles are in flight; rows past a tile's last read that one again and
    // are masked when they arrive.
    const int nct = (pos + 15) / 16, nt = nct + (N + 15) / 16;
    const int parts = a.splits * kWaves, part = sp * kWaves + wave;
    const int t0 = (int)((long long)nt * part / parts), t1 = (int)((long long)nt * (part + 1) / parts);
    const float *kc = a.kc + (size_t)b * a.max_seq * a.kd + kvh * HD, *kn = a.kd_out + (size_t)b * N * a.kd + kvh * HD;
    const float *vc = a.vc + (size_t)b * a.max_seq * a.kd + kvh * HD, *vn = a.vd_out + (size_t)b * N * a.kd + kvh * HD;
    float k[NS][KS], v[NS][4][DT];
    auto load = [&](auto set, int t) {
        constexpr int S = decltype(set)::value;
        const bool draft = t >= nct;
        const int p0 = 16 * (draft ? t - nct : t), n = min(16, (draft ? N : pos) - p0);
        const float *kb = (draft ? kn : kc) + (size_t)p0 * a.kd, *vb = (draft ? vn : vc) + (size_t)p0 * a.kd;
        load_vec<KS, KV>(kb + min(li, n - 1) * a.kd + g * KS, k[S]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float *vp = vb + min(4 * g + r, n - 1) * a.kd;
            if constexpr (HD == 16 * DT || HD % DT == 0) {
                // (whole lanes of DT dimensions)
                load_vec<DT, DT == 3 ? 1 : DT>(vp + (DT * li < HD ? DT * li : 0), v[S][r]);
            } else {
#pragma unroll
                for (int d = 0; d < DT; ++d) v[S][r][d] = vp[DT * li + d < HD ? DT * li + d : 0];
            }
        }
    };
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    using S2 = std::integral_constant<int, 2>;
    if (t0 < t1) load(S0{}, t0);
    if (t0 + 1 < t1) load(S1{}, t0 + 1);
    if (t0 + 2 < t1) load(S2{}, t0 + 2);

    // Query rows r = 16 QT rb + 16 c + li, node r / G, head r % G; past the
    // last row: that row again.  Scores in log2 units.  The queries of nodes
    // that are no token are whatever the workspace holds: their maximum starts
    // at infinity, which no score passes, so that they have no say in when the
    // wave's maxima move.
    float q[QT][KS], m[QT];
    unsigned long long anc[QT];
    const float scale = a.scale * 1.4426950408889634f;
#pragma unroll
    for (int c = 0; c < QT; ++c) {
        const int r = min(rb * ROWS + 16 * c + li, rows - 1), n = r / G;
        load_vec<KS, KV>(a.q + ((size_t)b * N + n) * a.qd + (kvh * G + r % G) * HD + g * KS, q[c]);
    }
    const Node node = tree_node(par, lane, 0, lane < N);
    const unsigned long long live = __ballot(lane < N && node_pos(node, pos, a.max_seq) >= 0);
#pragma unroll
    for (int c = 0; c < QT; ++c) {
        const int n = min(rb * ROWS + 16 * c + li, rows - 1) / G;
        anc[c] = (unsigned long long)__shfl((unsigned)(node.anc >> 32), n) << 32 |
                 (unsigned)__shfl((unsigned)node.anc, n);
        m[c] = live >> n & 1 ? kLow : INFINITY;
#pragma unroll
        for (int s = 0; s < KS; ++s) q[c][s] *= scale;
    }

    float l[QT];
    fx4 o[QT][DT];
#pragma unroll
    for (int c = 0; c < QT; ++c) {
        l[c] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[c][d] = fx4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    auto step = [&](auto set, int t) {
        constexpr int S = decltype(set)::value;
        const bool draft = t >= nct;
        const int p0 = 16 * (draft ? t - nct : t);
        const int n = min(16, (draft ? N : pos) - p0);   // positions of the tile
        fx4 s[QT];
#pragma unroll
        for (int c = 0; c < QT; ++c) s[c] = fx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int c = 0; c < QT; ++c)
                s[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[S][i], q[c][i], s[c], 0, 0, 0);
        float w[4][DT];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int d = 0; d < DT; ++d)
                w[r][d] = HD == 16 * DT || DT * li + d < HD ? v[S][r][d] : 0.0f;
        unsigned in = 0xffffu;   // bit j: position p0 + j counts
        if (draft || n < 16) {
            in = draft ? (unsigned)(live >> p0) & 0xffffu : (1u << n) - 1;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    w[r][d] = in >> (4 * g + r) & 1 ? w[r][d] : 0.0f;
#pragma unroll
            for (int c = 0; c < QT; ++c) {
                const unsigned see = (draft ? in & (unsigned)(anc[c] >> p0) : in) >> (4 * g);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!(see >> r & 1)) s[c][r] = -INFINITY;
            }
        }
        if (t + NS < t1) load(set, t + NS);
        float over = kLow;
#pragma unroll
        for (int c = 0; c < QT; ++c)
            over = fmaxf(over, fmaxf(fmaxf(s[c][0], s[c][1]), fmaxf(s[c][2], s[c][3])) - m[c]);
        if (__any(over > kSlack)) {
#pragma unroll
            for (int c = 0; c < QT; ++c) {
                float x = fmaxf(fmaxf(s[c][0], s[c][1]), fmaxf(s[c][2], s[c][3]));
                x = fmaxf(x, __shfl_xor(x, 16));
                x = fmaxf(x, __shfl_xor(x, 32));
                x = fmaxf(x, m[c]);
                const float f = __builtin_amdgcn_exp2f(m[c] - x);
                m[c] = x;
                l[c] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[c][d] = o[c][d] * f;
            }
        }
#pragma unroll
        for (int c = 0; c < QT; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[c][r] = __builtin_amdgcn_exp2f(s[c][r] - m[c]);
                l[c] += s[c][r];
            }
        if (draft) {
            // A probability that the mask makes zero must not meet an
            // infinity or NaN of a node that its row does not see: such
            // values leave the product and are added where they are seen.
            float chk = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int d = 0; d < DT; ++d) chk = fmaf(w[r][d], 0.0f, chk);
            if (__any(chk != 0.0f)) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int d = 0; d < DT; ++d) w[r][d] = fabsf(w[r][d]) < INFINITY ? w[r][d] : 0.0f;
#pragma unroll 1
                for (int j = 0; j < n; ++j) {
                    if (!(in >> j & 1)) continue;
#pragma unroll
                    for (int c = 0; c < QT; ++c) {
                        const float pr = j % 4 == 0 ? s[c][0] : j % 4 == 1 ? s[c][1] : j % 4 == 2 ? s[c][2] : s[c][3];
                        const float pj = __shfl(pr, (j / 4) * 16 + li);
#pragma unroll
                        for (int d = 0; d < DT; ++d)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const int dim = DT * (4 * g + r) + d;
                                const float x = vn[(size_t)(p0 + j) * a.kd + (dim < HD ? dim : 0)];
                                if (!(fabsf(x) < INFINITY) && dim < HD && (anc[c] >> (p0 + j) & 1))
                                    o[c][d][r] += pj * x;
                            }
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < QT; ++c)
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    o[c][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[r][d], s[c][r], o[c][d], 0, 0, 0);
    };
    for (int t = t0; t < t1; t += NS) {
        step(S0{}, t);
        if (t + 1 < t1) step(S1{}, t + 1);
        if (t + 2 < t1) step(S2{}, t + 2);
    }

    // The wave's partial outputs; true where one is not finite.
    auto put = [&](bool again) {
        bool more = false;
#pragma unroll
        for (int c = 0; c < QT; ++c) {
            float x = l[c] + __shfl_xor(l[c], 16);
            x += __shfl_xor(x, 32);
            if (g == 0 && !again) {
                sm_m[wave][16 * c + li] = m[c];
                sm_l[wave][16 * c + li] = x;
            }
            const float inv = part_inv(x);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    float &out = sm_o[wave][16 * c + li][DT * (4 * g + r) + d];
                    if (!again || !(fabsf(out) < INFINITY)) out = o[c][d][r] * inv;
                    more |= !(fabsf(o[c][d][r]) < INFINITY) && m[c] < INFINITY;
                }
        }
        return more;
    };
    // Values from 2^92 or so on may sum to infinity, as a probability is up to
    // 2^kSlack: then the range once more, tile by tile, with maxima so high that
    // the probabilities' sum is 1 at most, for the dimensions that need it.
    if (__any(put(false))) {
#pragma unroll
        for (int c = 0; c < QT; ++c) {
            m[c] += kSlack + 20.0f;   // (fewer than 2^20 positions)
            l[c] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[c][d] = fx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll 1
        for (int t = t0; t < t1; ++t) {
            load(S0{}, t);
            step(S0{}, t);
        }
        put(true);
    }
    // The waves' outputs, in wave order.
    __syncthreads();
    const size_t bk = (size_t)b * a.nkv + kvh;
    for (int e = tid; e < ROWS * HD; e += 256) {
        const int row = e / HD, dim = e % HD, r = rb * ROWS + row;
        if (r >= rows) continue;
        float M = sm_m[0][row];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) M = fmaxf(M, sm_m[w][row]);
        float f[kWaves], L = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            f[w] = __builtin_amdgcn_exp2f(sm_m[w][row] - M) * sm_l[w][row];
            L += f[w];
        }
        const float inv = a.splits == 1 ? 1.0f / L : part_inv(L);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) O = fmaf(f[w] * inv, sm_o[w][row][dim], O);
        if (a.splits == 1) {
            a.o[((size_t)b * N + r / G) * a.qd + (kvh * G + r % G) * HD + dim] = O;
        } else {
            float *pp = a.part + ((bk * rows + r) * a.splits + sp) * (HD + 2);
            pp[2 + dim] = O;
            if (dim == 0) {
                pp[0] = M;
                pp[1] = L;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Many query rows (more than 32): the same products on the fp16 matrix cores,
// each operand as two fp16 terms (v_mfma_f32_32x32x16_f16, three for a product).
// x = h + l with h = fp16(x), l = fp16(x - h): 11 + 11 significant bits and
// the sign of l, so a product of the terms hh + hl + lh is off by about 2^-22
// of it at worst, where the float products' chain rounds its running sum at
// 2^-24 eight times as often.  (Three bf16 terms hold all 24 bits at any scale but cost
// six products and 11 instead of 4 VALU instructions per pair split: 120 us
// where this form takes 83 us for trees of 64 over 2048 positions, 64 sequences.)  fp16's
// range is narrow, so operands are scaled by powers of two first, which is exact:
//   Q   each row to a maximum in [2^11, 2^12);
//   K   the range's first tile to [2^8, 2^9), the later ones by the same factor; its
//       inverse and Q's join the exponential's fused multiply-add;
//   P   e^(s - m) by 2^12, m lagging by 2^3 at most: up to 2^15;
//   V   each dimension of the first tile to [2^8, 2^9), the later ones likewise.
// What is small beside those maxima keeps an absolute error: 2^-25 scaled, 2^-33 of
// the first tile's largest |K| or of a dimension's largest |V| there, 2^-37 of a row's
// largest probability.  Where that might show, a wave takes its range again with
// float products: after a |K| or a query (in log2 units) of 2^12 or more, a
// scaled K or V of 2^15 or more, an infinity (or, among the nodes, a NaN)
// in V, or where in some dimension the largest |V| is more than 2^10 times the
// largest of some four to eight positions (not all 0).  And where the absolute
// errors of K (2^-25 over its factor) and of Q (2^-36 of the row's maximum) can move
// a score by more than kMostError: sum_d |q_d| 2^-25 / factor + HD max|q| 2^-36
// max|K|, a bound that all errors of one sign would reach (a key dimension of
// 4000 beside others of 0.003, queries of 333: 9e-5 in the output without the
// rule, 8e-7 with it).  And where a row's output is small beside the values that
// it is made of, below kLeastOut of each dimension's largest |V| in the root mean
// square: V's errors are 2^-21 of it there, P's of n positions sqrt(n) 2^-25 (a
// position with values 1e-5 of the others' that takes all of the attention: up to
// 6e-4 without the rule and P by 2^7).  Outputs that cancel to 1/sqrt(n) of
// N(0, 1) values stay above it up to half a million positions.
//
// A workgroup's four waves are RW blocks of 32 query rows times PW = 4 / RW tiles
// of 32 positions; K and V of the PW tiles are split once by the workgroup and
// kept in LDS in operand order:
//   S^T = K Q^T    A = K: lane l position l % 32, dimensions 16 s + 8 (l / 32) ..
//                  + 7 of k step s; B = Q, split once, in registers.
//   O^T = V^T P^T  the accumulators of S^T are the B operand: element j of k
//                  step t, lane half h, is register 8 t + j, position 8 (2 t +
//                  j / 4) + 4 h + j % 4, and V is laid out to match.
// Measured (8/2 heads of 64): 64 trees of 64 over 2048 positions 83 us, 182
// TFLOP/s of float products (the matrix cores 32 % busy; exponentials and
// splitting beside them); 64 of 16 over 1024 27 us; two of 32 over 32768 32 us,
// 64 MB at 2.1 TB/s.  The rules for taking a range again cost 2 % of a call (64
// shuffles at its end); where every range is taken again the three calls of those
// shapes take 847 instead of 155, 157 instead of 55 and 233 instead of 50 us.
typedef _Float16 hx2 __attribute__((ext_vector_type(2)));
typedef _Float16 hx8 __attribute__((ext_vector_type(8)));
typedef float fx2 __attribute__((ext_vector_type(2)));

template <int HD> struct SplitShape {
    static constexpr int KS = (HD + 15) / 16, DB = (HD + 31) / 32;
    static constexpr int KB = 2 * KS * 1024, VB = 2 * 2 * DB * 1024;   // bytes per 32 positions
};

struct Halves {
    ux4 t[2];   // high and low terms of eight floats
};
__device__ __forceinline__ Halves halve8(const float (&x)[8], float scale) {
    Halves f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = x[2 * i], b = x[2 * i + 1];
        const hx2 h = __builtin_convertvector((fx2){a * scale, b * scale}, hx2);
        // (scale a power of two: one rounding, to an exact difference; v_fma_mix_f32)
        const hx2 l = __builtin_convertvector(
            (fx2){fmaf(a, scale, -(float)h[0]), fmaf(b, scale, -(float)h[1])}, hx2);
        f.t[0][i] = __builtin_bit_cast(unsigned, h);
        f.t[1][i] = __builtin_bit_cast(unsigned, l);
    }
    return f;
}
__device__ __forceinline__ fx16 mma16(ux4 a, ux4 b, fx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(hx8, a),
                                                  __builtin_bit_cast(hx8, b), c, 0, 0, 0);
}
// c += the product of two split operands, the small terms first.
__device__ __forceinline__ fx16 mma_halves(const ux4 (&a)[2], const Halves &b, fx16 c) {
    c = mma16(a[1], b.t[0], c);
    c = mma16(a[0], b.t[1], c);
    return mma16(a[0], b.t[0], c);
}
// Binary exponent of a finite |x| (its bits): floor(log2), -127 for subnormals.
__device__ __forceinline__ int expo(unsigned bits) { return (int)(bits >> 23) - 127; }
__device__ __forceinline__ float pow2(int e) {   // -126 <= e <= 127
    return __uint_as_float((unsigned)(e + 127) << 23);
}

template <int HD, int RW>
__global__ __launch_bounds__(256, 2) void tree_attn_split_kernel(TreeArgs a, int blocks) {
    constexpr int PW = 4 / RW, KS = SplitShape<HD>::KS, DB = SplitShape<HD>::DB;
    constexpr int KB = SplitShape<HD>::KB, VB = SplitShape<HD>::VB;
    constexpr int KI = (64 * KS * PW + 255) / 256, VI = (128 * DB * PW + 255) / 256;   // items per thread
    constexpr int LDO = 32 * DB + 4;
    constexpr int STAGE = PW * (KB + VB), MERGE = PW > 1 ? RW * 32 * LDO * 4 : 0;
    __shared__ __align__(16) char sm[STAGE > MERGE ? STAGE : MERGE];
    __shared__ float sm_m[4][32], sm_l[4][32];
    // Of the first tiles: the largest |K|, and |V| by dimension (bits).  Over
    // the range: the largest |V| and the least of any eight positions' largest
    // by dimension, and whether a key or value was out of range.
    constexpr int DV = 32 * DB;
    __shared__ unsigned sm_maxk[PW], sm_maxv[PW][DV], sm_most[PW][DV], sm_least[PW][DV];
    __shared__ unsigned sm_mostk;   // the range's largest |K|
    __shared__ float sm_qsum[4][32], sm_qmax[4][32];   // of the waves' rows: sum |q|, max |q|
    __shared__ int sm_odd;
    // Every eighth workgroup runs on one XCD: it takes an eighth of the
    // (sequence, kv head, split) triples, with all row blocks of each.
    const int triples = a.seqs * a.nkv * a.splits;
    const int slot = blockIdx.x >> 3, rb = slot % blocks;
    const int id = (blockIdx.x & 7) * ((triples + 7) / 8) + slot / blocks;
    if (slot / blocks >= (triples + 7) / 8 || id >= triples) return;
    const int sp = id % a.splits, bk = id / a.splits;
    const int kvh = bk % a.nkv, b = bk / a.nkv;
    const int N = a.N, G = a.nh / a.nkv, rows = N * G;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5;
    const int rw = wave % RW, pw = wave / RW;

    const int pos = __builtin_amdgcn_readfirstlane(a.pos[b]);
    const Node node = tree_node(lane < N ? a.parent[(size_t)b * N + lane] : -2, lane, 0, lane < N);
    const int np = node_pos(node, pos, a.max_seq);
    const unsigned long long live = __ballot(lane < N && np >= 0);
    if (!live) return;

    // Tiles of 32: 0 .. nct - 1 cached positions, the others nodes; this split
    // takes t0 .. t1 - 1, PW at a time.
    const int nct = (pos + 31) / 32, nt = nct + (N + 31) / 32;
    const int t0 = (int)((long long)nt * sp / a.splits), t1 = (int)((long long)nt * (sp + 1) / a.splits);
    const size_t cache0 = (size_t)b * a.max_seq * a.kd + kvh * HD;
    const size_t draft0 = (size_t)b * N * a.kd + kvh * HD;
    struct Tile {
        const float *k, *v;
        unsigned in;   // bit j: position j of the tile counts
        int p0, n;     // first node or position, how many
        bool draft;
    };
    auto tile_at = [&](int t) {
        Tile x;
        const int u = min(t, nt - 1);
        x.draft = u >= nct;
        x.p0 = 32 * (x.draft ? u - nct : u);
        x.n = min(32, (x.draft ? N : pos) - x.p0);
        x.in = x.draft ? (unsigned)(live >> x.p0) : x.n == 32 ? ~0u : (1u << x.n) - 1;
        if (t >= t1) x.in = 0;
        x.k = (x.draft ? a.kd_out + draft0 : a.kc + cache0) + (size_t)x.p0 * a.kd;
        x.v = (x.draft ? a.vd_out + draft0 : a.vc + cache0) + (size_t)x.p0 * a.kd;
        return x;
    };

    // Item i of a thread: K: position j, dimensions 8 c .. + 7 of tile w; V:
    // dimension d of the eight positions of (k step, half) th of tile w.
    // Offsets into a tile; dimensions past HD read the row's first and count as 0.
    auto item = [&](int i, int per, int &rest) {   // tile of item i, and the item within it
        const int idx = tid + 256 * i;
        if (per == 256) { rest = tid; return i; }
        rest = idx % per;
        return idx / per;
    };
    // Loads run two steps ahead, in two sets of registers.
    float kr[2][KI][8], vr[2][VI][8];
    unsigned koff[KI], voff[VI];
#pragma unroll
    for (int i = 0; i < KI; ++i) {
        int k;
        item(i, 64 * KS, k);
        koff[i] = (k & 31) * a.kd + 8 * (k >> 5);
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
        int k;
        item(i, 128 * DB, k);
        const int d = k % (32 * DB), th = k / (32 * DB);
        voff[i] = (16 * (th >> 1) + 4 * (th & 1)) * a.kd + (d < HD ? d : 0);
    }
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    auto load = [&](auto set, int t) {
        float (&kr_)[KI][8] = kr[decltype(set)::value], (&vr_)[VI][8] = vr[decltype(set)::value];
#pragma unroll
        for (int i = 0; i < KI; ++i) {
            int k;
            const int w = item(i, 64 * KS, k);
            if (64 * KS * PW % 256 && w >= PW) break;
            const Tile x = tile_at(t + w);
            const int j = k & 31, d0 = 8 * (k >> 5);
            if (x.in == ~0u) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (HD % 16 && d0 >= HD) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) kr_[i][4 * h + e] = 0.0f;
                        continue;
                    }
                    const fx4 v = *reinterpret_cast<const fx4 *>(x.k + koff[i] + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) kr_[i][4 * h + e] = v[e];
                }
            } else {
                const bool ok = x.in >> j & 1 && d0 < HD;
                const float *p = x.k + (ok ? koff[i] : 0);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const fx4 v = *reinterpret_cast<const fx4 *>(p + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) kr_[i][4 * h + e] = ok ? v[e] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < VI; ++i) {
            int k;
            const int w = item(i, 128 * DB, k);
            if (128 * DB * PW % 256 && w >= PW) break;
            const Tile x = tile_at(t + w);
            const int d = k % (32 * DB), th = k / (32 * DB);
            if (x.in == ~0u) {
#pragma unroll
                for (int e = 0; e < 8; ++e) vr_[i][e] = (x.v + (8 * (e >> 2) + (e & 3)) * a.kd)[voff[i]];
                if (HD % 32 && d >= HD)
#pragma unroll
                    for (int e = 0; e < 8; ++e) vr_[i][e] = 0.0f;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int j = 8 * (2 * (th >> 1) + (e >> 2)) + 4 * (th & 1) + (e & 3);
                    const bool ok = x.in >> j & 1 && d < HD;
                    const float v = x.v[ok ? voff[i] + (8 * (e >> 2) + (e & 3)) * a.kd : 0];
                    vr_[i][e] = ok ? v : 0.0f;
                }
            }
        }
    };
    auto largest = [&](const float (&x)[8]) {
        float u = fmaxf(fabsf(x[0]), fabsf(x[1]));
#pragma unroll
        for (int e = 2; e < 8; ++e) u = fmaxf(u, fabsf(x[e]));
        return u;
    };
    float sk[PW], sv[VI];             // factors of K by tile, of V by item
    float tk[PW], tv[VI];             // what is not below these is out of range
    float vmost[VI], vleast[VI];      // the item's largest |V| over the range, and the least but 0
    float kmost = 0.0f;               // the largest |K| of the range
    bool out = false;                 // a key or value was out of range
#pragma unroll
    for (int i = 0; i < VI; ++i) { vmost[i] = 0.0f; vleast[i] = INFINITY; }
    // The largest |V| of an item's positions as it counts for the range: few
    // positions are small together by chance: two or three count from 2^14
    // on, one from 2^20.
    auto check = [&](auto set, int t) {   // (t: the set's tiles)
#pragma unroll
        for (int i = 0; i < KI; ++i) {
            int k;
            const int w = item(i, 64 * KS, k);
            if (64 * KS * PW % 256 && w >= PW) break;
            const float top = largest(kr[decltype(set)::value][i]);
            kmost = fmaxf(kmost, top);
            out |= top >= (PW > 1 && w ? tk[PW - 1] : tk[0]);
        }
#pragma unroll
        for (int i = 0; i < VI; ++i) {
            int k;
            const int w = item(i, 128 * DB, k);
            if (128 * DB * PW % 256 && w >= PW) break;
            const float (&x)[8] = vr[decltype(set)::value][i];
            float top = largest(x);
            bool odd = top >= tv[i];
            vmost[i] = fmaxf(vmost[i], top);
            const Tile y = tile_at(t + w);
            if (y.in != ~0u) {
                const int n = __popc(y.in >> (16 * (k / (64 * DB)) + 4 * (k / (32 * DB) & 1)) & 0x0f0fu);
                top *= n >= 4 ? 1.0f : n >= 2 ? 0x1p4f : 0x1p10f;
            }
            vleast[i] = fminf(vleast[i], top > 0.0f ? top : INFINITY);
            if (y.draft) {
                float chk = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) chk = fmaf(x[e], 0.0f, chk);
                odd |= chk != 0.0f;
            }
            out |= odd;
        }
    };
    auto store = [&](auto set) {
#pragma unroll
        for (int i = 0; i < KI; ++i) {
            int k;
            const int w = item(i, 64 * KS, k);
            if (64 * KS * PW % 256 && w >= PW) break;
            const int j = k & 31, c = k >> 5;
            const Halves f = halve8(kr[decltype(set)::value][i], PW > 1 && w ? sk[PW - 1] : sk[0]);
            char *p = sm + w * (KB + VB) + (c >> 1) * 1024 + (j + 32 * (c & 1)) * 16;
#pragma unroll
            for (int q = 0; q < 2; ++q) *reinterpret_cast<ux4 *>(p + q * KS * 1024) = f.t[q];
        }
#pragma unroll
        for (int i = 0; i < VI; ++i) {
            int k;
            const int w = item(i, 128 * DB, k);
            if (128 * DB * PW % 256 && w >= PW) break;
            const int d = k % (32 * DB), th = k / (32 * DB);
            const Halves f = halve8(vr[decltype(set)::value][i], sv[i]);
            char *p = sm + w * (KB + VB) + KB + ((d >> 5) * 2 + (th >> 1)) * 1024 + ((d & 31) + 32 * (th & 1)) * 16;
#pragma unroll
            for (int q = 0; q < 2; ++q) *reinterpret_cast<ux4 *>(p + q * 2 * DB * 1024) = f.t[q];
        }
    };
    if (tid < PW) sm_maxk[tid] = 0;
    if (tid == 0) sm_odd = 0, sm_mostk = 0;
    for (int i = tid; i < PW * DV; i += 256) {
        sm_maxv[i / DV][i % DV] = sm_most[i / DV][i % DV] = 0;
        sm_least[i / DV][i % DV] = ~0u;
    }
    __syncthreads();
    load(S0{}, t0);
    if (t0 + PW < t1) load(S1{}, t0 + PW);

    // The lane's query row (past the last one: that row again), scores in
    // log2 units; qs undoes the row's factor.  Rows of nodes that are no token
    // (whatever the workspace holds) have no say in the wave's decisions: they
    // do not count for its range, and their maximum starts at infinity, which no
    // score passes.
    const int r = (rb * RW + rw) * 32 + li, rq = min(r, rows - 1), qn = rq / G;
    const float *qrow = a.q + ((size_t)b * N + qn) * a.qd + (kvh * G + rq % G) * HD;
    const unsigned long long anc = (unsigned long long)__shfl((unsigned)(node.anc >> 32), qn) << 32 |
                                   (unsigned)__shfl((unsigned)node.anc, qn);
    const bool token = live >> qn & 1;
    const float scale = a.scale * 1.4426950408889634f;
    Halves fq[KS];
    float qs;
    bool odd;   // the wave's range is to be taken again
    {
        float v[KS][8];
        unsigned u = 0;
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int d0 = 16 * s + 8 * lh + 4 * i;
                const bool in = d0 < HD;
                const fx4 x = *reinterpret_cast<const fx4 *>(qrow + (in ? d0 : 0));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = in ? x[e] * scale : 0.0f;
                    v[s][4 * i + e] = y;
                    u = max(u, __float_as_uint(y) & 0x7fffffffu);
                    sum += fabsf(y);
                }
            }
        sum += __shfl_xor(sum, 32);
        u = max(u, (unsigned)__shfl_xor(u, 32));
        if (lh == 0) {
            sm_qsum[wave][li] = sum;
            sm_qmax[wave][li] = __uint_as_float(u);
        }
        odd = __any(token && u >= __float_as_uint(kMostKey));
        const int e = min(11 - expo(u), 126);
#pragma unroll
        for (int s = 0; s < KS; ++s) fq[s] = halve8(v[s], pow2(e));
        qs = pow2(-e);
    }

    float m = token ? kLow : INFINITY, l = 0.0f;
    fx16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
    auto of_dim = [&](float x, int d, int e) {   // lane (dimension of register e of o[d])'s x
        return __shfl(x, 32 * d + 8 * (e >> 2) + 4 * lh + (e & 3));
    };
    // The factors, from the first tiles' maxima.
#pragma unroll
    for (int i = 0; i < KI; ++i) {
        int k;
        const int w = item(i, 64 * KS, k);
        if (64 * KS * PW % 256 && w >= PW) break;
        const float u = wave_max(largest(kr[0][i]));
        if (lane == 0) atomicMax(&sm_maxk[w], __float_as_uint(u));
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
        int k;
        const int w = item(i, 128 * DB, k);
        if (128 * DB * PW % 256 && w >= PW) break;
        atomicMax(&sm_maxv[w][k % DV], __float_as_uint(largest(vr[0][i])));
    }
    __syncthreads();
    // 2^e for a maximum of u (0: fill's instead).
    auto factor = [&](unsigned u, unsigned fill) {
        u = u ? u : fill;
        return u ? min(8 - expo(u), 126) : 8;
    };
    auto bound = [&](int e) { return 15 - e > 127 ? INFINITY : pow2(15 - e); };
    unsigned fill[PW];
    float ik = 1.0f;   // undoes the factor of the wave's own K
#pragma unroll
    for (int w = 0; w < PW; ++w) {
        const int e = factor(sm_maxk[w], 0);
        sk[w] = pow2(e);
        tk[w] = fminf(kMostKey, bound(e));
        if (w == pw) ik = pow2(-e);
        fill[w] = __float_as_uint(wave_max(__uint_as_float(sm_maxv[w][lane % DV])));
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
        int k;
        const int w = item(i, 128 * DB, k);
        if (128 * DB * PW % 256 && w >= PW) break;
        const int e = factor(sm_maxv[w][k % DV], PW > 1 && w ? fill[PW - 1] : fill[0]);
        sv[i] = pow2(e);
        tv[i] = bound(e);
    }
    int le = factor(sm_maxv[pw][lane % DV], PW > 1 && pw ? fill[PW - 1] : fill[0]);   // of dimension `lane`
    const float fac0 = ik * qs;
    float one = 1.0f;
    asm("" : "+s"(one));   // (a factor that the compiler does not see through)

    auto step = [&](auto set, int t) {
        __syncthreads();   // (the last tiles are read)
        check(set, t);
        store(set);
        if (t + 2 * PW < t1) load(set, t + 2 * PW);
        __syncthreads();
        const char *kp = sm + pw * (KB + VB) + lane * 16, *vp = kp + KB;
        const Tile x = tile_at(t + pw);
        // Of the SIMD's two waves the one at its products goes first, the other's
        // exponentials and splits fill in (64 trees of 64: 85 us without, 80).
        __builtin_amdgcn_s_setprio(1);
        fx16 s;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const ux4 fk[2] = {*reinterpret_cast<const ux4 *>(kp + i * 1024),
                               *reinterpret_cast<const ux4 *>(kp + (KS + i) * 1024)};
            s = mma_halves(fk, fq[i], s);
        }
        __builtin_amdgcn_s_setprio(0);
        float fac = fac0;
        // Register e: position 8 (e / 4) + 4 lh + e % 4.
        if (x.in != ~0u || x.draft) {
            const unsigned see = (x.draft ? x.in & (unsigned)(anc >> x.p0) : x.in) >> (4 * lh);
#pragma unroll
            for (int e = 0; e < 16; ++e)
                s[e] = see >> (8 * (e >> 2) + (e & 3)) & 1 ? s[e] * fac : -INFINITY;
            fac = 1.0f;
        }
        float top = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
        top *= fac;
        if (__any(top - m > kSplitSlack)) {
            const float y = fmaxf(fmaxf(top, __shfl_xor(top, 32)) - kSplitLift, m);
            const float f = __builtin_amdgcn_exp2f(m - y);
            m = y;
            l *= f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= f;
        }
        float p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            p[e] = __builtin_amdgcn_exp2f(fmaf(s[e], fac, -m));
            l += p[e];
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const Halves fp = halve8({p[8 * i], p[8 * i + 1], p[8 * i + 2], p[8 * i + 3], p[8 * i + 4],
                                      p[8 * i + 5], p[8 * i + 6], p[8 * i + 7]}, one);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const ux4 fv[2] = {*reinterpret_cast<const ux4 *>(vp + (2 * d + i) * 1024),
                                   *reinterpret_cast<const ux4 *>(vp + (2 * DB + 2 * d + i) * 1024)};
                o[d] = mma_halves(fv, fp, o[d]);
            }
        }
        __builtin_amdgcn_s_setprio(0);
    };
    for (int t = t0; t < t1; t += 2 * PW) {
        step(S0{}, t);
        if (t + PW < t1) step(S1{}, t + PW);
    }

    // Was everything within the split's range?
#pragma unroll
    for (int i = 0; i < VI; ++i) {
        int k;
        const int w = item(i, 128 * DB, k);
        if (128 * DB * PW % 256 && w >= PW) break;
        atomicMax(&sm_most[w][k % DV], __float_as_uint(vmost[i]));
        atomicMin(&sm_least[w][k % DV], __float_as_uint(vleast[i]));
    }
    kmost = wave_max(kmost);
    if (lane == 0) atomicMax(&sm_mostk, __float_as_uint(kmost));
    if (out) sm_odd = 1;
    __syncthreads();
    {
        const float ek = sm_qsum[wave][li] * pow2(max(-25 - factor(sm_maxk[pw], 0), -126));
        const float eq = sm_qmax[wave][li] * (HD * 0x1p-36f) * __uint_as_float(sm_mostk);
        odd |= __any(token && !(ek + eq <= kMostError));
        const unsigned most = sm_most[pw][lane % DV], least = sm_least[pw][lane % DV];
        odd |= sm_odd || __any(most && expo(most) - expo(least) > 10);
        const float g = most ? pow2(min(max(-le - expo(most), -126), 127)) : 0.0f;
        float ss = 0.0f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float y = o[d][e] * of_dim(g, d, e);
                ss = fmaf(y, y, ss);
            }
        ss += __shfl_xor(ss, 32);
        const float sum = (l + __shfl_xor(l, 32)) * kLeastOut;
        odd |= __any(token && ss < __popcll(__ballot(most && lane < DV)) * (sum * sum));
    }
    if (odd) {
        // Float products (v_mfma_f32_32x32x2_f32), by each wave for itself,
        // straight from memory.  Infinities and NaN of V are added where they
        // are seen.
        m = kLow;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
        // V's own factor per dimension, so that no sum passes the float range.
        le = 12 - min(max(expo(sm_most[pw][lane % DV]), -114), 127);
        float fv[DB];   // of dimension 32 d + li
#pragma unroll
        for (int d = 0; d < DB; ++d) fv[d] = __shfl(pow2(le), 32 * d + li);
#pragma unroll 1
        for (int t = t0 + pw; t < t1; t += PW) {
            const Tile x = tile_at(t);
            const bool mine = x.in >> li & 1;
            const float *kk = x.k + (mine ? li : 0) * a.kd;
            fx16 s;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll 1
            for (int d = lh; d < HD; d += 2)
                s = __builtin_amdgcn_mfma_f32_32x32x2f32(mine ? kk[d] : 0.0f, qrow[d] * scale, s, 0, 0, 0);
            const unsigned see = (x.draft ? x.in & (unsigned)(anc >> x.p0) : x.in) >> (4 * lh);
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = see >> (8 * (e >> 2) + (e & 3)) & 1 ? s[e] : -INFINITY;
                top = fmaxf(top, s[e]);
            }
            top = fmaxf(fmaxf(top, __shfl_xor(top, 32)), m);
            const float f = __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= f;
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = __builtin_amdgcn_exp2f(s[e] - m);
                l += s[e];
                const int j = 8 * (e >> 2) + 4 * lh + (e & 3);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const int dim = 32 * d + li;
                    const bool ok = x.in >> j & 1 && dim < HD;
                    const float v = x.v[ok ? (unsigned)(j * a.kd + dim) : 0u];
                    const bool fine = fabsf(v) < INFINITY;
                    bad |= ok && !fine;
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(ok && fine ? v * fv[d] : 0.0f,
                                                                s[e], o[d], 0, 0, 0);
                }
            }
            if (__any(bad))
#pragma unroll 1
                for (int j = 0; j < x.n; ++j) {
                    float pr = s[0];
#pragma unroll
                    for (int e = 1; e < 16; ++e)
                        if (4 * (j >> 3) + (j & 3) == e) pr = s[e];
                    const float pj = __shfl(pr, li + 32 * (j >> 2 & 1));
                    const bool seen = x.in >> j & 1 && (!x.draft || anc >> (x.p0 + j) & 1);
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int dim = 32 * d + 8 * (e >> 2) + 4 * lh + (e & 3);
                            const float v = x.v[(unsigned)(j * a.kd + (dim < HD ? dim : 0))];
                            if (seen && dim < HD && !(fabsf(v) < INFINITY)) o[d][e] += pj * v;
                        }
                }
        }
    }
    l += __shfl_xor(l, 32);
    {   // the normalised output, then V's own scale
        const float inv = PW == 1 && a.splits == 1 ? 1.0f / l : part_inv(l);
        const float f = pow2(-le);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * inv * of_dim(f, d, i);
    }

    // Registers e of o[d]: dimension 32 d + 8 (e / 4) + 4 lh + e % 4.
    auto put = [&]() {
        if (r >= rows) return;
        float *dst = a.splits == 1
            ? a.o + ((size_t)b * N + r / G) * a.qd + (kvh * G + r % G) * HD
            : a.part + (((size_t)bk * rows + r) * a.splits + sp) * (HD + 2) + 2;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int dim = 32 * d + 8 * (e >> 2) + 4 * lh + (e & 3);
                if (dim < HD) dst[dim] = o[d][e];
            }
        if (a.splits > 1 && lh == 0) {
            dst[-2] = m;
            dst[-1] = l;
        }
    };
    if constexpr (PW > 1) {
        // The position waves' outputs, in wave order.
        float *buf = reinterpret_cast<float *>(sm) + (size_t)rw * 32 * LDO + li * LDO;
        for (int w = 1; w < PW; ++w) {
            __syncthreads();
            if (pw == w) {
                if (lh == 0) {
                    sm_m[rw][li] = m;
                    sm_l[rw][li] = l;
                }
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<fx4 *>(buf + 32 * d + 2 * e + 4 * lh) = fx4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
            }
            __syncthreads();
            if (pw == 0) {
                const float m2 = sm_m[rw][li], y = fmaxf(m, m2);
                const float l1 = __builtin_amdgcn_exp2f(m - y) * l;
                const float l2 = __builtin_amdgcn_exp2f(m2 - y) * sm_l[rw][li];
                m = y;
                l = l1 + l2;
                const float inv = a.splits == 1 ? 1.0f / l : part_inv(l);
                const float f1 = l1 * inv, f2 = l2 * inv;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        o[d][e] = fmaf(f2, buf[32 * d + 8 * (e >> 2) + 4 * lh + (e & 3)], o[d][e] * f1);
            }
        }
        if (pw) return;
    }
    put();
}

// Joins the splits' partials.  A workgroup per query row, W waves: lane l holds
// the weights of splits l and l + 64 (kMaxSplits of them), lane d then sums
// dimension d over every W-th split, eight loads at a time, and the waves' sums are
// added in wave order.
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
    constexpr int W = 4;
    __shared__ float sm[W][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t row = blockIdx.x;   // (kv head of a sequence) rows + r
    const int G = a.nh / a.nkv, rows = a.N * G, hd = a.hd, S = a.splits;
    const int r = (int)(row % rows), kvh = (int)(row / rows % a.nkv);
    const size_t xrow = row / rows / a.nkv * a.N + r / G;
    if (a.row_p[xrow] < 0) return;
    const float *pp = a.part + row * S * (hd + 2);
    float m[2], w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const bool in = lane + 64 * h < S;
        const float *ps = pp + (size_t)(in ? lane + 64 * h : 0) * (hd + 2);
        m[h] = in ? ps[0] : kLow;
        w[h] = in ? ps[1] : 0.0f;
    }
    const float M = wave_max(fmaxf(m[0], m[1]));
#pragma unroll
    for (int h = 0; h < 2; ++h) w[h] *= __builtin_amdgcn_exp2f(m[h] - M);
    const float inv = 1.0f / wave_sum(w[0] + w[1]);
    w[0] *= inv;
    w[1] *= inv;
    const int d = min(lane, hd - 1);
    float O = 0.0f;
    for (int s0 = wave; s0 < S; s0 += 8 * W) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = pp[(size_t)min(s0 + u * W, S - 1) * (hd + 2) + 2 + d];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int s = s0 + u * W;
            if (s < S) O = fmaf(lane_of(s < 64 ? w[0] : w[1], s & 63), v[u], O);
        }
    }
    sm[wave][lane] = O;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int u = 1; u < W; ++u) O += sm[u][lane];
    if (lane < hd) a.o[xrow * a.qd + (kvh * G + r % G) * hd + lane] = O;
}

// The same for up to NS <= 8 splits, of many rows mostly: hd / 4 threads take a
// row, four dimensions each, and read every split's m and l themselves (64 trees
// of 64, two splits: 6.2 us, 4 TB/s; a wave per row 15.6).
template <int NS>
__global__ __launch_bounds__(256) void tree_merge_few_kernel(TreeArgs a, int blocks) {
    const int G = a.nh / a.nkv, rows = a.N * G, hd = a.hd, S = a.splits, per = hd / 4;
    const int pair = blockIdx.x / blocks;   // kv head of a sequence
    const int i = (blockIdx.x - pair * blocks) * 256 + threadIdx.x;
    const int r = i / per, d = 4 * (i - r * per);
    if (r >= rows) return;
    const int node = r / G, seq = pair / a.nkv, kvh = pair - seq * a.nkv;
    const size_t xrow = (size_t)seq * a.N + node;
    const float *pp = a.part + ((size_t)pair * rows + r) * S * (hd + 2);
    const bool live = a.row_p[xrow] >= 0;
    float2 ml[NS], v[NS][2];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const float *ps = pp + (size_t)min(s, S - 1) * (hd + 2);
        ml[s] = *reinterpret_cast<const float2 *>(ps);
        v[s][0] = *reinterpret_cast<const float2 *>(ps + 2 + d);
        v[s][1] = *reinterpret_cast<const float2 *>(ps + 4 + d);
    }
    if (!live) return;
    float M = kLow, L = 0.0f, w[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) M = fmaxf(M, ml[s].x);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        w[s] = s < S ? __builtin_amdgcn_exp2f(ml[s].x - M) * ml[s].y : 0.0f;
        L += w[s];
    }
    L = 1.0f / L;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        if (s >= S) break;
        const float f = w[s] * L;
        o.x = fmaf(f, v[s][0].x, o.x);
        o.y = fmaf(f, v[s][0].y, o.y);
        o.z = fmaf(f, v[s][1].x, o.z);
        o.w = fmaf(f, v[s][1].y, o.w);
    }
    *reinterpret_cast<float4 *>(a.o + xrow * a.qd + (kvh * G + r - node * G) * hd + d) = o;
}

template <int HD> void launch_qt(const TreeArgs &a, const TreePlan &p, hipStream_t s) {
    const size_t triples = (size_t)a.seqs * a.nkv * p.splits;
    const dim3 grid((unsigned)(triples * p.blocks)), grid8((unsigned)((triples + 7) / 8 * 8 * p.blocks)), wg(256);
    if (p.rows == 16)      hipLaunchKernelGGL((tree_attn_kernel<HD, 1>), grid, wg, 0, s, a, p.blocks);
    else if (p.rows == 32) hipLaunchKernelGGL((tree_attn_kernel<HD, 2>), grid, wg, 0, s, a, p.blocks);
    else if (p.rows == 64) hipLaunchKernelGGL((tree_attn_split_kernel<HD, 2>), grid8, wg, 0, s, a, p.blocks);
    else                   hipLaunchKernelGGL((tree_attn_split_kernel<HD, 4>), grid8, wg, 0, s, a, p.blocks);
}

template <bool QKV> void launch_proj_mma(const TreeArgs &a, int NC, hipStream_t s) {
    const int M = QKV ? a.d : a.qd, t64 = (NC + 63) / 64, t128 = (NC + 127) / 128;
    const long long cus = device_cus();
    auto groups = [&](int rows, int tiles) { return (long long)((a.B + rows - 1) / rows) * tiles; };
    auto grid = [&](int rows, int tiles) { return dim3((unsigned)(((a.B + 8 * rows - 1) / (8 * rows)) * 8 * tiles)); };
    // The larger the tile, the fewer times X is split and W read; 64 x 128
    // takes a CU to itself, so its rounds have to be full.  us per sublayer with
    // 32 x 64, 32 x 128, 64 x 128, and by this rule (launch by launch): d = 512
    // (8/2 heads of 64), 512 rows 27.2 32.9 45.5 26.9, 1024 34.5 36.2 48.7 32.9,
    // 4096 75.2 68.7 74.6 66.9; d = 1024 (16/4 heads), 1024 rows 81.3 73.6 75.8
    // 67.8, 2048 152 124 125 125, 4096 237 187 167 167; d = 2048 (16/4), 1024 rows
    // 149 129 100 100.
    const long long big = groups(64, t128), rounds = (big + cus - 1) / cus;
    if (8 * big >= (M >= 1024 ? 6 : 7) * cus * rounds)
        hipLaunchKernelGGL((proj_mma_kernel<QKV, 2, 4>), grid(64, t128), dim3(256), 0, s, a, t128);
    else if (4 * groups(32, t128) >= 3 * cus)
        hipLaunchKernelGGL((proj_mma_kernel<QKV, 1, 4>), grid(32, t128), dim3(256), 0, s, a, t128);
    else
        hipLaunchKernelGGL((proj_mma_kernel<QKV, 1, 2>), grid(32, t64), dim3(256), 0, s, a, t64);
}

}  // namespace

size_t split_weight_bytes(int K, int N) {
    return (size_t)((N + 31) / 32) * ((K + 15) / 16) * 3 * 1024;
}

hipError_t launch_pack_split(const float *src, unsigned short *dst, int K, int N, int col0,
                             unsigned *range, hipStream_t s) {
    if (K <= 0 || N <= 0) return hipErrorInvalidValue;
    const size_t n = (size_t)((K + 7) / 8) * N;
    hipLaunchKernelGGL(pack_split_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, src,
                       dst, K, N, col0, range);
    return hipGetLastError();
}

TreePlan tree_plan(int seqs, int N, int nh, int nkv, int hd, int max_seq) {
    TreePlan p{};
    const int rows = N * (nh / nkv);
    // Query rows per block: all of them share one read of a tile, as far as 128
    // (from 33 on split, tree_attn_split_kernel), unless the whole call is
    // little: then it is the length of one wave's work that counts.  us per
    // sublayer with 16, 32, 64, 128 (heads of 64, 4 per kv head): one sequence
    // of 1024 positions, N = 8 20.1 22.5 23.9 23.7, N = 32 21.0 22.9 24.3 24.6; four
    // of 4096, N = 16 28.2 28.4 33.1 32.2, N = 32 36.5 38.3 38.6 39.0, N = 64 49.3
    // 49.6 46.2 43.1; 64 of 1024, N = 8 43.9 41.2 46.4 46.5, N = 16 66.3 50.7 51.1
    // 51.4, N = 32 115 85.4 70.1 65.8; 256 of 1024, N = 8 119 88.5 96.3 104.
    // Positions are counted as the cache's capacity: where the sequences are in it
    // is known to the device only.
    const bool little = (long long)seqs * nkv * rows * max_seq < kLittle;
    p.rows = rows <= 16 || little ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    p.blocks = (rows + p.rows - 1) / p.rows;
    const long long base = (long long)seqs * nkv * p.blocks;
    const long long tiles = (max_seq + 15) / 16 + (N + 15) / 16;
    // One workgroup per CU where a wave takes whole rows alone, two where four
    // share their tiles (their barriers leave gaps), a tile per wave at least.
    // us per sublayer by workgroups per CU, 1/2, 1, 2, 4 (d = 512, 8/2 heads of
    // 64): 64 sequences of 1024 positions, N = 1 27.8 29.2 30.3 34.4, N = 16 61.2
    // 51.5 51.0 64.0, N = 32 82.6 68.4 66.0 78.3; of 2048, N = 64 144 145 129 137;
    // one of 1024, N = 32 23.4 21.0 21.7 21.7.  By the splits allowed, 32, 64,
    // 128: one sequence of 32768, N = 32 65.2 45.8 38.1; of 65536, N = 16 83.0
    // 55.8 43.8.  A sequence at position 1000 takes 20.2 us in a cache of 1100,
    // 25.0 in one of 131072 (N = 8; N = 32 20.9 and 29.1): most of its 128 splits
    // are empty.
    const long long goal = (p.rows <= 32 ? 1LL : 2LL) * device_cus();
    const long long want = (goal + base - 1) / base, most = (tiles + kWaves - 1) / kWaves;
    p.splits = (int)std::max(1LL, std::min(std::min(want, most), (long long)kMaxSplits));
    p.part_floats = p.splits > 1 ? (size_t)seqs * nkv * rows * p.splits * (hd + 2) : 0;
    return p;
}

hipError_t launch_attn_tree(const TreeArgs &a, hipStream_t s) {
    if (a.B <= 0) return hipSuccess;
    const int gqa = a.nh / a.nkv;
    if (a.hd > 64 || a.hd % 8 || a.hd <= 0 || gqa > 8 || gqa < 1 || a.nh % a.nkv || a.d % 4 ||
        a.N < 1 || a.N > kTreeMaxNodes || a.B != a.seqs * a.N)
        return hipErrorInvalidValue;
    const TreePlan p = tree_plan(a.seqs, a.N, a.nh, a.nkv, a.hd, a.max_seq);
    if (p.splits != a.splits || (p.part_floats && !a.part)) return hipErrorInvalidValue;
    const int NC = a.qd + 2 * a.kd;
    auto t16 = [](int n) { return (unsigned)((n + kPT - 1) / kPT); };
    const bool small = a.B <= kPVRows, many = a.B > kTreeMmaRows && a.wqkv_s && a.wo_s;
    if (many)       launch_proj_mma<true>(a, NC, s);
    else if (small) hipLaunchKernelGGL((projv_kernel<true, TreeArgs>), dim3((unsigned)(NC / 4)), dim3(256), 0, s, a);
    else            hipLaunchKernelGGL((proj16_kernel<true, TreeArgs>), dim3(t16(NC), t16(a.B)), dim3(1024), 0, s, a);
    switch (a.hd) {
        case 8:  launch_qt<8>(a, p, s); break;
        case 16: launch_qt<16>(a, p, s); break;
        case 24: launch_qt<24>(a, p, s); break;
        case 32: launch_qt<32>(a, p, s); break;
        case 40: launch_qt<40>(a, p, s); break;
        case 48: launch_qt<48>(a, p, s); break;
        case 56: launch_qt<56>(a, p, s); break;
        default: launch_qt<64>(a, p, s); break;
    }
    if (p.splits > 8) {
        hipLaunchKernelGGL(tree_merge_kernel, dim3((unsigned)a.B * a.nh), dim3(256), 0, s, a);
    } else if (p.splits > 1) {
        const int blocks = (a.N * gqa * (a.hd / 4) + 255) / 256;
        const dim3 grid((unsigned)(a.seqs * a.nkv * blocks));
        if (p.splits == 2) hipLaunchKernelGGL(tree_merge_few_kernel<2>, grid, dim3(256), 0, s, a, blocks);
        else if (p.splits <= 4) hipLaunchKernelGGL(tree_merge_few_kernel<4>, grid, dim3(256), 0, s, a, blocks);
        else hipLaunchKernelGGL(tree_merge_few_kernel<8>, grid, dim3(256), 0, s, a, blocks);
    }
    if (many)       launch_proj_mma<false>(a, a.d, s);
    else if (small) hipLaunchKernelGGL((projv_kernel<false, TreeArgs>), dim3((unsigned)(a.d / 4)), dim3(256), 0, s, a);
    else            hipLaunchKernelGGL((proj16_kernel<false, TreeArgs>), dim3(t16(a.d), t16(a.B)), dim3(1024), 0, s, a);
    return hipGetLastError();
}

}  // namespace moe
