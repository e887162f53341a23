// tree_verify.hip — which drafted tokens a target model accepts, and the
// accepted tokens' keys and values into the caches, gfx950.
//
// Verification, sequence by sequence: p the target's distribution after a
// node, q the distribution its children were drawn from (independently), u
// given uniform numbers.  From the root (node 0), the children of the
// current node are tried in index order; child c with token t is accepted
// with probability min(1, p_j(t) / q(t)), where j counts the children
// rejected before it and p_0 = p, p_{j+1} = max(p_j - q, 0) normalised; the
// walk goes on from an accepted child, and when none is left the next token
// is drawn from p_j.  (Every token of the result is then distributed as the
// target's.)  The recursion closes: with p_j = r_j / W_j,
//   r_j = max(p - a_j q, 0),  W_j = sum r_j,  a_0 = 0, W_0 = 1,
//   max(r_j / W_j - q, 0) = max(p - a_j q - W_j q, 0) / W_j, so a_{j+1} = a_j + W_j:
// one number is the whole state, a rejection costs one pass over the two
// rows, and an acceptance (u q(t) W_j < r_j(t)) reads two floats.  Without q
// (drafts that were looked up: q is 1 at the child's token) r_{j+1} is r_j
// with that token taken out.
// Sums and cumulative sums are in 64 bits: the results are whole numbers that
// follow from comparing them, and in 32 bits they would hang on the order of
// summation.  Children have larger indices than their parent, so one pass
// over the nodes in index order is the whole walk.
//
// What it costs is reading rows: a CU takes 44 GB/s from memory, 23 us for the
// two rows of a pass over 131072 tokens (its 64-bit additions 8 us of them); the
// whole card 4 TB/s.  A sequence needs one pass for its last decision and one per
// rejection before it, one after the other.  So
//   - a row is cut into segments, a wave's work, and the first pass that a
//     sequence needs (everything before it is a few floats) is shared by `parts`
//     workgroups; the last of them to arrive walks on;
//   - it does so alone over short rows, and with the others' help over long
//     ones (verify_plan has both sides measured);
//   - with q, only tokens with p > a q can count in a later pass at the node (a
//     grows; at the second rejection one token in seven or so): a pass that
//     another of that workgroup's may follow leaves those in LDS, and later
//     passes read them there;
//   - without q, one pass leaves out the tokens of all the node's children and
//     the sum after each rejection is that plus the children's that are left
//     (no differences of nearly equal sums).
//   - the walk itself is a few instructions per child tried: every wave holds
//     the nodes, one per lane.
// Measured: 64 trees of 32 nodes over 131072 tokens 47-54 us (the last sequence's
// five passes, 5 us of reading and 3 us of handing over each; 79 us with the first
// pass shared only), 64 of 16 over 32768 23-26 us, one chain of 6 over 4096 7.5 us
// (the launch), 33 trees of 24 looked-up nodes over 50001 13 us.
#include "handoff.h"
#include "moe_internal.h"
#include "moe_math.h"
#include <algorithm>

namespace moe {
namespace {

constexpr int kMaxSegs = 512;     // segments of a row
constexpr int kListPairs = 19000; // pairs kept in LDS
constexpr int kListZero = kListPairs;     // behind them one that is zero, and one to write to that nobody reads
constexpr int kQuads = 4;         // float4s of a row that a lane has in flight

// Doubles across the wave.
// (rows of 16 lanes through DPP, then the rows)
template <int N> __device__ inline double shr0(double v) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)u, 0x110 + N, 0xF, 0xF, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), 0x110 + N, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ inline double lane64(double v, int l) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = __builtin_amdgcn_readlane((int)u, l);
    const unsigned hi = __builtin_amdgcn_readlane((int)(u >> 32), l);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ inline double wave_sum64(double v) {
    v += shr0<1>(v);
    v += shr0<2>(v);
    v += shr0<4>(v);
    v += shr0<8>(v);
    return (lane64(v, 15) + lane64(v, 31)) + (lane64(v, 47) + lane64(v, 63));
}
__device__ inline double wave_scan64(double v, int lane) {   // inclusive
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const double u = __shfl_up(v, s);
        if (lane >= s) v += u;
    }
    return v;
}
__device__ inline double wave_back_scan64(double v, int lane) {   // of the lane and those above
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const double u = __shfl_down(v, s);
        if (lane + s < 64) v += u;
    }
    return v;
}
// What is left of the target's distribution at one node: r(x) from p(x) and
// q(x); with q null p(x), less the tokens that gone holds.  No less than 0, and
// what is no number is 0; q likewise, so that r only falls as a grows.
struct Left {
    const float *p, *q;
    double a;
    const int *gone;
    int ngone;
};
__device__ inline double left_of(float p, float q, double a) {
    return fmax(fma(-a, (double)fmaxf(q, 0.0f), (double)p), 0.0);
}

struct VerifySmem {
    double seg[kMaxSegs];      // sums of the segments
    int off[kMaxSegs], cnt[kMaxSegs];   // their pairs in the list
    double total, after[64];
    int parent[64], token[64], gone[64], path[64];
    float u[64], pt[64], qt[64];
    bool first[64];            // no earlier child of the parent has the token
    int ngone, listed, flag, claimed;   // listed: pairs asked room for (more than there is: no list)
    unsigned mask;
    float2 list[kListPairs + 2];

    // The list's room where the lanes' words for segs segments stand behind it
    // (0: none do), and those words.
    __device__ static int room(int segs) { return kListPairs - 16 * segs; }
    __device__ unsigned short *lanes(int segs) { return reinterpret_cast<unsigned short *>(list + room(segs)); }
};

// Rows start at any float: four-byte aligned vector loads.
typedef float fx4u __attribute__((ext_vector_type(4), aligned(4)));

// Tokens x .. x + 3 of a row, 0 past the end.
__device__ inline fx4u load4(const float *row, unsigned x, unsigned V) {
    if (x + 4 <= V) return *reinterpret_cast<const fx4u *>(row + x);
    fx4u v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j = 0; j < 3; ++j)
        if (x + j < V) v[j] = row[x + j];
    return v;
}

__device__ inline void cstore64(unsigned long long *p, unsigned long long v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline unsigned long long cload64(const unsigned long long *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// sm.seg[s] for the segments s0 <= s < s1 (len tokens each); the caller's
// barrier follows.  A wave takes every WAVES-th segment, lane l the tokens 4 l .. + 3 of
// each 256; the next kQuads float4s of the rows are in flight while it adds:
// every load is unconditional (a lane past the row's end reads its last four
// tokens again and leaves out what is not its own; V >= 4), so that the waits are
// for the loads of a step and not for all.
// LIST (segments of kQuads float4s per lane at most): pairs with something left
// go to the list as well, if there is room; a segment's are together and in its
// lanes' order, where is a matter of timing and of no other consequence.
// LANES: where each lane's begin in its segment's and how many there are is kept
// too, in a word 32 begin + number (all the list's segments are s0 .. s1 - 1).
template <int WAVES, bool Q, bool LIST, bool LANES = false>
__device__ void sum_segs(const Left &f, int V, int len, int s0, int s1, VerifySmem &sm) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = len / (256 * kQuads);   // per segment
    int s = s0 + wave, step = 0;
    if (s >= s1) return;
    const unsigned end = (unsigned)V - 4;
    fx4u pv[kQuads], qv[kQuads];
    auto load = [&](int s, int step, fx4u (&pv)[kQuads], fx4u (&qv)[kQuads]) {
        const unsigned x0 = (unsigned)s * len + 256u * kQuads * step + 4u * lane;
#pragma unroll
        for (int e = 0; e < kQuads; ++e) {
            const unsigned x = min(x0 + 256u * e, end);
            pv[e] = *reinterpret_cast<const fx4u *>(f.p + x);
            if (Q) qv[e] = *reinterpret_cast<const fx4u *>(f.q + x);
        }
    };
    load(s, 0, pv, qv);
    double t = 0.0;
    for (;;) {
        int s2 = s, step2 = step + 1;
        if (step2 == steps) {
            s2 = s + WAVES;
            step2 = 0;
        }
        fx4u pn[kQuads], qn[kQuads];
        const bool more = s2 < s1;
        load(more ? s2 : s, more ? step2 : step, pn, qn);
        const unsigned x0 = (unsigned)s * len + 256u * kQuads * step;
        if (x0 + 256u * kQuads > (unsigned)V) {   // (uniform) the row's end
#pragma unroll
            for (int e = 0; e < kQuads; ++e) {
                const unsigned x = x0 + 256u * e + 4u * lane, xc = min(x, end);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (xc + i < x) {
                        pv[e][i] = 0.0f;
                        if (Q) qv[e][i] = 0.0f;
                    }
            }
        }
        if (!Q)
            for (int j = 0; j < f.ngone; ++j) {   // (uniform; few tokens fall into a step)
                const unsigned g = (unsigned)f.gone[j];
                if (g < x0 || g >= x0 + 256u * kQuads) continue;
#pragma unroll
                for (int e = 0; e < kQuads; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (g == min(x0 + 256u * e + 4u * lane, end) + i) pv[e][i] = 0.0f;
            }
        unsigned keep = 0;   // LIST: bit 4 e + i
#pragma unroll
        for (int e = 0; e < kQuads; ++e) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const double r = left_of(pv[e][i], Q ? qv[e][i] : 0.0f, f.a);
                t += r;
                if (LIST) keep |= r > 0.0 ? 1u << (4 * e + i) : 0u;
            }
        }
        if (LIST) {
            // Room for the lanes' pairs: lane by lane.
            const int own = __popc(keep);
            int upto = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int u = __shfl_up(upto, d);
                if (lane >= d) upto += u;
            }
            if (LANES) sm.lanes(s1 - s0)[(s - s0) * 64 + lane] = (unsigned short)((upto - own) * 32 + own);
            const int all = __builtin_amdgcn_readlane(upto, 63);
            int at = 0;
            if (lane == 0) {
                at = atomicAdd(&sm.listed, all);
                sm.off[s] = at;
                sm.cnt[s] = all;
            }
            at = __builtin_amdgcn_readfirstlane(at);
            if (at + all <= sm.room(LANES ? s1 - s0 : 0)) {
                at += upto - own;
#pragma unroll
                for (int e = 0; e < kQuads; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (keep >> (4 * e + i) & 1) sm.list[at++] = make_float2(pv[e][i], qv[e][i]);
            }
        }
        if (step2 == 0) {
            t = wave_sum64(t);
            if (lane == 0) sm.seg[s] = t;
            t = 0.0;
        }
        if (!more) break;
        s = s2;
        step = step2;
#pragma unroll
        for (int e = 0; e < kQuads; ++e) {
            pv[e] = pn[e];
            if (Q) qv[e] = qn[e];
        }
    }
}

// The same for rows of one to three tokens.
__device__ void sum_tiny(const Left &f, int V, VerifySmem &sm) {
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int x = 0; x < V; ++x) {
            bool out = false;
            for (int j = 0; j < f.ngone; ++j) out |= f.gone[j] == x;
            if (!out) t += left_of(f.p[x], f.q ? f.q[x] : 0.0f, f.a);
        }
        sm.seg[0] = t;
    }
}

// The same from the list, its pairs to the lanes in turn.
template <int WAVES> __device__ void sum_list(double a, int s0, int s1, VerifySmem &sm) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int s = s0 + wave; s < s1; s += WAVES) {
        const int c = __builtin_amdgcn_readfirstlane(sm.cnt[s]), o = __builtin_amdgcn_readfirstlane(sm.off[s]);
        double t = 0.0;
        for (int i = lane; i < c; i += 64) {
            const float2 v = sm.list[o + i];
            t += left_of(v.x, v.y, a);
        }
        t = wave_sum64(t);
        if (lane == 0) sm.seg[s] = t;
    }
}

// The same, each lane taking what was its own, in order: the bits that sum_segs
// gives (the tokens left out add 0).  Lanes keep only what still counts: the
// first pass takes the longest lane's number of steps, up to 16, the later ones
// some 7 (64 trees of 16 over 131072 tokens 49.9 us where pairs to the lanes in
// turn took 45.8, but then the bits hang on who adds up the part).
template <int WAVES> __device__ void sum_lanes(double a, int s0, int s1, VerifySmem &sm) {
    constexpr int U = 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int s = s0 + wave; s < s1; s += WAVES) {
        unsigned short *word = sm.lanes(s1 - s0) + (s - s0) * 64 + lane;
        const int w = *word, own = w & 31, at = sm.off[s] + (w >> 5);
        int n = 0;
        double t = 0.0;
        for (int i = 0; __any(i < own); i += U) {
            float2 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = sm.list[i + u < own ? at + i + u : kListZero];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const double r = left_of(v[u].x, v[u].y, a);
                t += r;
                sm.list[i + u < own ? at + n : kListZero + 1] = v[u];
                n += r > 0.0;
            }
        }
        *word = (unsigned short)((w & ~31) | n);
        t = wave_sum64(t);
        if (lane == 0) sm.seg[s] = t;
    }
}

// Lane l's share of the segments: s in [l c, (l + 1) c), c = ceil(segs / 64).
__device__ inline double lane_segs(int segs, const VerifySmem &sm, int lane) {
    const int c = (segs + 63) / 64;
    double t = 0.0;
    for (int s = lane * c; s < min((lane + 1) * c, segs); ++s) t += sm.seg[s];
    return t;
}

// Every thread, after the segments' barrier: the sum of all of them.
__device__ double total_of(int segs, VerifySmem &sm) {
    if (threadIdx.x < 64) {
        const double t = wave_sum64(lane_segs(segs, sm, threadIdx.x));
        if (threadIdx.x == 0) sm.total = t;
    }
    __syncthreads();
    const double t = sm.total;
    __syncthreads();
    return t;
}

// One wave: the first token whose cumulative sum passes target; where
// rounding keeps every one from it, the last with anything left in the
// segment that should hold it.
__device__ int find_left(const Left &f, int V, int len, int segs, double target,
                         const VerifySmem &sm, int lane) {
    // The lane, then the segment, that holds it.
    const double own = lane_segs(segs, sm, lane), upto = wave_scan64(own, lane);
    unsigned long long pass = __ballot(own > 0.0 && upto > target);
    const unsigned long long some = __ballot(own > 0.0);
    if (!some) return -1;
    int l = pass ? __ffsll((long long)pass) - 1 : 63 - __clzll((long long)some);
    double before = __shfl(upto - own, l);
    const int c = (segs + 63) / 64;
    int seg = -1;
    double cum = before;
    for (int s = l * c; s < min((l + 1) * c, segs); ++s) {
        const double t = sm.seg[s];
        if (t > 0.0) {
            seg = s;
            before = cum;
            if (cum + t > target) break;
        }
        cum += t;
    }
    if (seg < 0) return -1;
    // Within the segment, 64 E tokens at a time, lane i E in a row.
    constexpr int E = 8;
    int last = -1;   // the last token with anything left so far
    for (int x0 = seg * len; x0 < min(seg * len + len, V); x0 += 64 * E) {
        const int x = x0 + lane * E, end = min(seg * len + len, V);
        double r[E], mine = 0.0;
        fx4u pv[E / 4], qv[E / 4];
#pragma unroll
        for (int e = 0; e < E / 4; ++e) {
            pv[e] = load4(f.p, min(x + 4 * e, end), end);
            qv[e] = f.q ? load4(f.q, min(x + 4 * e, end), end) : fx4u{0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (int j = 0; j < f.ngone; ++j) {
            const int off = f.gone[j] - x;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (off == e) pv[e / 4][e % 4] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            r[e] = left_of(pv[e / 4][e % 4], qv[e / 4][e % 4], f.a);
            mine += r[e];
        }
        const double to = before + wave_scan64(mine, lane);
        pass = __ballot(mine > 0.0 && to > target);
        const unsigned long long any = __ballot(mine > 0.0);
        if (any) {
            l = pass ? __ffsll((long long)pass) - 1 : 63 - __clzll((long long)any);
            int found = -1;
            cum = to - mine;
            bool done = false;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (r[e] > 0.0 && !done) {
                    found = x + e;
                    cum += r[e];
                    done = cum > target;
                }
            last = __shfl(found, l);
            if (pass) break;
        }
        before = __shfl(to, 63);
    }
    return last;
}

// A sequence's words in the workspace, zero between launches.
struct VerifyWords {
    int arrived, left;         // parts that have added up the first pass; that are through
    int posted;                // passes whose total is in the workspace
    int claim[kVerifyParts], done[kVerifyParts];   // the latest pass that part k was taken for; is stored for
};

// Workgroup (sequence b, part): everything up to the first pass and its part
// of that.  The last one to arrive leads.
// Without TOGETHER it walks on alone (1024 threads: its loads are what bounds
// it; with 512, 64 sequences over 32768 tokens take 3 us more).
// TOGETHER (there is a q; 512 threads, 1024 would spill): every workgroup of a
// sequence walks by itself, on the passes' totals, which the leader adds up and
// posts.  None waits without an end for another: a workgroup that sees no total
// for some time leaves, a part that its own workgroup has not claimed when the
// leader is done with its own falls to the leader, and so does a claimed one
// that stays away (it is the same sum, to the bit: from a list or from the rows
// each lane adds its own tokens in order).
template <int THREADS, bool TOGETHER>
__global__ __launch_bounds__(THREADS) void tree_verify_kernel(VerifyArgs a, VerifyPlan pl) {
    constexpr int WAVES = THREADS / 64;
    __shared__ VerifySmem sm;
    const int b = blockIdx.x / pl.parts, part = blockIdx.x % pl.parts;
    const int tid = threadIdx.x, N = a.N, V = a.V, segs = pl.segs;
    const size_t row0 = (size_t)b * N;
    const bool has_q = TOGETHER || a.q;
    if (tid < N) {
        const int par = a.parent[row0 + tid], t = a.token[row0 + tid];
        const bool child = par >= 0 && par < tid && t >= 0 && t < V;
        sm.parent[tid] = tid == 0 ? par : child ? par : -1;
        sm.token[tid] = t;
        sm.u[tid] = a.u_accept[row0 + tid];
        sm.pt[tid] = child ? a.p[(row0 + par) * a.ldp + t] : 0.0f;
        sm.qt[tid] = child ? (has_q ? fmaxf(a.q[(row0 + par) * a.ldq + t], 0.0f) : 1.0f) : 0.0f;
        sm.path[tid] = -1;
    }
    __syncthreads();
    if (sm.parent[0] != -1) {   // no root: no sequence
        if (part == 0 && tid < N) a.path[row0 + tid] = -1;
        if (part == 0 && tid == 0) {
            a.n_acc[b] = -1;
            a.next[b] = -1;
        }
        return;
    }
    if (!has_q && tid < N) {
        bool first = tid > 0 && sm.parent[tid] >= 0;
        for (int j = 1; j < tid; ++j)
            if (sm.parent[j] == sm.parent[tid] && sm.token[j] == sm.token[tid]) first = false;
        sm.first[tid] = first;
    }
    __syncthreads();

    int cur = 0, n = 0, i = 1;
    bool summed = false, listed = false;
    double w = 1.0;
    Left f{a.p + row0 * a.ldp, has_q ? a.q + row0 * a.ldq : nullptr, 0.0, sm.gone, 0};
    if (tid == 0) {
        sm.path[0] = 0;
        sm.list[kListZero] = make_float2(0.0f, 0.0f);
    }

    // Lane i's node i, and the nodes whose token no earlier sibling has.
    const int lane = tid & 63;
    const int my_parent = lane < N ? sm.parent[lane] : -1;
    const float my_u = lane < N ? sm.u[lane] : 0.0f, my_p = lane < N ? sm.pt[lane] : 0.0f,
                my_q = lane < N ? sm.qt[lane] : 0.0f;
    const unsigned long long firsts = __ballot(!has_q && lane < N && sm.first[lane]);
    auto children = [&](int from) {   // of cur, from node `from` on
        return __ballot(my_parent == cur) & (from < 64 ? ~0ull << from : 0);
    };
    auto node = [](float v, int i) {
        return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i));
    };
    // Walks on from child i; true where a pass over f is due: f then is what
    // is left after the rejection of child i, or at the end (i == N) the
    // node's own row.
    auto walk = [&]() -> bool {
        for (;; ++i) {
            const unsigned long long left = children(i);
            if (!left) break;
            i = __ffsll((long long)left) - 1;
            const double u = (double)node(my_u, i), qt = (double)node(my_q, i);
            double r = left_of(node(my_p, i), has_q ? (float)qt : 0.0f, f.a);
            if (!has_q && !(firsts >> i & 1)) r = 0.0;
            if (u * qt * w < r) {
                cur = i;
                ++n;
                if (tid == 0) sm.path[n] = i;
                f.p = a.p + (row0 + i) * a.ldp;
                if (has_q) f.q = a.q + (row0 + i) * a.ldq;
                f.a = 0.0;
                f.ngone = 0;
                w = 1.0;
                summed = listed = false;
            } else if (has_q) {
                f.a += w;
                return true;
            } else if (!summed) {
                return true;
            } else {
                w = sm.after[i];
            }
        }
        i = N;
        if (summed && w != 0.0) return false;
        f.q = nullptr;   // no child rejected, or nothing left: the node's own row
        f.a = 0.0;
        f.ngone = 0;
        return true;
    };
    const bool shared = pl.parts > 1;
    auto pass = [&](int s0, int s1, bool own) {
        const bool last = i >= N;
        if (!has_q && !last) {
            // The children's tokens, each once.
            __syncthreads();
            if (tid < 64) {
                const bool out = tid < N && tid > 0 && sm.parent[tid] == cur && sm.first[tid];
                const unsigned long long m = __ballot(out);
                if (out) sm.gone[__popcll(m & ((1ull << tid) - 1))] = sm.token[tid];
                if (tid == 0) sm.ngone = __popcll(m);
            }
            __syncthreads();
            f.ngone = sm.ngone;
        }
        if (V < 4) {
            sum_tiny(f, V, sm);
            return;
        }
        if (!f.q) {
            sum_segs<WAVES, false, false>(f, V, pl.len, s0, s1, sm);
            return;
        }
        // Is there another child to be tried at the node?
        if (own) listed = pl.len == 256 * kQuads && children(i + 1);
        if (own && listed) {
            __syncthreads();
            if (tid == 0) sm.listed = 0;
            __syncthreads();
            sum_segs<WAVES, true, true, TOGETHER>(f, V, pl.len, s0, s1, sm);
        } else {
            sum_segs<WAVES, true, false>(f, V, pl.len, s0, s1, sm);
        }
    };
    // After a pass with the total t: w, and without q the sums after each
    // further rejection: the later children's, added up from the last one on
    // (nothing is subtracted, so what is left of large and small tokens is as
    // exact as its own sum, and no child's infinity outlives it).
    auto settle = [&](double t) {
        w = t;
        if (!has_q && i < N) {
            if (tid < 64) {
                const bool in = tid < N && tid > 0 && sm.parent[tid] == cur && sm.first[tid];
                const double v = in && sm.pt[tid] > 0.0f ? (double)sm.pt[tid] : 0.0;
                const double later = __shfl_down(wave_back_scan64(v, tid), 1);
                sm.after[tid] = w + (tid < 63 ? later : 0.0);
            }
            __syncthreads();
            w = sm.after[i];
        }
        summed = true;
        ++i;
    };

    const int p0 = (int)((long long)segs * part / pl.parts), p1 = (int)((long long)segs * (part + 1) / pl.parts);
    VerifyWords *words = reinterpret_cast<VerifyWords *>(a.words) + (shared ? b : 0);
    unsigned long long *sums = a.sums + (shared ? (size_t)b * (segs + kTreeMaxNodes) : 0);
    auto cload = [](const int *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto cput = [](int *p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto count = [&](int *p) {   // every thread: is this the last part to count?
        publish();
        if (tid == 0)
            sm.flag = __hip_atomic_fetch_add(p, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == pl.parts - 1;
        __syncthreads();
        return sm.flag != 0;
    };
    auto put_sums = [&]() {
        for (int s = p0 + tid; s < p1; s += THREADS)
            cstore64(sums + s, __builtin_bit_cast(unsigned long long, sm.seg[s]));
    };
    auto get_sums = [&](unsigned parts) {   // of these parts
        if (tid < segs && parts >> (((tid + 1) * pl.parts - 1) / segs) & 1)
            sm.seg[tid] = __builtin_bit_cast(double, cload64(sums + tid));
        __syncthreads();
    };
    bool leads = true;
    if (!TOGETHER) {
        walk();   // (a pass is always due: a sequence ends with one)
        pass(p0, p1, !shared);
        __syncthreads();
        if (shared) {
            put_sums();
            if (!count(&words->arrived)) return;
            if (tid == 0) cput(&words->arrived, 0);
            get_sums(~(1u << part));
        }
        settle(total_of(segs, sm));
        while (i <= N && walk()) {
            __syncthreads();
            const bool list = f.q && listed && sm.listed <= sm.room(TOGETHER ? p1 - p0 : 0);
            __syncthreads();    // (every thread has seen sm.listed)
            if (list) sum_list<WAVES>(f.a, 0, segs, sm);
            else      pass(0, segs, true);
            __syncthreads();
            settle(total_of(segs, sm));
        }
    } else {
        unsigned long long *totals = sums + segs;
        auto claim = [&](int k, int j) {   // part k of pass j
            int was = j - 1;
            return __hip_atomic_compare_exchange_strong(&words->claim[k], &was, j, __ATOMIC_RELAXED,
                                                        __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        const long long start = wall_clock64();   // (100 MHz)
        long long once = 0;                       // what the first pass took
        bool mine = true, due = walk();
        for (int j = 0; due; ++j) {
            const bool last = i >= N;
            unsigned todo = mine ? 1u << part : 0u, theirs = 0;   // parts to add up here; by others
            bool own = true;
            for (int stage = 0;; ++stage) {
                while (todo) {
                    const int k = __ffs(todo) - 1;
                    todo &= todo - 1;
                    __syncthreads();
                    const bool list = own && f.q && listed && sm.listed <= sm.room(TOGETHER ? p1 - p0 : 0);
                    __syncthreads();    // (every thread has seen sm.listed)
                    if (list) sum_lanes<WAVES>(f.a, p0, p1, sm);
                    else      pass((int)((long long)segs * k / pl.parts), (int)((long long)segs * (k + 1) / pl.parts), own);
                }
                own = false;
                __syncthreads();
                if (j == 0 || !leads || stage == 2) break;
                // The leader's own part is done: what nobody has claimed, then
                // what stays away.
                if (tid < 64) {
                    const int k = min(tid, kVerifyParts - 1);
                    const bool other = tid < pl.parts && tid != part;
                    unsigned long long m;
                    if (stage == 0) {
                        m = __ballot(other && claim(k, j));
                    } else {
                        const bool wait = other && (theirs >> k & 1);
                        const long long from = wall_clock64();
                        do m = __ballot(wait && cload(&words->done[k]) != j);
                        while (m && wall_clock64() - from < 10000 + 8 * once);
                    }
                    if (tid == 0) sm.mask = (unsigned)m;
                }
                __syncthreads();
                todo = sm.mask;
                if (stage == 0) theirs = ~(1u << part);
                theirs &= ~todo;
                __syncthreads();
            }
            if (j == 0) {
                put_sums();
                leads = count(&words->arrived);
                theirs = ~(1u << part);
                once = wall_clock64() - start;
                __syncthreads();
            } else if (!leads && mine) {
                put_sums();
                publish();
                if (tid == 0) cput(&words->done[part], j);
            }
            if (leads) {
                get_sums(theirs);
                const double t = total_of(segs, sm);
                if (!last && tid == 0) {
                    cstore64(totals + j, __builtin_bit_cast(unsigned long long, t));
                    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
                    cput(&words->posted, j + 1);
                }
                settle(t);
            } else {
                if (last) break;
                if (tid == 0) {
                    sm.claimed = claim(part, j + 1);   // (should there be one)
                    const long long from = wall_clock64();
                    bool got;
                    while (!(got = cload(&words->posted) > j) && wall_clock64() - from < 2000 + 4 * once)
                        __builtin_amdgcn_s_sleep(4);
                    sm.flag = got;
                    if (got) sm.total = __builtin_bit_cast(double, cload64(totals + j));
                }
                __syncthreads();
                if (!sm.flag) break;
                const double t = sm.total;
                mine = sm.claimed;
                __syncthreads();
                settle(t);
            }
            due = i <= N && walk();
        }
    }
    if (leads) {
        if (tid < N) a.path[row0 + tid] = sm.path[tid];
        if (tid < 64) {
            const bool fine = w > 0.0 && w < (double)INFINITY;
            const int x = fine ? find_left(f, V, pl.len, segs, (double)a.u_sample[b] * w, sm, tid) : -1;
            if (tid == 0) {
                a.n_acc[b] = n;
                a.next[b] = x;
            }
        }
    }
    // The last one through clears the words.
    if (TOGETHER && count(&words->left))
        if (tid < (int)(sizeof(VerifyWords) / sizeof(int))) cput(&words->arrived + tid, 0);
}

// The position after a step: pos, and the accepted rows that fit the cache.
__device__ inline int advanced(int pos, int n_acc, int N, int max_seq) {
    if (pos < 0 || pos >= max_seq || n_acc < 0) return pos;
    return pos + min(min(n_acc, N - 1) + 1, max_seq - pos);
}

// Thread (float4 of a row): blockIdx.y = 2 block + (0 keys, 1 values).  Rows
// of 8 blocks for 64 sequences 4.2 us, for one 2.9 (the launch and three
// dependent loads).
__global__ __launch_bounds__(256) void tree_commit_kernel(CommitArgs a) {
    const int quads = a.kv_dim / 4;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i < (size_t)a.B * a.N * quads) {
        const int e = (int)(i % quads);
        const size_t row = i / quads;
        const int j = (int)(row % a.N), b = (int)(row / a.N);
        const int pos = a.pos[b], from = a.path[row];
        if (j <= a.n_acc[b] && from >= 0 && from < a.N && pos >= 0 && pos < a.max_seq &&
            j < a.max_seq - pos) {
            const int blk = blockIdx.y >> 1;
            const float *src = blockIdx.y & 1 ? a.vd[blk] : a.kd[blk];
            float *dst = blockIdx.y & 1 ? a.vc[blk] : a.kc[blk];
            const float4 v = *reinterpret_cast<const float4 *>(
                src + ((size_t)b * a.N + from) * a.kv_dim + 4 * e);
            *reinterpret_cast<float4 *>(dst + ((size_t)b * a.max_seq + pos + j) * a.kv_dim + 4 * e) = v;
        }
    }
    if (a.pos_out && blockIdx.y == 0 && i < (size_t)a.B)
        a.pos_out[i] = advanced(a.pos[i], a.n_acc[i], a.N, a.max_seq);
}

__global__ __launch_bounds__(256) void tree_advance_kernel(const int *pos, const int *n_acc,
                                                           int *pos_out, int B, int N,
                                                           int max_seq) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < B) pos_out[b] = advanced(pos[b], n_acc[b], N, max_seq);
}

}  // namespace

VerifyPlan verify_plan(int B, int V, bool has_q) {
    VerifyPlan p{};
    // At most kMaxSegs segments, each a lane's kQuads float4s or a multiple.
    p.len = 256 * kQuads * ((V - 1) / (256 * kQuads * kMaxSegs) + 1);
    p.segs = (V - 1) / p.len + 1;
    // A workgroup per CU, of eight segments at least.
    p.parts = std::min({std::max(1, device_cus() / std::max(B, 1)), (p.segs + 7) / 8, kVerifyParts});
    // Later passes with help: a hand-over costs 3 us, a CU alone reads a segment
    // of both rows in 0.18.  us (trees of 16, alone and together, mean of six
    // seeds) with one sequence over 65536 tokens 16.2 17.3, 131072 19.4 15.2; 8
    // sequences 65536 23.6 22.3, 131072 38.9 25.1; 64 sequences (4 parts) 65536
    // 34.5 34.4, 131072 69.5 51.0.  Below that it loses (8 over 16384 16.0 23.8, 64
    // over 32768 24.2 31.4), and with two parts too (100 over 65536 41.5 48.9).
    // Without q nodes rarely need more than one pass: 8 over 262144 14.1 15.7.
    p.together = has_q && p.parts >= 4 && p.segs >= 64;
    p.sum_bytes = p.parts > 1 ? (size_t)B * (p.segs + kTreeMaxNodes) * 8 : 0;
    p.word_bytes = p.parts > 1 ? (size_t)B * sizeof(VerifyWords) : 0;
    return p;
}

hipError_t launch_tree_verify(const VerifyArgs &a, const VerifyPlan &p, hipStream_t s) {
    if (a.B <= 0) return hipSuccess;
    if (a.N < 1 || a.N > kTreeMaxNodes || a.V < 1 || p.parts < 1 || p.parts > kVerifyParts)
        return hipErrorInvalidValue;
    const dim3 grid((unsigned)((size_t)a.B * p.parts));
    if (p.together) hipLaunchKernelGGL((tree_verify_kernel<512, true>), grid, dim3(512), 0, s, a, p);
    else            hipLaunchKernelGGL((tree_verify_kernel<1024, false>), grid, dim3(1024), 0, s, a, p);
    return hipGetLastError();
}

hipError_t launch_tree_commit(const CommitArgs &a, hipStream_t s) {
    if (a.B <= 0 || a.blocks <= 0) return hipSuccess;
    if (a.blocks > kCommitBlocks || a.N < 1 || a.kv_dim < 4 || a.kv_dim % 4)
        return hipErrorInvalidValue;
    const size_t n = (size_t)a.B * a.N * (a.kv_dim / 4);
    hipLaunchKernelGGL(tree_commit_kernel, dim3((unsigned)((n + 255) / 256), 2 * a.blocks), dim3(256),
                       0, s, a);
    return hipGetLastError();
}

hipError_t launch_tree_advance(const int *pos, const int *n_acc, int *pos_out, int B, int N,
                               int max_seq, hipStream_t s) {
    if (B <= 0) return hipSuccess;
    hipLaunchKernelGGL(tree_advance_kernel, dim3((unsigned)((B + 255) / 256)), dim3(256), 0, s, pos,
                       n_acc, pos_out, B, N, max_seq);
    return hipGetLastError();
}

}  // namespace moe
