// Gated linear recurrences for sm_100a.
//
//   forward    h[t] = gate[t]*h[t-1] + x[t],  h[-1] = init (0 when absent)
//   backward   u[t] = g[t] + c[t+1],  c[t] = gate[t]*u[t],  c[T] = upstream gradient of the
//              last state;  dx[t] = u[t],  dgate[t] = u[t]*h[t-1],  dinit = c[0]
//
// Both are a chain of maps c -> A*c + H, and maps compose: a run of steps is one map, found
// without knowing the state it starts from.  Every warp takes a tile of the time axis, finds
// its map, learns its first state by joining the maps of the tiles before it, and only then
// writes its states: one pass over the data, each value read once and written once, which is
// what bounds these kernels (forward 12 bytes a value, backward 20 with all gradients).
// Tiles come through a two-stage ring in shared memory filled by cp.async: a stage is refilled
// as soon as its values are in registers, so the loads of the next tiles are in flight while
// the tiles of this step wait for one another's maps.  CTAs stay and walk the blocks of lanes,
// the ring running on from one block to the next (a CTA per block spent most of a short scan
// on starting and draining).  Tiles are joined in time order, so results do not depend on how
// CTAs are scheduled, at three levels:
//   warps of a CTA        through shared memory, one block barrier a step;
//   CTAs of a cluster     through distributed shared memory, one cluster barrier a step,
//                         where there are too few lanes to fill the card;
//   segments of the axis  through device scratch, by a first launch that finds the segments'
//                         maps, where clusters are not enough (the data is read twice).
// Maps hold the products of their gates, which may leave float's range where no state does (growing gates and a
// small state, a state of 1e30 that decays).  A CTA watches for that (Watch) and, where it may have happened,
// walks its lanes once more, step by step as the recurrence is written.
// Time runs in scan order r: t = r forward, t = T-1-r backward.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "program.hpp"

namespace cg = cooperative_groups;

namespace ttb {

namespace {

constexpr int kWarps = 8;  // warps of a CTA (16 where lanes are adjacent and few enough for a CTA an SM)

struct Operand {
    const float* p;  // null: absent
    int64_t so, st, s1, s2;
};

struct ScanArgs {
    Operand in[SI_COUNT];
    float* out[SO_COUNT];
    float2* maps;     // [segments][lanes] maps of the time segments (segments > 1)
    int64_t lanes, inner, n2, T;
    int64_t seg_len;  // steps of a segment
    int segments;
    int group;        // log2 of the adjacent lanes of a warp that dgate is summed over
    int64_t units;    // blocks of lanes * segments, walked by the clusters of the grid
    int steps;        // of a unit
    int W;            // warps of a CTA along time; the others take further lanes
    int vec;          // bit k: operand k moves as vectors
};

enum Pass { ONLY = 0, MAPS = 1, JOINED = 2 };  // the whole scan; its segments' maps; the scan from them

__device__ __forceinline__ float apply(float2 m, float c) { return fmaf(m.x, c, m.y); }

// First m, then n.
__device__ __forceinline__ float2 join(float2 m, float2 n) { return make_float2(m.x * n.x, apply(n, m.y)); }

__device__ __forceinline__ float max_abs(float a, float b, float c) {  // NaN propagates
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// What a thread has seen of the maps (A, H) and the states, and whether the maps do.  Products must not overflow: a
// thread's run of steps has |A| <= 2 and a tile |A| <= 16, else it is GROWN (a step's tiles are 2^32 at most then).  A
// product below the normal range has lost some 2^-146 at most, which is next to nothing (2^-119) of states of 2^27,
// unless a run behind it grows.  So maps do unless one is GROWN, or one is TINY (|A| < 2^-90; part of a tile may
// have 2^-121) and one LARGE: a run grows, or an H or a state is above 2^20 (states between tiles may then be
// 2^27).  An H that is not finite is GROWN too: the state it stands for starts from 0 and may overflow where the
// true one, from another, does not.  The bits need not be one lane's: that costs time only.
enum Range { GROWN = 1, TINY = 2, LARGE = 4 };
constexpr float kTiny = 8.077935669e-28f, kLarge = 1048576.0f;  // 2^-90, 2^20
struct Watch {
    float run = 0.0f, tile = 0.0f, least = 1.0f, most = 0.0f;  // largest |A| of runs, of tiles, least |A|, largest |H|
    __device__ __forceinline__ void runs(float a, float b) { run = max_abs(run, a, b); }
    __device__ __forceinline__ void tile_of(float a) {
        tile = max_abs(tile, a, a);
        product(a);
    }
    __device__ __forceinline__ void product(float a) { least = fminf(least, fabsf(a)); }
    __device__ __forceinline__ void states(float h, float s) { most = max_abs(most, h, s); }
    __device__ __forceinline__ int range() const {
        return (run <= 2.0f && tile <= 16.0f && most <= 3.402823466e38f ? 0 : GROWN) | (least < kTiny ? TINY : 0) | (run <= 1.0f && most <= kLarge ? 0 : LARGE);
    }
};
__device__ __forceinline__ bool maps_do(int range) { return (range & GROWN) == 0 && (range & (TINY | LARGE)) != (TINY | LARGE); }

// The map of N steps in scan order, its gates' product as it comes.
template <bool BACKWARD, int N, class G, class X>
__device__ __forceinline__ float2 tile_map(G gate, X x) {
    float2 m = make_float2(gate(0), BACKWARD ? gate(0) * x(0) : x(0));
#pragma unroll
    for (int j = 1; j < N; ++j) {
        m.x *= gate(j);
        m.y = BACKWARD ? gate(j) * (x(j) + m.y) : fmaf(gate(j), m.y, x(j));
    }
    return m;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// Asynchronous copy of BYTES (4, 8 or 16).
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const float* src) {
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }
__device__ __forceinline__ void copies_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Maps and states that the tiles of a step exchange.  Double-buffered: a buffer is written
// again two steps later, after a barrier that every reader passes behind its reads.
template <int NW, int LW>  // warps of the CTA, lanes of a warp's tile
struct Exchange {
    float2 warp[2][NW][LW];
    // only where W = NW (otherwise one step covers the axis):
    float2 cta[2][8][LW];  // by rank in the cluster
    float state[2][LW];    // the last warp's state behind a step, for the next one
    int range[NW], cta_range[8];  // Range bits of the warps, and of the cluster's CTAs
};
// The Range bits of all warps of the CTA.
template <int NW, int LW>
__device__ __forceinline__ int block_range(Exchange<NW, LW>& ex, int range) {
    range = __reduce_or_sync(0xffffffffu, range);
    __syncthreads();  // (they may still be read for the unit before)
    if ((threadIdx.x & 31) == 0) ex.range[threadIdx.x >> 5] = range;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) range |= ex.range[w];
    return range;
}

// A CTA's place: its rank in its cluster, the cluster's first unit and how many clusters walk them.
struct Place {
    int rank, size;
    int64_t first, clusters;
};
__device__ __forceinline__ Place place() {
    Place p;
    cg::cluster_group cl = cg::this_cluster();
    p.size = static_cast<int>(cl.num_blocks());
    p.rank = static_cast<int>(cl.block_rank());
    p.first = blockIdx.x / p.size;
    p.clusters = gridDim.x / p.size;
    return p;
}

// Lane -> (outer, inner) index.
__device__ __forceinline__ void split_lane(const ScanArgs& a, int64_t lane, int64_t& o, int64_t& i) {
    if (a.lanes <= 0x7fffffff) {
        const unsigned q = static_cast<unsigned>(lane), n = static_cast<unsigned>(a.inner);
        o = q / n;
        i = q % n;
    } else {
        o = lane / a.inner;
        i = lane % a.inner;
    }
}

__device__ __forceinline__ void split_inner(const ScanArgs& a, int64_t i, int64_t& i1, int64_t& i2) {
    if (a.n2 == a.inner) i1 = 0;
    else if (a.inner <= 0x7fffffff) i1 = static_cast<unsigned>(i) / static_cast<unsigned>(a.n2);
    else i1 = i / a.n2;
    i2 = i - i1 * a.n2;
}

// A segment's map as the first launch leaves it: NaN for A where it does not do.
__device__ __forceinline__ float2 segment_map(float gates, float h, int range) {
    return make_float2(maps_do(range) && fabsf(gates) <= 4294967296.0f ? gates : __int_as_float(0x7fc00000), h);
}

// The state before segment `seg` of a lane, from the maps of the segments before it and the lane's
// first state.  The warps of the CTA (all on the same lanes) join a share of the maps each,
// loading 8 at a time; LW lanes a warp, `writer` one thread of a lane.
template <int NW, int LW>
__device__ __forceinline__ float segment_state(const ScanArgs& a, Exchange<NW, LW>& ex, int seg, int64_t lane, bool live,
                                               float c, int warp, int l, bool writer, Watch& watch) {
    const int share = (seg + NW - 1) / NW, begin = min(seg, warp * share), end = min(seg, begin + share);
    float2 m = make_float2(1.0f, 0.0f);
    for (int s0 = begin; s0 < end; s0 += 8) {
        float2 q[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            q[u] = live && s0 + u < end ? __ldcg(a.maps + (s0 + u) * a.lanes + lane) : make_float2(1.0f, 0.0f);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            m = join(m, q[u]);
            // (a segment that grows is LARGE; one whose map does not do, and joins that would overflow, GROWN)
            const float grows = fabsf(q[u].x) <= 4294967296.0f ? fminf(fabsf(q[u].x), 1.5f) : INFINITY;
            watch.runs(grows, fabsf(m.x) <= 4294967296.0f ? 0.0f : INFINITY);
            watch.product(m.x);
            watch.states(q[u].y, c);
        }
    }
    __syncthreads();  // (the unit before may still be reading)
    if (writer) ex.warp[0][warp][l] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) c = apply(ex.warp[0][w][l], c);
    __syncthreads();
    return c;
}

// A CTA's part in the exchange, one lane per thread: thread l of a warp handles lane l of its
// tile (LW = 32), or all threads the tile's one row (LW = 1; `writer` is one of them).
template <int NW, int LW>
struct Joiner {
    Exchange<NW, LW>& ex;
    const Place& at;
    int W, wt, wr, warp, l;
    int buf = 0;

    // m: the map of this warp's tile.  Returns the state before the tile; c is the state before
    // the first step (later steps find theirs in the exchange).
    __device__ __forceinline__ float first(float2 m, float c, bool first_step, bool writer, Watch& watch) {
        watch.tile_of(m.x);
        if (writer) ex.warp[buf][warp][l] = m;
        __syncthreads();
        if (at.size > 1) {
            cg::cluster_group cl = cg::this_cluster();
            if (wt == 0 && writer) {
                float2 all = m;
#pragma unroll
                for (int w = 1; w < NW; ++w) all = join(all, ex.warp[buf][w][l]);
                watch.product(all.x);
                for (int q = 0; q < at.size; ++q) cl.map_shared_rank(&ex, q)->cta[buf][at.rank][l] = all;
            }
            cl.sync();
        }
        float s = first_step ? c : ex.state[buf][l];
        if (at.size > 1) {
#pragma unroll
            for (int q = 0; q < 7; ++q)
                if (q < at.rank) s = apply(ex.cta[buf][q][l], s);
        }
        if (W == NW) {
            float2 q[NW - 1];  // (all loaded, so that the loads do not wait for one another)
#pragma unroll
            for (int w = 0; w < NW - 1; ++w) q[w] = ex.warp[buf][w][l];
#pragma unroll
            for (int w = 0; w < NW - 1; ++w) s = w < wt ? apply(q[w], s) : s;
        } else {
            for (int w = 0; w < wt; ++w) s = apply(ex.warp[buf][wr * W + w][l], s);
        }
        watch.states(m.y, s);
        return s;
    }
    // s: the state behind this warp's tile.  The step's last tile hands it to the next step
    // (not behind the last step: another CTA of the cluster may have left).
    __device__ __forceinline__ void hand_on(float s, bool last_step, bool writer) {
        if (wt == W - 1 && at.rank == at.size - 1 && !last_step && writer) {
            if (at.size > 1) {
                cg::cluster_group cl = cg::this_cluster();
                for (int q = 0; q < at.size; ++q) cl.map_shared_rank(&ex, q)->state[buf ^ 1][l] = s;
            } else {
                ex.state[buf ^ 1][l] = s;
            }
        }
        buf ^= 1;
    }
    // The product of all gates of a step (for a segment's map; one lane group a CTA).
    __device__ __forceinline__ void gates_of_step(float& gates, Watch& watch) const {
#pragma unroll
        for (int w = 0; w < NW; ++w) gates *= ex.warp[buf][w][l].x;
        watch.product(gates);
    }
};

// The steps of a row before its vector v of four (in scan order), cut at CUT steps' boundaries.
template <bool BACKWARD, int CUT>
__device__ __forceinline__ int64_t steps_before(const ScanArgs& a, int64_t row, int64_t v) {
    const int shift = static_cast<int>(static_cast<unsigned>(row) * static_cast<unsigned>(a.T) & (CUT - 1));
    const int64_t vectors = (a.T + shift + CUT - 1) / CUT * (CUT / 4);
    const int64_t t = min(max(4 * (BACKWARD ? vectors - v : v) - shift, static_cast<int64_t>(0)), a.T);
    return BACKWARD ? a.T - t : t;
}

// The units of a CTA (a cluster's first one) once more, `lanes` lanes a unit, a thread a lane: the recurrence step by
// step, from the axis's begin to the unit's end.  CUT: of rows; 0 for lanes side by side, 32 of which are a warp's.
// Two batches of loads under way, so latency bounds it: 1 x 65536 x 1024 takes 8.6 ms instead of 0.15, 2000 rows of
// 8191 1.0 ms instead of 0.04.  (Steps without maps inside the tiles' loop, the warps in turn, were faster where
// they happened, and the loop's code slower where they did not: 4 to 19 %.)
template <bool BACKWARD, int CUT>
__device__ __noinline__ void walk_again(const ScanArgs& a, int64_t first, int64_t clusters, int lanes) {
    const int64_t all = (a.units - first + clusters - 1) / clusters * lanes;
    const bool want_gate = BACKWARD && a.out[SO_GATE];
    for (int64_t q = threadIdx.x; q - (threadIdx.x & 31) < all; q += blockDim.x) {
        const int64_t unit = first + q / lanes * clusters, block = unit / a.segments, seg = unit - block * a.segments;
        const int64_t lane = block * lanes + q % lanes;
        const bool live = q < all && lane < a.lanes;
        int64_t begin = seg * a.seg_len, end = begin + a.seg_len;
        if (CUT > 0) {
            begin = live ? steps_before<BACKWARD, CUT < 4 ? 4 : CUT>(a, lane, begin) : 0;
            end = live ? steps_before<BACKWARD, CUT < 4 ? 4 : CUT>(a, lane, end) : 0;
        } else {
            end = min(end, a.T);
        }
        int64_t o = 0, i = 0, i1, i2;
        if (live) split_lane(a, lane, o, i);
        split_inner(a, i, i1, i2);
        const int64_t t0 = BACKWARD ? a.T - 1 : 0;
        auto ptr = [&](int k, int64_t t) {
            const Operand& p = a.in[k];
            return live && p.p ? p.p + o * p.so + i1 * p.s1 + i2 * p.s2 + t * p.st : nullptr;
        };
        auto per_step = [&](int k) { return BACKWARD ? -a.in[k].st : a.in[k].st; };
        const float *gate = ptr(SI_GATE, t0), *x = ptr(SI_X, t0), *h = ptr(SI_H, t0 - 1), *init = ptr(SI_INIT, 0);
        const int64_t gs = per_step(SI_GATE), xs = per_step(SI_X), hs = per_step(SI_H);
        const float* carry = ptr(SI_CARRY, 0);
        float c = carry ? __ldg(carry) : 0.0f;
        constexpr int N = CUT > 0 ? 8 : 16;  // (16 steps of rows spill registers)
        struct Batch {
            float g[N], x[N], h[N];
        };
        // the steps r0 .. r0 + N - 1 before r1 (the others: gate 1, x 0), and the states before them
        auto load = [&](Batch& b, int64_t r0, int64_t r1, bool states) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const bool in = live && r0 + j < r1;
                b.g[j] = in ? __ldg(gate + (r0 + j) * gs) : 1.0f;
                b.x[j] = in && x ? __ldg(x + (r0 + j) * xs) : 0.0f;
                if constexpr (BACKWARD) {
                    const float* q = r0 + j == a.T - 1 ? init : h + (r0 + j) * hs;
                    b.h[j] = in && states && q ? __ldg(q) : 0.0f;
                }
            }
        };
        auto walk = [&](int64_t r0, int64_t r1, bool write) {
            const bool states = write && want_gate;
            Batch now, next;
            load(now, r0, r1, states);
            for (; r0 < r1; r0 += N) {
                load(next, r0 + N, r1, states);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float main = BACKWARD ? now.x[j] + c : fmaf(now.g[j], c, now.x[j]);
                    c = BACKWARD ? now.g[j] * main : main;
                    if (!write || r0 + j >= r1) continue;
                    const int64_t row = o * a.T + (BACKWARD ? a.T - 1 - r0 - j : r0 + j);
                    if (live && a.out[SO_MAIN]) a.out[SO_MAIN][row * a.inner + i] = main;
                    if constexpr (BACKWARD) {
                        if (!want_gate) continue;
                        float dg = main * now.h[j];
                        for (int d = 1; d >> a.group == 0; d *= 2) dg += __shfl_xor_sync(0xffffffffu, dg, d);
                        if (live && (i & ((1 << a.group) - 1)) == 0) a.out[SO_GATE][row * (a.inner >> a.group) + (i >> a.group)] = dg;
                    }
                }
                now = next;
            }
        };
        walk(0, begin, false);
        walk(begin, end, true);
        if (live && end == a.T && a.out[SO_LANE]) a.out[SO_LANE][lane] = c;
    }
}

// At a CTA's end: its units again where a thread of the cluster has seen maps that do not do.
template <bool BACKWARD, int CUT, int NW, int LW>
__device__ __forceinline__ void settle(const ScanArgs& a, Exchange<NW, LW>& ex, const Place& at, const Watch& watch, int lanes) {
    int range = watch.range();
    if (at.size == 1) {
        if (!__syncthreads_or(range & (GROWN | LARGE))) return;
        range = block_range(ex, range);
    } else {
        cg::cluster_group cl = cg::this_cluster();
        range = block_range(ex, range);
        if (threadIdx.x == 0) cl.map_shared_rank(&ex, 0)->cta_range[at.rank] = range;
        cl.sync();  // (the cluster's results are written, too)
        if (at.rank > 0) return;
        for (int q = 0; q < at.size; ++q) range |= ex.cta_range[q];
    }
    if (!maps_do(range)) walk_again<BACKWARD, CUT>(a, at.first, at.clusters, lanes);
}

template <int V>
__device__ __forceinline__ void load_shared(const float* p, float* v) {
    if constexpr (V == 4) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        v[0] = f.x;
        v[1] = f.y;
        v[2] = f.z;
        v[3] = f.w;
    } else if constexpr (V == 2) {
        const float2 f = *reinterpret_cast<const float2*>(p);
        v[0] = f.x;
        v[1] = f.y;
    } else {
        v[0] = *p;
    }
}
template <int V>
__device__ __forceinline__ void store_vec(float* p, const float* v, bool stream) {
    if constexpr (V == 4) {
        const float4 f = make_float4(v[0], v[1], v[2], v[3]);
        if (stream) __stcs(reinterpret_cast<float4*>(p), f);
        else *reinterpret_cast<float4*>(p) = f;
    } else if constexpr (V == 2) {
        const float2 f = make_float2(v[0], v[1]);
        if (stream) __stcs(reinterpret_cast<float2*>(p), f);
        else *reinterpret_cast<float2*>(p) = f;
    } else {
        if (stream) __stcs(p, v[0]);
        else *p = v[0];
    }
}

// ---- lanes side by side in memory ([.., T, lanes]): a warp's tile is TILE steps of 32 adjacent
// lanes, 16 or, forward, 24.  A thread takes V adjacent lanes and a V-th of the
// steps (32/V threads lie across the lanes, V behind one another in time), so that operands move
// in 4*V bytes a thread and 128 bytes a row whatever V is; the V threads of a lane join their
// maps by shuffles.  Operands whose lanes are adjacent move as V-vectors, operands broadcast over
// the lanes behind n1 as one value (V > 1 is only cut where each operand is one or the other);
// V = 1 takes any strides.  A thread reads back what it copied itself, or a thread of its warp
// (broadcast values), so the ring needs no block barrier.
// 8 x 2048 x 1024: 33 us forward (6.1 TB/s), 61 us backward with all gradients (5.5 TB/s: 256 CTAs on the
// 296 places of the card); 1 x 65536 x 1024 150 us (5.4 TB/s, a cluster barrier a step).  Where there are fewer
// lanes a step's latency bounds it, not the bytes: a gate per head of 64 lanes, 4 x 2048 x 1024, 23 and
// 35 us (3.0 and 2.9 TB/s).
template <bool BACKWARD>
constexpr int kArrays = BACKWARD ? 3 : 2;

template <bool BACKWARD, int TILE, int NW>
struct ColTile {
    float in[2][kArrays<BACKWARD>][NW][TILE * 32];  // [stage][operand][warp][step][thread][V]
    float carry[2][NW][32];                         // [stage][warp][lane]: a unit's first states
    Exchange<NW, 32> ex;
};

template <bool BACKWARD, int PASS, int V, int TILE, int NW>
__global__ void __launch_bounds__(NW * 32, 16 / NW) scan_cols_kernel(const __grid_constant__ ScanArgs a) {
    constexpr int TS = TILE / V, COLS = 32 / V, NA = kArrays<BACKWARD>;
    extern __shared__ __align__(16) unsigned char raw[];
    ColTile<BACKWARD, TILE, NW>& sh = *reinterpret_cast<ColTile<BACKWARD, TILE, NW>*>(raw);
    const Place at = place();
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31, W = a.W;
    const int wt = warp % W, wr = warp / W;
    const int col = l % COLS, sub = l / COLS;
    const bool want_gate = BACKWARD && PASS != MAPS && a.out[SO_GATE];
    // Places on the axis count from the segment's begin, in scan order; a segment has less than 2^31 steps.
    const int stride = at.size * W * TILE;  // of this warp's tiles
    const int own = (at.rank * W + wt) * TILE + sub * TS;
    auto block_of = [&](int64_t unit) { return a.segments == 1 ? unit : unit / a.segments; };
    auto first_lane = [&](int64_t unit) { return (block_of(unit) * (NW / W) + wr) * 32; };
    auto run_len = [&](int r0, int end) { return min(max(end - r0, 0), TS); };  // this thread's steps from r0 on
    // A thread's values of an operand in the ring: V a step, or one of an operand that is broadcast over the
    // lanes.  That one is copied by the first thread that shares it and read by all of them (each copying its
    // own, 32 threads from one address are served one after the other: 33 instead of 9 wavefronts a tile).
    auto slot = [&](int stage, int k, bool one) { return &sh.in[stage][k][warp][one ? l : l * V]; };
    auto is_one = [&](int k) { return a.n2 > 1 && a.in[k].s2 == 0; };
    auto leader = [&](int64_t i2) { return static_cast<int>(max(static_cast<int64_t>(0), col * V - i2)) / V; };  // its column

    // ---- the ring: a place ahead of the computation.  Pointers move on by a step, not by multiplications:
    // 64-bit products and comparisons were a third of the kernel's instructions.
    struct {
        int64_t unit;
        int r0, end, hend, step;     // hend: the end of the steps with a state before them
        bool leads;
        const float *gate, *x, *h, *init;  // of the thread's first step at r0 (h: of the step before it)
    } ahead;
    auto aim = [&](int64_t unit) {
        ahead.unit = unit;
        ahead.step = 0;
        if (unit >= a.units) return;
        const int64_t lane = first_lane(unit) + col * V, begin = (unit - block_of(unit) * a.segments) * a.seg_len;
        const bool live = lane < a.lanes;
        ahead.r0 = own;
        ahead.end = live ? static_cast<int>(min(a.seg_len, a.T - begin)) : 0;
        ahead.hend = live ? static_cast<int>(min(a.seg_len, a.T - 1 - begin)) : 0;
        int64_t o = 0, i = 0, i1, i2;
        if (live) split_lane(a, lane, o, i);
        split_inner(a, i, i1, i2);
        ahead.leads = leader(i2) == col;
        const int64_t t = BACKWARD ? a.T - 1 - begin - own : begin + own;
        auto ptr = [&](int k, int64_t time) {
            const Operand& q = a.in[k];
            return q.p ? q.p + o * q.so + i1 * q.s1 + i2 * q.s2 + time * q.st : nullptr;
        };
        ahead.gate = ptr(SI_GATE, t);
        ahead.x = ptr(SI_X, t);
        ahead.h = ptr(SI_H, t - 1);
        ahead.init = ptr(SI_INIT, 0);
    };
    // copies of one operand: n steps in scan order from q on
    auto fetch = [&](const float* q, int k, int stage, int arr, int n) {
        const int64_t step = BACKWARD ? -a.in[k].st : a.in[k].st;
        const bool one = is_one(k);
        if (one && !ahead.leads) return;
        const uint32_t dst = smem_addr(slot(stage, arr, one));
        if (V > 1 && !one) {
#pragma unroll
            for (int j = 0; j < TS; ++j, q += step)
                if (j < n) copy_async<4 * V>(dst + j * 128 * V, q);
        } else {
#pragma unroll
            for (int j = 0; j < TS; ++j, q += step)
                if (j < n) copy_async<4>(dst + j * 128 * V, q);
        }
    };
    auto moved = [&](const float*& q, int k) { q += BACKWARD ? -stride * a.in[k].st : stride * a.in[k].st; };
    auto issue = [&](int stage) {
        if (ahead.unit < a.units) {
            const int n = run_len(ahead.r0, ahead.end);
            if (n > 0) {
                fetch(ahead.gate, SI_GATE, stage, 0, n);
                if (a.in[SI_X].p) fetch(ahead.x, SI_X, stage, 1, n);
                if (want_gate) {  // the states before each step; before t = 0 there is init
                    const int nh = run_len(ahead.r0, ahead.hend);
                    fetch(ahead.h, SI_H, stage, NA - 1, nh);
                    if (nh < n && ahead.init) {
                        const uint32_t dst = smem_addr(slot(stage, NA - 1, false)) + nh * 128 * V;
#pragma unroll
                        for (int v = 0; v < V; ++v) copy_async<4>(dst + 4 * v, ahead.init + v * a.in[SI_INIT].s2);
                    }
                }
            }
            if (PASS == ONLY && ahead.step == 0 && a.in[SI_CARRY].p) {  // the unit's first states, lane by lane
                const int64_t lane = first_lane(ahead.unit) + l;
                if (lane < a.lanes) {
                    int64_t o, i, i1, i2;
                    split_lane(a, lane, o, i);
                    split_inner(a, i, i1, i2);
                    copy_async<4>(smem_addr(&sh.carry[stage][warp][l]),
                                  a.in[SI_CARRY].p + o * a.in[SI_CARRY].so + i1 * a.in[SI_CARRY].s1 + i2 * a.in[SI_CARRY].s2);
                }
            }
            ahead.r0 += stride;
            moved(ahead.gate, SI_GATE);
            moved(ahead.x, SI_X);
            if (want_gate) moved(ahead.h, SI_H);
            if (++ahead.step == a.steps) aim(ahead.unit + at.clusters);
        }
        copies_commit();
    };
    aim(at.first);
    issue(0);
    issue(1);
    if (at.size > 1) cg::this_cluster().sync();  // every CTA runs before another writes to it

    Joiner<NW, 32> joiner{sh.ex, at, W, wt, wr, warp, l};
    const bool one_gate = is_one(SI_GATE), one_x = is_one(SI_X), one_h = is_one(SI_H);
    const bool shares = one_gate || one_x || one_h;
    Watch watch;
    int stage = 0;
    for (int64_t unit = at.first; unit < a.units; unit += at.clusters) {
        const int seg = static_cast<int>(unit - block_of(unit) * a.segments);
        const int64_t lane0 = first_lane(unit), lane = lane0 + col * V;
        const bool live = lane < a.lanes;
        const int64_t begin = seg * a.seg_len;
        const int end = live ? static_cast<int>(min(a.seg_len, a.T - begin)) : 0;
        const int hend = live ? static_cast<int>(min(a.seg_len, a.T - 1 - begin)) : 0;
        const int last_end = live && begin + end == a.T ? end : -1;  // the axis ends here
        int64_t o = 0, i = 0;
        if (live) split_lane(a, lane, o, i);
        int64_t i1, i2;
        split_inner(a, i, i1, i2);
        const int shared_by = leader(i2) - col;  // where the thread that copies a broadcast value is
        // results of the thread's first step
        const int64_t row = o * a.T + (BACKWARD ? a.T - 1 - begin - own : begin + own);
        float* ym0 = a.out[SO_MAIN] + row * a.inner + i;
        float* yg0 = a.out[SO_GATE] + row * (a.inner >> a.group) + (i >> a.group);
        float c = 0.0f, gates = 1.0f;
        if constexpr (PASS == MAPS) watch = Watch();  // (a unit's own)
        if constexpr (PASS == JOINED) {
            const bool in = lane0 + l < a.lanes;
            if (in && a.in[SI_CARRY].p) {
                int64_t oc, ic;
                split_lane(a, lane0 + l, oc, ic);
                c = __ldg(a.in[SI_CARRY].p + oc * a.in[SI_CARRY].so + ic / a.n2 * a.in[SI_CARRY].s1 + ic % a.n2 * a.in[SI_CARRY].s2);
            }
            c = segment_state<NW, 32>(a, sh.ex, seg, lane0 + l, in, c, warp, l, true, watch);
        }
        int r0 = own;
        for (int k = 0; k < a.steps; ++k, r0 += stride, stage ^= 1) {
            const int n = run_len(r0, end);
            float ga[TS][V], xv[TS][V], hv[BACKWARD ? TS : 1][V];
            copies_wait_one();
            if (shares) __syncwarp();  // (broadcast values come from another thread's copies)
            auto read = [&](const float* q, bool one, int count, float none, float (*dst)[V]) {
                if (one) q += shared_by;
#pragma unroll
                for (int j = 0; j < TS; ++j) {
                    if (one) {
                        const float f = q[j * 32 * V];
#pragma unroll
                        for (int v = 0; v < V; ++v) dst[j][v] = f;
                    } else {
                        load_shared<V>(q + j * 32 * V, dst[j]);
                    }
                }
                if (count < TS) {
#pragma unroll
                    for (int j = 0; j < TS; ++j)
#pragma unroll
                        for (int v = 0; v < V; ++v)
                            if (j >= count) dst[j][v] = none;
                }
            };
            read(slot(stage, 0, one_gate), one_gate, n, 1.0f, ga);
            read(slot(stage, 1, one_x), one_x, a.in[SI_X].p ? n : 0, 0.0f, xv);
            if constexpr (BACKWARD) {
                const int nh = run_len(r0, hend);
                read(slot(stage, NA - 1, one_h), one_h, want_gate ? (a.in[SI_INIT].p ? n : nh) : 0, 0.0f, hv);
                if (one_h && want_gate && a.in[SI_INIT].p && nh < n) {  // init need not be broadcast where h is
#pragma unroll
                    for (int j = 0; j < TS; ++j)
                        if (j == nh) load_shared<V>(slot(stage, NA - 1, false) + j * 32 * V, hv[j]);
                }
            }
            if (PASS == ONLY && k == 0) c = a.in[SI_CARRY].p && lane0 + l < a.lanes ? sh.carry[stage][warp][l] : 0.0f;
            if (shares) __syncwarp();
            issue(stage);
            // this thread's maps, those of the threads before it in time, and the tile's
            float2 m[V], before[V];
#pragma unroll
            for (int v = 0; v < V; ++v) m[v] = tile_map<BACKWARD, TS>([&](int j) { return ga[j][v]; }, [&](int j) { return xv[j][v]; });
#pragma unroll
            for (int v = 0; v < V; v += 2) watch.runs(m[v].x, m[V > 1 ? v + 1 : 0].x);
#pragma unroll
            for (int d = COLS; d < 32; d *= 2) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float2 b = make_float2(__shfl_up_sync(0xffffffffu, m[v].x, d), __shfl_up_sync(0xffffffffu, m[v].y, d));
                    const float2 q = join(b, m[v]);
                    m[v] = l >= d ? q : m[v];
                }
            }
            float2 tile = m[0];
            if constexpr (V > 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    before[v] = make_float2(__shfl_up_sync(0xffffffffu, m[v].x, COLS), __shfl_up_sync(0xffffffffu, m[v].y, COLS));
                    // lane l's map lies with the last of its threads, 32 - COLS + l / V, at v = l % V
                    const float2 w = make_float2(__shfl_sync(0xffffffffu, m[v].x, 32 - COLS + l / V),
                                                 __shfl_sync(0xffffffffu, m[v].y, 32 - COLS + l / V));
                    tile = l % V == v ? w : tile;
                }
            }
            const bool last = k + 1 == a.steps;
            const float first = joiner.first(tile, c, k == 0, true, watch);
            if constexpr (PASS == MAPS) {
                joiner.gates_of_step(gates, watch);
                const float s = apply(tile, first);
                const int range = last ? block_range(sh.ex, watch.range()) : 0;
                if (last && lane0 + l < a.lanes && wt == W - 1) a.maps[seg * a.lanes + lane0 + l] = segment_map(gates, s, range);
                joiner.hand_on(s, last, true);
            } else {
                float s[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    s[v] = V > 1 ? __shfl_sync(0xffffffffu, first, col * V + v) : first;
                    if (V > 1) s[v] = sub > 0 ? apply(before[v], s[v]) : s[v];
                }
                const int64_t step = BACKWARD ? -a.inner : a.inner, step_g = BACKWARD ? -(a.inner >> a.group) : 0;
                float *ym = ym0, *yg = yg0;
                ym0 += stride * step;
                if (want_gate) yg0 += stride * step_g;
                const int nm = a.out[SO_MAIN] ? n : 0, ng = want_gate ? n : 0;
#pragma unroll
                for (int j = 0; j < TS; ++j, ym += step, yg += step_g) {  // (past the end: gate 1, x 0, the state stays)
                    float main[V], dg[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        if (BACKWARD) {
                            main[v] = xv[j][v] + s[v];
                            dg[v] = main[v] * hv[BACKWARD ? j : 0][v];
                            s[v] = ga[j][v] * main[v];
                        } else {
                            main[v] = s[v] = fmaf(ga[j][v], s[v], xv[j][v]);
                        }
                    }
                    if (j < nm) store_vec<V>(ym, main, BACKWARD);
                    if (!BACKWARD || a.group == 0) {
                        if (j < ng) store_vec<V>(yg, dg, true);
                    } else {  // summed over the lanes of a group within the warp (lanes that are not live hold 0)
                        float t = dg[0];
#pragma unroll
                        for (int v = 1; v < V; ++v) t += dg[v];
#pragma unroll
                        for (int d = 1; d < COLS; d *= 2) {
                            const float w = __shfl_xor_sync(0xffffffffu, t, d);
                            if (d * V >> a.group == 0) t += w;
                        }
                        if (j < ng && (col * V & ((1 << a.group) - 1)) == 0) *yg = t;
                    }
                }
                // the thread of the last step has the last state as it was stored
                if (n > 0 && r0 + n == last_end && a.out[SO_LANE]) store_vec<V>(a.out[SO_LANE] + lane, s, false);
                float behind = s[0];  // the state behind the tile, of lane l
                if (V > 1) {
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const float w = __shfl_sync(0xffffffffu, s[v], 32 - COLS + l / V);
                        if (l % V == v) behind = w;
                    }
                }
                joiner.hand_on(behind, last, true);
            }
        }
    }
    copies_wait_all();
    if constexpr (PASS != MAPS) settle<BACKWARD, 0>(a, sh.ex, at, watch, NW / W * 32);
}

// ---- time adjacent in memory ([.., T]): a warp's tile is 640 (backward 384) steps of one row, a
// run of 20 (12) adjacent steps per thread (an odd number of 16-byte vectors, so that the
// threads' runs lie in different banks), the runs' maps joined by shuffles.  Rows of up to
// SUB runs less 3 steps take SUB threads, 32/SUB rows a warp.  Tiles move between global and shared memory in coalesced
// vectors, in and out.  Rows need not start on 16 bytes: vectors are cut at the result's 16-byte
// boundaries (`shift` steps before the row's first one), so whole vectors move as 16 bytes and only
// ragged ends value by value.  Rows of whole warps are cut at 128-byte boundaries, so that tiles do not
// share lines (2000 rows of 8191: 38.0 us forward and 61.4 backward against 38.8 and 63.1).
// That is 5.2 and 5.3 TB/s; the step's barrier and 33 (60) instructions a value bound it.
template <int SUB>
constexpr int kRowCut = SUB == 32 ? 32 : 4;
template <bool BACKWARD>
constexpr int kRowRun = BACKWARD ? 12 : 20;

template <bool BACKWARD>
struct RowTile {
    float in[2][2][32 * kRowRun<BACKWARD>];                     // gate, x
    float h[BACKWARD ? 2 : 1][BACKWARD ? 32 * (kRowRun<BACKWARD> + 4) : 4];  // [stage]: rows apart by 4, for [-1]
    float out[32 * kRowRun<BACKWARD>];
    float carry[2][8];
};
template <bool BACKWARD>
constexpr size_t rows_smem() {
    return kWarps * sizeof(RowTile<BACKWARD>) + sizeof(Exchange<kWarps, 1>);
}

template <bool FIRST, class A, class B>
struct Select {
    using type = A;
};
template <class A, class B>
struct Select<false, A, B> {
    using type = B;
};

template <bool BACKWARD, int PASS, int SUB>
__global__ void __launch_bounds__(kWarps * 32, 2) scan_rows_kernel(const __grid_constant__ ScanArgs a) {
    constexpr int NW = kWarps, NA = kArrays<BACKWARD>, kRun = kRowRun<BACKWARD>, kTile = 32 * kRun, kVectors = kTile / 4;
    constexpr int R = 32 / SUB, VR = SUB * kRun / 4;  // rows a warp, vectors of a row's tile
    extern __shared__ __align__(16) unsigned char raw[];
    const Place at = place();
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31, W = a.W;
    const int wt = warp % W, wr = warp / W, sr = l / SUB, ls = l % SUB;  // ls: the thread's place in its row
    RowTile<BACKWARD>& tile = reinterpret_cast<RowTile<BACKWARD>*>(raw)[warp];
    Exchange<NW, 1>& ex = *reinterpret_cast<Exchange<NW, 1>*>(raw + NW * sizeof(RowTile<BACKWARD>));
    const bool want_gate = BACKWARD && PASS != MAPS && a.out[SO_GATE];
    const int64_t stride = static_cast<int64_t>(at.size) * W * VR;  // of this warp's tiles, in vectors of four
    const int64_t own = (static_cast<int64_t>(at.rank) * W + wt) * VR;
    // A unit's rows for this warp and its segment (without a division where there is one segment).
    struct Rows {
        int64_t row0, begin, end;  // segment in vectors of four, scan order
        int seg;
    };
    auto rows_of = [&](int64_t unit) {
        Rows r;
        const int64_t block = a.segments == 1 ? unit : unit / a.segments;
        r.seg = static_cast<int>(unit - block * a.segments);
        r.row0 = (block * (NW / W) + wr) * R;
        r.begin = r.seg * a.seg_len;
        r.end = r.begin + a.seg_len;
        return r;
    };
    // A row's tile at r0 (vectors, scan order): where it lies.  A tile that is cut short keeps, backward, its
    // high end; vectors [lo, lo + n) of it exist, the tile's first is v0 of the row.
    using Count = typename Select<SUB == 32, int64_t, int>::type;  // rows of a few threads are short
    struct Cutout {
        Count v0, vectors;
        int lo, n, shift;
    };
    auto cutout = [&](int64_t row, Count end, Count r0) {
        Cutout q;
        q.shift = static_cast<int>(static_cast<unsigned>(row) * static_cast<unsigned>(a.T) & (kRowCut<SUB> - 1));
        q.vectors = (static_cast<Count>(a.T) + q.shift + kRowCut<SUB> - 1) / kRowCut<SUB> * (kRowCut<SUB> / 4);
        const Count last = row < a.lanes ? min(q.vectors, end) : r0;
        q.n = static_cast<int>(max(static_cast<Count>(0), min(static_cast<Count>(VR), last - r0)));
        q.v0 = BACKWARD ? q.vectors - r0 - VR : r0;  // may be negative where n < VR
        q.lo = BACKWARD ? VR - q.n : 0;
        return q;
    };
    // all of the tile is inside the row: nothing to check vector by vector
    auto whole_tile = [&](const Cutout& q) {
        return q.n == VR && 4 * q.v0 >= q.shift && 4 * (q.v0 + VR) - q.shift <= a.T;
    };
    // A tile that is not (rows of whole warps): bit q says whether the thread's vector l + 32*q is inside the row.
    auto inside_vectors = [&](const Cutout& q) {
        unsigned m = 0;
#pragma unroll
        for (int u = 0; u < kVectors / 32; ++u) {
            const int v = l + 32 * u;
            const Count t = 4 * (q.v0 + v) - q.shift;
            if (v >= q.lo && v < q.lo + q.n && t >= 0 && t + 3 < a.T) m |= 1u << u;
        }
        return m;
    };
    // The steps of a row outside whole vectors, at most three at each end, are moved by eight threads: this
    // thread's step t, returned is its place in the tile (-1: none).
    auto edge = [&](const Cutout& q, Count& t) {
        const Count tail = static_cast<Count>(a.T) - ((static_cast<int>(a.T & 3) + q.shift) & 3);
        t = l < 4 ? l : tail + (l - 4);
        const bool is = l < 4 ? l < (-q.shift & 3) : l < 8 && t < a.T;
        const Count at_t = t + q.shift - 4 * q.v0;
        return is && at_t >= 4 * q.lo && at_t < 4 * (q.lo + q.n) ? static_cast<int>(at_t) : -1;
    };
    auto h_row = [&](int stage, int r) { return &tile.h[BACKWARD ? stage : 0][BACKWARD ? 4 + r * (SUB * kRun + 4) : 0]; };
    const int need = 1 << SI_GATE | (a.in[SI_X].p ? 1 << SI_X : 0) | (want_gate ? 1 << SI_H : 0);
    int64_t ahead_unit = at.first;
    Rows ahead = rows_of(ahead_unit);
    Count ahead_r0 = static_cast<Count>(ahead.begin + own);
    int ahead_step = 0;
    auto issue = [&](int stage) {
        if (ahead_unit < a.units) {
            const Cutout mine = cutout(ahead.row0 + sr, static_cast<Count>(ahead.end), ahead_r0);
            const int64_t at_t = 4 * static_cast<int64_t>(mine.v0) - mine.shift;
            if (SUB == 32 && whole_tile(mine) && (a.vec & need) == need) {
                auto copy = [&](int op, float* dst) {
                    const float* p = a.in[op].p + ahead.row0 * a.in[op].so + at_t + 4 * l;
                    const uint32_t to = smem_addr(dst + 4 * l);
#pragma unroll
                    for (int q = 0; q < kVectors / 32; ++q) copy_async<16>(to + 512 * q, p + 128 * q);
                };
                copy(SI_GATE, tile.in[stage][0]);
                if (a.in[SI_X].p) copy(SI_X, tile.in[stage][1]);
                if (want_gate) copy(SI_H, h_row(stage, 0));
            } else if (SUB == 32 && (a.vec & need) == need) {
                const unsigned in = inside_vectors(mine);
                Count t;
                const int e = edge(mine, t);
                auto copy = [&](int op, float* dst) {
                    const float* row = a.in[op].p + ahead.row0 * a.in[op].so;
                    const float* p = row + at_t + 4 * l;
                    const uint32_t to = smem_addr(dst + 4 * l);
#pragma unroll
                    for (int q = 0; q < kVectors / 32; ++q)
                        if (in >> q & 1) copy_async<16>(to + 512 * q, p + 128 * q);
                    if (e >= 0) copy_async<4>(smem_addr(dst + e), row + t);
                };
                copy(SI_GATE, tile.in[stage][0]);
                if (a.in[SI_X].p) copy(SI_X, tile.in[stage][1]);
                if (want_gate) copy(SI_H, h_row(stage, 0));
            } else {
#pragma unroll 1
                for (int q = 0; q < kVectors / 32; ++q) {
                    const int at_v = l + 32 * q, v = at_v % VR;
                    const int64_t row = ahead.row0 + at_v / VR;
                    const Cutout k = SUB == 32 ? mine : cutout(row, static_cast<Count>(ahead.end), ahead_r0);
                    if (v < k.lo || v >= k.lo + k.n) continue;
                    const Count t = 4 * (k.v0 + v) - k.shift;
                    const bool whole = t >= 0 && t + 3 < a.T;
#pragma unroll
                    for (int arr = 0; arr < NA; ++arr) {
                        const int op = arr == 0 ? SI_GATE : arr == 1 ? SI_X : SI_H;
                        if (arr == 1 && !a.in[SI_X].p) continue;
                        if (arr == 2 && !want_gate) continue;
                        const float* p = a.in[op].p + row * a.in[op].so;
                        const uint32_t to = smem_addr(arr == 2 ? h_row(stage, at_v / VR) + 4 * v : &tile.in[stage][arr & 1][4 * at_v]);
                        if ((a.vec >> op & 1) && whole) {
                            copy_async<16>(to, p + t);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (t + j >= 0 && t + j < a.T) copy_async<4>(to + 4 * j, p + (t + j) * a.in[op].st);
                        }
                    }
                }
            }
            const int64_t row = ahead.row0 + sr;
            if (ls == 0 && row < a.lanes) {
                if (PASS == ONLY && ahead_step == 0 && a.in[SI_CARRY].p)
                    copy_async<4>(smem_addr(&tile.carry[stage][sr]), a.in[SI_CARRY].p + row * a.in[SI_CARRY].so);
                const int64_t t = at_t + 4 * mine.lo;
                if (want_gate && t > -4 * mine.n) {  // (otherwise none of the vectors is inside the row)
                    // the state before the tile's first step in memory, in front of it: init before t = 0
                    float* dst = h_row(stage, sr) + 4 * mine.lo + (t < 0 ? -static_cast<int>(t) : 0) - 1;
                    if (t > 0) copy_async<4>(smem_addr(dst), a.in[SI_H].p + row * a.in[SI_H].so + (t - 1) * a.in[SI_H].st);
                    else if (a.in[SI_INIT].p) copy_async<4>(smem_addr(dst), a.in[SI_INIT].p + row * a.in[SI_INIT].so);
                    else *dst = 0.0f;
                }
            }
            ahead_r0 += static_cast<Count>(stride);
            if (++ahead_step == a.steps) {
                ahead_step = 0;
                ahead_unit += at.clusters;
                ahead = rows_of(ahead_unit);
                ahead_r0 = static_cast<Count>(ahead.begin + own);
            }
        }
        copies_commit();
    };
    issue(0);
    issue(1);
    if (at.size > 1) cg::this_cluster().sync();  // every CTA runs before another writes to it
    Joiner<NW, 1> joiner{ex, at, W, wt, wr, warp, 0};
    const int run = (BACKWARD ? SUB - 1 - ls : ls) * kRun;  // this thread's run within its row's tile
    Watch watch;
    int stage = 0;
    for (int64_t unit = at.first; unit < a.units; unit += at.clusters) {
        const Rows here = rows_of(unit);
        const int seg = here.seg;
        const int64_t row0 = here.row0, row = row0 + sr;
        const bool live = row < a.lanes;
        float c = 0.0f, gates = 1.0f;
        if constexpr (PASS == MAPS) watch = Watch();  // (a unit's own)
        if constexpr (PASS == JOINED) {
            if (live && a.in[SI_CARRY].p) c = __ldg(a.in[SI_CARRY].p + row * a.in[SI_CARRY].so);
            c = segment_state<NW, 1>(a, ex, seg, row, live, c, warp, 0, l == 0, watch);
        }
        Count r0 = static_cast<Count>(here.begin + own);
        for (int k = 0; k < a.steps; ++k, stage ^= 1, r0 += static_cast<Count>(stride)) {
            const Cutout cut = cutout(row, static_cast<Count>(here.end), r0);
            const Count t0 = 4 * cut.v0 - cut.shift + run;  // the run's first step in memory
            copies_wait_one();
            __syncwarp();
            if (SUB == 32 && cut.n == 0) {  // the axis ended before this warp's tile
                if (PASS == ONLY && k == 0) c = a.in[SI_CARRY].p && live ? tile.carry[stage][0] : 0.0f;
                __syncwarp();
                issue(stage);
                const float s = joiner.first(make_float2(1.0f, 0.0f), c, k == 0, l == 0, watch);
                if constexpr (PASS == MAPS) {
                    joiner.gates_of_step(gates, watch);
                    const int range = k + 1 == a.steps ? block_range(ex, watch.range()) : 0;
                    if (k + 1 == a.steps && live && wt == W - 1 && l == 0) a.maps[seg * a.lanes + row] = segment_map(gates, s, range);
                }
                joiner.hand_on(s, k + 1 == a.steps, l == 0);
                continue;
            }
            const int at_run = sr * SUB * kRun + run;
            float ga[kRun], xv[kRun], hv[BACKWARD ? kRun : 1];
#pragma unroll
            for (int j = 0; j < kRun; j += 4) {
                load_shared<4>(&tile.in[stage][0][at_run + j], ga + j);
                load_shared<4>(&tile.in[stage][1][at_run + j], xv + j);
            }
            if constexpr (BACKWARD) {
                if (want_gate) {  // the state before each step
                    const float* q = h_row(stage, sr) + run;
                    float h[kRun];
#pragma unroll
                    for (int j = 0; j < kRun; j += 4) load_shared<4>(q + j, h + j);
                    hv[0] = q[-1];
#pragma unroll
                    for (int j = 1; j < kRun; ++j) hv[j] = h[j - 1];
                }
            }
            // steps [in0, in1) of the run are inside the tile and the row: the others leave the state as it is
            const int in0 = max(4 * cut.lo - run, t0 < 0 ? static_cast<int>(max(t0, static_cast<Count>(-kRun))) * -1 : 0);
            const int in1 = min(4 * (cut.lo + cut.n) - run, static_cast<int>(min(static_cast<Count>(a.T) - t0, static_cast<Count>(kRun))));
            if (in0 > 0 || in1 < kRun) {
#pragma unroll
                for (int j = 0; j < kRun; ++j) {
                    const bool inside = j >= in0 && j < in1;
                    ga[j] = inside ? ga[j] : 1.0f;
                    xv[j] = inside ? xv[j] : 0.0f;
                }
            }
            if (!a.in[SI_X].p) {
#pragma unroll
                for (int j = 0; j < kRun; ++j) xv[j] = 0.0f;
            }
            if (PASS == ONLY && k == 0) c = a.in[SI_CARRY].p && live ? tile.carry[stage][sr] : 0.0f;
            __syncwarp();
            issue(stage);
            float2 q = tile_map<BACKWARD, kRun>([&](int j) { return ga[BACKWARD ? kRun - 1 - j : j]; },
                                                [&](int j) { return xv[BACKWARD ? kRun - 1 - j : j]; });
            watch.runs(q.x, q.x);
#pragma unroll
            for (int d = 1; d < SUB; d *= 2) {
                const float2 b = make_float2(__shfl_up_sync(0xffffffffu, q.x, d), __shfl_up_sync(0xffffffffu, q.y, d));
                const float2 n = join(b, q);
                q = ls >= d ? n : q;
            }
            const float2 b = make_float2(__shfl_up_sync(0xffffffffu, q.x, 1), __shfl_up_sync(0xffffffffu, q.y, 1));
            const bool last = k + 1 == a.steps;
            float s = c;
            if constexpr (SUB == 32) {
                const float2 m = make_float2(__shfl_sync(0xffffffffu, q.x, 31), __shfl_sync(0xffffffffu, q.y, 31));
                s = joiner.first(m, c, k == 0, l == 0, watch);
                if constexpr (PASS == MAPS) {
                    joiner.gates_of_step(gates, watch);
                    s = apply(m, s);
                    const int range = last ? block_range(ex, watch.range()) : 0;
                    if (last && live && wt == W - 1 && l == 0) a.maps[seg * a.lanes + row] = segment_map(gates, s, range);
                    joiner.hand_on(s, last, l == 0);
                    continue;
                }
            }
            if constexpr (SUB < 32) {
                watch.tile_of(q.x);
                watch.states(q.y, s);
            }
            float y = ls > 0 ? apply(b, s) : s;
            // results over the inputs' registers: x becomes h or dx, h becomes dgate
            if constexpr (BACKWARD) {
#pragma unroll
                for (int j = kRun - 1; j >= 0; --j) {
                    xv[j] += y;
                    y = ga[j] * xv[j];
                    if (want_gate) hv[j] *= xv[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < kRun; ++j) xv[j] = y = fmaf(ga[j], y, xv[j]);
            }
            auto write = [&](float* out, const float* v) {
                float* to = &tile.out[sr * SUB * kRun + run];
#pragma unroll
                for (int j = 0; j < kRun; j += 4) *reinterpret_cast<float4*>(to + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                __syncwarp();
                if constexpr (SUB == 32) {
                    float* to_g = out + row * a.T + 4 * cut.v0 - cut.shift + 4 * l;
                    auto move = [&](unsigned in) {
#pragma unroll
                        for (int u = 0; u < kVectors / 32; ++u) {
                            float f[4];
                            load_shared<4>(&tile.out[4 * l + 128 * u], f);
                            if (in >> u & 1) store_vec<4>(to_g + 128 * u, f, BACKWARD);
                        }
                    };
                    if (whole_tile(cut)) {
                        move(~0u);
                    } else {
                        move(inside_vectors(cut));
                        Count t;
                        const int e = edge(cut, t);
                        if (e >= 0) out[row * a.T + t] = tile.out[e];
                    }
                } else {
#pragma unroll 1
                    for (int u = 0; u < kVectors / 32; ++u) {
                        const int at_v = l + 32 * u, v = at_v % VR;
                        const int64_t r = row0 + at_v / VR;
                        const Cutout e = cutout(r, static_cast<Count>(here.end), r0);
                        if (v < e.lo || v >= e.lo + e.n) continue;
                        const Count t = 4 * (e.v0 + v) - e.shift;
                        float f[4];
                        load_shared<4>(&tile.out[4 * at_v], f);
                        if (t >= 0 && t + 3 < a.T) {
                            store_vec<4>(out + r * a.T + t, f, BACKWARD);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (t + j >= 0 && t + j < a.T) out[r * a.T + t + j] = f[j];
                        }
                    }
                }
                __syncwarp();
            };
            if (a.out[SO_MAIN]) write(a.out[SO_MAIN], xv);
            if constexpr (BACKWARD) {
                if (want_gate) write(a.out[SO_GATE], hv);
            }
            // behind the tile's last run
            if (SUB == 32) s = __shfl_sync(0xffffffffu, y, 31);
            if (live && cut.n > 0 && r0 + cut.n == cut.vectors && ls == SUB - 1 && a.out[SO_LANE]) a.out[SO_LANE][row] = y;
            if constexpr (SUB == 32) joiner.hand_on(s, last, l == 0);
        }
    }
    copies_wait_all();
    if constexpr (PASS != MAPS) settle<BACKWARD, kRowCut<SUB>>(a, ex, at, watch, NW / W * R);
}

// ---- a few steps (a token for each of many sequences): a thread walks V lanes, nothing to join.
// A token of 64 x 4096 lanes: 7 us, most of it a launch's latency.
constexpr int kShort = 16;

template <bool BACKWARD, int V>
__global__ void __launch_bounds__(256) scan_short_kernel(ScanArgs a) {
    const int64_t lane = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * V;
    if (lane >= a.lanes) return;
    int64_t o, i;
    split_lane(a, lane, o, i);
    int64_t i1, i2;
    split_inner(a, i, i1, i2);
    auto ptr = [&](int k) { return a.in[k].p ? a.in[k].p + o * a.in[k].so + i1 * a.in[k].s1 + i2 * a.in[k].s2 : nullptr; };
    const float *gate = ptr(SI_GATE), *x = ptr(SI_X), *carry = ptr(SI_CARRY), *h = ptr(SI_H), *init = ptr(SI_INIT);
    auto load = [&](const float* p, int k, float* v) {
        if (V > 1 && (a.vec >> k & 1)) {
            load_shared<V>(p, v);
        } else {
#pragma unroll
            for (int u = 0; u < V; ++u) v[u] = p[u * a.in[k].s2];
        }
    };
    float s[V];
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = 0.0f;
    if (carry) load(carry, SI_CARRY, s);
    const int T = static_cast<int>(a.T);
    const int64_t y0 = o * a.T * a.inner + i;
    for (int r0 = 0; r0 < T; r0 += 4) {
        float ga[4][V], xv[4][V], hv[BACKWARD ? 4 : 1][V];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int t = BACKWARD ? T - 1 - r0 - j : r0 + j;
            if (r0 + j >= T) continue;
            load(gate + t * a.in[SI_GATE].st, SI_GATE, ga[j]);
#pragma unroll
            for (int v = 0; v < V; ++v) xv[j][v] = 0.0f;
            if (x) load(x + t * a.in[SI_X].st, SI_X, xv[j]);
            if (BACKWARD) {
#pragma unroll
                for (int v = 0; v < V; ++v) hv[j][v] = 0.0f;
                if (a.out[SO_GATE]) {
                    if (t > 0) load(h + (t - 1) * a.in[SI_H].st, SI_H, hv[j]);
                    else if (init) load(init, SI_INIT, hv[j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (r0 + j >= T) continue;
            const int64_t y = y0 + (BACKWARD ? T - 1 - r0 - j : r0 + j) * a.inner;
            float main[V], dg[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (BACKWARD) {
                    main[v] = xv[j][v] + s[v];
                    dg[v] = main[v] * hv[BACKWARD ? j : 0][v];
                    s[v] = ga[j][v] * main[v];
                } else {
                    main[v] = s[v] = fmaf(ga[j][v], s[v], xv[j][v]);
                }
            }
            if (a.out[SO_MAIN]) store_vec<V>(a.out[SO_MAIN] + y, main, false);
            if (BACKWARD && a.out[SO_GATE]) store_vec<V>(a.out[SO_GATE] + y, dg, false);
        }
    }
    if (a.out[SO_LANE]) store_vec<V>(a.out[SO_LANE] + lane, s, false);
}

// Of the lanes that dgate is summed over, those that a warp sums: groups that do not line up with warps are
// summed by a second launch alone.
int64_t warp_group(const ScanDesc& d) {
    const int64_t g = d.group;
    return g % 32 == 0 ? 32 : g == 2 || g == 4 || g == 8 || g == 16 ? g : 1;
}

// The widest vectors of lanes: every operand has adjacent lanes behind n1 whose vectors are
// aligned wherever they start (buffers start on 16 bytes), or is broadcast over them.
int widest(const ScanDesc& d) {
    for (int v = 4; v > 1; v /= 2) {
        bool ok = d.n2 % v == 0 && (warp_group(d) == 1 || d.group % v == 0);
        for (int k = 0; k < SI_COUNT && ok; ++k) {
            const ScanStrides& s = d.in[k];  // (all 0 where absent)
            if (s.s2 == 0) continue;
            ok = s.s2 == 1 && s.so % v == 0 && s.st % v == 0 && s.s1 % v == 0 && s.off % v == 0;
        }
        if (ok) return v;
    }
    return 1;
}

// How a scan is cut: threads of a row, lanes per thread, warps along time, CTAs of a cluster along
// time, segments.
struct Cut {
    bool rows, direct;
    int sub = 32, V = 1, tile = 16, warps = kWarps, W = 1, cluster = 1, segments = 1;
    int64_t seg_len = 1, blocks = 0, steps = 0;
};

Cut cut(const ScanDesc& d) {
    Cut c;
    const int64_t inner = d.n1 * d.n2, lanes = d.outer * inner;
    // (no steps: the first state alone is handed through, whatever the groups)
    c.direct = d.T == 0 || (d.T <= kShort && warp_group(d) == 1);
    c.rows = inner == 1 && !c.direct;  // (no groups there: they are lanes)
    if (inner > 1) c.V = widest(d);
    if (c.direct) {
        // (a few lanes only: one each, for more threads)
        if (lanes < 148 * 256 * c.V) c.V = 1;
        c.blocks = (lanes + 256 * c.V - 1) / (256 * c.V);
        return c;
    }
    // rows count time in vectors of four, from the boundary at or before their first step on: at most `cut` less
    // the power of two that divides both T and it
    auto row_vectors = [&](int64_t cut) {
        int64_t two = cut;
        while (d.T % two != 0) two /= 2;
        return (d.T + cut - two + cut - 1) / cut * (cut / 4);
    };
    int64_t len = c.rows ? row_vectors(kRowCut<4>) : d.T;
    const int run = d.backward ? kRowRun<true> : kRowRun<false>;
    while (c.rows && c.sub > 4 && len <= c.sub / 2 * run / 4) c.sub /= 2;
    if (c.rows) c.tile = c.sub * run / 4;
    if (c.rows && c.sub == 32) len = row_vectors(kRowCut<32>);
    auto warps = [&](int64_t t) {  // along time
        int w = 1;
        while (w < kWarps && w * t < len) w *= 2;
        return w;
    };
    auto padded = [&](int64_t t) { return (len + warps(t) * t - 1) / (warps(t) * t) * warps(t) * t; };
    // 24 steps a tile are faster than 16 (fewer exchanges: 39 against 49 us for 8 x 2048 x 1024), unless
    // they pad the axis by a tenth more
    if (!c.rows && !d.backward && 10 * padded(24) <= 11 * padded(16)) c.tile = 24;
    const int64_t tile = c.tile;
    c.W = warps(tile);
    const int64_t groups = c.rows ? (lanes + 32 / c.sub - 1) / (32 / c.sub) : (lanes + 31) / 32;
    c.blocks = (groups + kWarps / c.W - 1) / (kWarps / c.W);
    // More CTAs along time while the blocks leave a quarter of the SMs idle and every CTA has a step of its
    // own, and only as many as run at the same time (two an SM, in clusters within the GPCs).  T = 2048,
    // 1024 lanes a sequence: 4 sequences 23 us with 1 CTA, 27 with 2; 2 sequences 22 with 1, 18 with 4;
    // 1 sequence 22 with 1, 14 with 8.
    if (c.blocks < 112)
        while (c.W == kWarps && c.cluster < 8 && c.blocks * c.cluster * 2 <= (c.cluster < 4 ? 280 : 256) &&
               c.cluster * c.W * tile * 2 <= len)
            c.cluster *= 2;
    // backward, a CTA an SM: 16 warps a CTA, twice the steps in flight (4 x 2048 x 1024: 33 against 38 us;
    // forward, with 24 steps a tile, 25 against 23)
    if (d.backward && c.V == 4 && c.W == kWarps && c.blocks >= 112 && c.blocks <= 148 && 16 * tile <= len) c.warps = c.W = 16;
    c.seg_len = len;
    if (c.blocks * c.cluster < 112 && len > c.cluster * c.W * tile) {
        c.cluster = 1;
        const int64_t step = c.W * tile, most = (len + step - 1) / step;
        int64_t want = (296 + c.blocks - 1) / c.blocks;
        if (want > most) want = most;
        c.seg_len = ((len + want - 1) / want + step - 1) / step * step;
        c.segments = static_cast<int>((len + c.seg_len - 1) / c.seg_len);
    }
    const int64_t span = c.cluster * c.W * tile;
    c.steps = (c.seg_len + span - 1) / span;
    return c;
}

template <auto Kernel, int NW = kWarps>
cudaError_t launch_kernel(size_t smem, const Cut& c, const ScanArgs& a, cudaStream_t stream) {
    static std::atomic<int> resident[64];  // CTAs that run at the same time, by device; 0: not found yet
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    int slots = dev < 64 ? resident[dev].load() : 0;
    if (slots == 0) {
        e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        int sms = 0;
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&slots, Kernel, NW * 32, smem);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
        slots *= sms;
        if (slots < 1) return cudaErrorInvalidConfiguration;
        if (dev < 64) resident[dev] = slots;
    }
    const int64_t clusters = c.cluster > 1 || a.units < slots ? a.units : slots;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * c.cluster));
    cfg.blockDim = dim3(NW * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(c.cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = c.cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, Kernel, a);
}

template <bool BACKWARD, int PASS, int TILE>
cudaError_t launch_cols(const Cut& c, const ScanArgs& a, cudaStream_t stream) {
    constexpr size_t smem = sizeof(ColTile<BACKWARD, TILE, kWarps>);
    if constexpr (PASS == ONLY && BACKWARD) {
        if (c.warps == 16)
            return launch_kernel<scan_cols_kernel<BACKWARD, PASS, 4, TILE, 16>, 16>(sizeof(ColTile<BACKWARD, TILE, 16>), c, a, stream);
    }
    if (c.V == 4) return launch_kernel<scan_cols_kernel<BACKWARD, PASS, 4, TILE, kWarps>>(smem, c, a, stream);
    if (c.V == 2) return launch_kernel<scan_cols_kernel<BACKWARD, PASS, 2, TILE, kWarps>>(smem, c, a, stream);
    return launch_kernel<scan_cols_kernel<BACKWARD, PASS, 1, TILE, kWarps>>(smem, c, a, stream);
}

template <bool BACKWARD, int PASS>
cudaError_t launch_pass(const Cut& c, const ScanArgs& a, cudaStream_t stream) {
    if (c.rows) {
        if constexpr (PASS == ONLY) {
            if (c.sub == 4) return launch_kernel<scan_rows_kernel<BACKWARD, PASS, 4>>(rows_smem<BACKWARD>(), c, a, stream);
            if (c.sub == 8) return launch_kernel<scan_rows_kernel<BACKWARD, PASS, 8>>(rows_smem<BACKWARD>(), c, a, stream);
            if (c.sub == 16) return launch_kernel<scan_rows_kernel<BACKWARD, PASS, 16>>(rows_smem<BACKWARD>(), c, a, stream);
        }
        return launch_kernel<scan_rows_kernel<BACKWARD, PASS, 32>>(rows_smem<BACKWARD>(), c, a, stream);
    }
    if constexpr (!BACKWARD) {
        if (c.tile == 24) return launch_cols<BACKWARD, PASS, 24>(c, a, stream);
    }
    return launch_cols<BACKWARD, PASS, 16>(c, a, stream);
}

template <bool BACKWARD>
cudaError_t launch_cut(const Cut& c, const ScanArgs& a, cudaStream_t stream) {
    if (c.direct) {
        const dim3 grid(static_cast<unsigned>(c.blocks));
        if (c.V == 4) scan_short_kernel<BACKWARD, 4><<<grid, 256, 0, stream>>>(a);
        else if (c.V == 2) scan_short_kernel<BACKWARD, 2><<<grid, 256, 0, stream>>>(a);
        else scan_short_kernel<BACKWARD, 1><<<grid, 256, 0, stream>>>(a);
        return cudaGetLastError();
    }
    if (c.segments == 1) return launch_pass<BACKWARD, ONLY>(c, a, stream);
    const cudaError_t e = launch_pass<BACKWARD, MAPS>(c, a, stream);
    return e != cudaSuccess ? e : launch_pass<BACKWARD, JOINED>(c, a, stream);
}

// dgate of groups of lanes from the sums of a warp's lanes, or from all lanes, in order and in double: a thread
// a sum, or a warp where a thread would walk far.  4 x 2048 x 16 heads of 64: 4 us, a launch; 26 x 4487 x 8 heads
// of 3 8 us, 4 x 56527 heads of 37 14 us.
__global__ void __launch_bounds__(256) gate_group_kernel(const float* __restrict__ part, float* __restrict__ out, int64_t n, int parts) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= n) return;
    double s = 0.0;
    for (int k = 0; k < parts; ++k) s += static_cast<double>(__ldg(part + i * parts + k));
    out[i] = static_cast<float>(s);
}
__global__ void __launch_bounds__(256) gate_group_warp_kernel(const float* __restrict__ part, float* __restrict__ out, int64_t n, int64_t parts) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (i >= n) return;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    const float* p = part + i * parts;
    int64_t k = threadIdx.x & 31;
    for (; k + 96 < parts; k += 128)
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] += static_cast<double>(__ldg(p + k + 32 * u));
    for (; k < parts; k += 32) s[0] += static_cast<double>(__ldg(p + k));
    double t = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int d = 16; d > 0; d /= 2) t += __shfl_xor_sync(0xffffffffu, t, d);
    if ((threadIdx.x & 31) == 0) out[i] = static_cast<float>(t);
}
cudaError_t sum_groups(const float* part, float* out, int64_t n, int64_t parts, cudaStream_t stream) {
    const bool thread = parts <= 64;
    const int64_t blocks = thread ? (n + 255) / 256 : (n + 7) / 8;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (thread) gate_group_kernel<<<grid, 256, 0, stream>>>(part, out, n, static_cast<int>(parts));
    else gate_group_warp_kernel<<<grid, 256, 0, stream>>>(part, out, n, parts);
    return cudaGetLastError();
}

int64_t maps_bytes(const ScanDesc& d, const Cut& c) {
    const int64_t b = c.segments > 1 ? c.segments * d.outer * d.n1 * d.n2 * static_cast<int64_t>(sizeof(float2)) : 0;
    return (b + 255) / 256 * 256;
}
int64_t group_parts(const ScanDesc& d) { return d.group / warp_group(d); }

}  // namespace

int64_t scan_scratch_bytes(const ScanDesc& d) {
    const int64_t sums = group_parts(d) > 1 ? d.outer * d.T * (d.n1 * d.n2 / warp_group(d)) * static_cast<int64_t>(sizeof(float)) : 0;
    return maps_bytes(d, cut(d)) + sums;
}

int scan_launch_count(const ScanDesc& d) {
    if (d.outer * d.n1 * d.n2 == 0) return 0;
    return (cut(d).segments > 1 ? 2 : 1) + (group_parts(d) > 1 && d.T > 0 ? 1 : 0);
}

int launch_scan(const ScanDesc& d, const float* const* in, float* const* out, void* scratch, void* stream) {
    const int64_t lanes = d.outer * d.n1 * d.n2;
    if (lanes == 0) return 0;
    const Cut c = cut(d);
    if (c.blocks * c.segments > 0x7fffffff / 8 || c.steps > 0x7fffffff || c.seg_len > 0x7f000000) return static_cast<int>(cudaErrorInvalidConfiguration);
    ScanArgs a;
    a.vec = 0;
    for (int k = 0; k < SI_COUNT; ++k) {
        const ScanStrides& s = d.in[k];
        a.in[k] = Operand{in[k] ? in[k] + s.off : nullptr, s.so, s.st, s.s1, s.s2};
        // rows: every row starts at the same place within 16 bytes as the result's
        if (c.rows ? s.st == 1 && s.off % 4 == 0 && (s.so - d.T) % 4 == 0 : s.s2 == 1) a.vec |= 1 << k;
    }
    for (int k = 0; k < SO_COUNT; ++k) a.out[k] = out[k];
    const bool sums = out[SO_GATE] && group_parts(d) > 1;
    if (sums) a.out[SO_GATE] = reinterpret_cast<float*>(static_cast<char*>(scratch) + maps_bytes(d, c));
    a.maps = static_cast<float2*>(scratch);
    a.lanes = lanes;
    a.inner = d.n1 * d.n2;
    a.n2 = d.n2;
    a.T = d.T;
    a.seg_len = c.seg_len;
    a.segments = c.segments;
    a.group = 0;
    while (1 << a.group < warp_group(d)) ++a.group;
    a.units = c.blocks * c.segments;
    a.steps = static_cast<int>(c.steps);
    a.W = c.W;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = d.backward ? launch_cut<true>(c, a, st) : launch_cut<false>(c, a, st);
    if (e == cudaSuccess && sums && d.T > 0) {
        e = sum_groups(a.out[SO_GATE], out[SO_GATE], lanes / d.group * d.T, group_parts(d), st);
    }
    return static_cast<int>(e);
}

}  // namespace ttb
