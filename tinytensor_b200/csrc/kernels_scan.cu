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
// the tiles of this step wait for one another's maps.  Tiles are joined in time order, so
// results do not depend on how CTAs are scheduled, at three levels:
//   warps of a CTA        through shared memory, one block barrier a step;
//   CTAs of a cluster     through distributed shared memory, one cluster barrier a step,
//                         where there are too few lanes to fill the card;
//   segments of the axis  through device scratch, by a first launch that finds the segments'
//                         maps, where clusters are not enough (the data is read twice).
// Time runs in scan order r: t = r forward, t = T-1-r backward.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "program.hpp"

namespace cg = cooperative_groups;

namespace ttb {

namespace {

constexpr int NW = 8;  // warps of a CTA

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
    int W;            // warps of a CTA along time; the others take further lanes
    int vec;          // bit k: operand k moves as vectors
};

enum Pass { ONLY = 0, MAPS = 1, JOINED = 2 };  // the whole scan; its segments' maps; the scan from them

// The map (A, H) applied to c.  A state of exactly 0 takes no part: the gates' product may
// have overflowed, and inf * 0 is NaN where the recurrence stays 0.
__device__ __forceinline__ float apply(float2 m, float c) { return c == 0.0f ? m.y : fmaf(m.x, c, m.y); }

// Product of gates.  A zero gate makes it zero whatever overflowed before; a product that
// underflows stays the smallest number, so that an infinite state stays infinite.
__device__ __forceinline__ float join_gates(float a, float b) {
    const float p = a * b;
    if (a == 0.0f || b == 0.0f) return 0.0f;
    return p == 0.0f ? copysignf(1.4e-45f, p) : p;
}

// First m, then n.
__device__ __forceinline__ float2 join(float2 m, float2 n) { return make_float2(join_gates(m.x, n.x), apply(n, m.y)); }

// The map of N steps in scan order.  Gates are multiplied plainly; where that gave NaN, a zero
// gate among them settles it (after an overflow 0 * inf).
template <bool BACKWARD, int N, class G, class X>
__device__ __forceinline__ float2 tile_map(G gate, X x) {
    float2 m = make_float2(gate(0), BACKWARD ? gate(0) * x(0) : x(0));
#pragma unroll
    for (int j = 1; j < N; ++j) {
        m.x *= gate(j);
        m.y = BACKWARD ? gate(j) * (x(j) + m.y) : fmaf(gate(j), m.y, x(j));
    }
    if (m.x != m.x) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (gate(j) == 0.0f) m.x = 0.0f;
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
template <int LW>  // lanes of a warp's tile
struct Exchange {
    float2 warp[2][NW][LW];
    // only where W = NW (otherwise one step covers the axis):
    float2 cta[2][8][LW];  // by rank in the cluster
    float state[2][LW];    // the last warp's state behind a step, for the next one
};

// Where a CTA works: its block of lanes, segment of the axis and place in its cluster.
struct Place {
    int64_t block;
    int seg, rank, size;
};
__device__ __forceinline__ Place place(const ScanArgs& a) {
    Place p;
    cg::cluster_group cl = cg::this_cluster();
    p.size = static_cast<int>(cl.num_blocks());
    p.rank = static_cast<int>(cl.block_rank());
    const unsigned unit = blockIdx.x / p.size;
    p.seg = static_cast<int>(unit % a.segments);
    p.block = unit / a.segments;
    return p;
}

// The state before a segment.
template <int PASS>
__device__ __forceinline__ float segment_state(const ScanArgs& a, int seg, int64_t lane, const float* carry) {
    float c = 0.0f;
    if (PASS != MAPS && carry) c = __ldg(carry);
    if constexpr (PASS == JOINED)
        for (int s = 0; s < seg; ++s) c = apply(a.maps[s * a.lanes + lane], c);
    return c;
}

// A CTA's part in the exchange, one lane per thread: thread l of a warp handles lane l of its
// tile (LW = 32), or all threads the tile's one row (LW = 1; `writer` is one of them).
template <int LW>
struct Joiner {
    Exchange<LW>& ex;
    const Place& at;
    int W, wt, wr, warp, l;
    int buf = 0;

    // m: the map of this warp's tile.  Returns the state before the tile; c is the state before
    // the first step (later steps find theirs in the exchange).
    __device__ __forceinline__ float first(float2 m, float c, bool first_step, bool writer) {
        if (writer) ex.warp[buf][warp][l] = m;
        __syncthreads();
        if (at.size > 1) {
            cg::cluster_group cl = cg::this_cluster();
            if (wt == 0 && writer) {
                float2 all = m;
#pragma unroll
                for (int w = 1; w < NW; ++w) all = join(all, ex.warp[buf][w][l]);
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
#pragma unroll
        for (int w = 0; w < NW - 1; ++w)
            if (w < wt) s = apply(ex.warp[buf][wr * W + w][l], s);
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
    __device__ __forceinline__ void gates_of_step(float& gates) const {
#pragma unroll
        for (int w = 0; w < NW; ++w) gates = join_gates(gates, ex.warp[buf][w][l].x);
    }
};

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

// ---- lanes side by side in memory ([.., T, lanes]): a warp's tile is 16 steps of 32 adjacent
// lanes.  A thread takes V adjacent lanes and 16/V adjacent steps (32/V threads lie across the
// lanes, V behind one another in time), so that operands move in 4*V bytes a thread and 128
// bytes a row whatever V is; the V threads of a lane join their maps by shuffles.  Operands
// whose lanes are adjacent move as V-vectors, operands broadcast over the lanes behind n1 as one
// value (V > 1 is only cut where each operand is one or the other); V = 1 takes any strides.
// A thread reads back only what it copied itself, so the ring needs no barrier.
constexpr int kTileSteps = 16;

template <bool BACKWARD>
constexpr int kArrays = BACKWARD ? 3 : 2;

template <bool BACKWARD>
constexpr size_t cols_smem() {
    return sizeof(Exchange<32>) + 2 * kArrays<BACKWARD> * NW * kTileSteps * 32 * sizeof(float);
}

template <bool BACKWARD, int PASS, int V>
__global__ void __launch_bounds__(NW * 32, BACKWARD ? 2 : 3) scan_cols_kernel(ScanArgs a) {
    constexpr int TS = kTileSteps / V, COLS = 32 / V, NA = kArrays<BACKWARD>;
    extern __shared__ __align__(16) unsigned char raw[];
    float* ring = reinterpret_cast<float*>(raw);  // [stage][operand][warp][step][thread][V]
    Exchange<32>& ex = *reinterpret_cast<Exchange<32>*>(raw + 2 * NA * NW * kTileSteps * 32 * sizeof(float));
    const Place at = place(a);
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31, W = a.W;
    const int wt = warp % W, wr = warp / W;
    const int col = l % COLS, sub = l / COLS;
    const int64_t lane0 = (at.block * (NW / W) + wr) * 32, lane = lane0 + col * V;
    const bool live = lane < a.lanes;
    int64_t o = 0, i = 0;
    if (live) {
        if (a.lanes <= 0x7fffffff) {
            const unsigned q = static_cast<unsigned>(lane), n = static_cast<unsigned>(a.inner);
            o = q / n;
            i = q % n;
        } else {
            o = lane / a.inner;
            i = lane % a.inner;
        }
    }
    const int64_t i1 = a.n2 == a.inner ? 0 : i / a.n2, i2 = i - i1 * a.n2;
    const float* p[SI_COUNT];
#pragma unroll
    for (int k = 0; k < SI_COUNT; ++k)
        p[k] = a.in[k].p ? a.in[k].p + o * a.in[k].so + i1 * a.in[k].s1 + i2 * a.in[k].s2 : nullptr;
    const bool want_gate = BACKWARD && PASS != MAPS && a.out[SO_GATE];
    const int64_t begin = at.seg * a.seg_len, end = min(a.T, begin + a.seg_len);
    const int64_t stride = static_cast<int64_t>(at.size) * W * kTileSteps;  // of this warp's tiles
    const int64_t own = begin + (static_cast<int64_t>(at.rank) * W + wt) * kTileSteps + sub * TS;
    auto run_len = [&](int64_t r0) {
        return live ? static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(TS), end - r0))) : 0;
    };
    auto slot = [&](int stage, int k) { return ring + (((stage * NA + k) * NW + warp) * kTileSteps * 32 + l * V); };
    // copies of one operand: n steps in scan order from time t on
    auto fetch = [&](int k, int stage, int arr, int64_t t, int n) {
        const int64_t step = BACKWARD ? -a.in[k].st : a.in[k].st;
        const float* q = p[k] + t * a.in[k].st;
        const uint32_t dst = smem_addr(slot(stage, arr));
        if (V > 1 && (a.vec >> k & 1)) {
#pragma unroll
            for (int j = 0; j < TS; ++j, q += step)
                if (j < n) copy_async<4 * V>(dst + j * 128 * V, q);
        } else {
#pragma unroll
            for (int j = 0; j < TS; ++j, q += step)
                if (j < n) copy_async<4>(dst + j * 128 * V, q);
        }
    };
    auto issue = [&](int64_t r0, int stage) {
        const int n = run_len(r0);
        const int64_t t = BACKWARD ? a.T - 1 - r0 : r0;
        if (n > 0) {
            fetch(SI_GATE, stage, 0, t, n);
            if (p[SI_X]) fetch(SI_X, stage, 1, t, n);
            // the states before each step; before t = 0 there is init
            if (want_gate) fetch(SI_H, stage, NA - 1, t - 1, static_cast<int>(min(static_cast<int64_t>(n), t)));
        }
        copies_commit();
    };
    issue(own, 0);
    issue(own + stride, 1);
    if (at.size > 1) cg::this_cluster().sync();  // every CTA runs before another writes to it

    // the exchange takes lane lane0 + l: its state before the segment
    float c = 0.0f;
    if (lane0 + l < a.lanes) {
        const float* q = nullptr;
        if (p[SI_CARRY]) {
            const int64_t ol = (lane0 + l) / a.inner, il = (lane0 + l) % a.inner;
            q = a.in[SI_CARRY].p + ol * a.in[SI_CARRY].so + il / a.n2 * a.in[SI_CARRY].s1 + il % a.n2 * a.in[SI_CARRY].s2;
        }
        c = segment_state<PASS>(a, at.seg, lane0 + l, q);
    }
    if (a.T == 0) {  // no steps: the last state is the first
        copies_wait_all();
        if (lane0 + l < a.lanes && wt == 0 && a.out[SO_LANE]) a.out[SO_LANE][lane0 + l] = c;
        return;
    }
    Joiner<32> joiner{ex, at, W, wt, wr, warp, l};
    float gates = 1.0f;
    const bool splat_gate = V > 1 && !(a.vec >> SI_GATE & 1), splat_x = V > 1 && !(a.vec >> SI_X & 1);
    const bool splat_h = V > 1 && !(a.vec >> SI_H & 1);
    int stage = 0;
    for (int64_t base = begin; base < end; base += stride, stage ^= 1) {
        const int64_t r0 = own + (base - begin);
        const int n = run_len(r0);
        float ga[TS][V], xv[TS][V], hv[BACKWARD ? TS : 1][V];
        copies_wait_one();
        auto read = [&](const float* q, bool splat, int count, float none, float (*dst)[V]) {
#pragma unroll
            for (int j = 0; j < TS; ++j) {
                if (splat) {
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
        read(slot(stage, 0), splat_gate, n, 1.0f, ga);
        read(slot(stage, 1), splat_x, p[SI_X] ? n : 0, 0.0f, xv);
        if constexpr (BACKWARD) {
            const int64_t t0 = a.T - 1 - r0;
            const int nh = want_gate ? static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(n), t0))) : 0;
            read(slot(stage, NA - 1), splat_h, nh, 0.0f, hv);
            if (want_gate && nh < n && p[SI_INIT]) {
#pragma unroll
                for (int j = 0; j < TS; ++j)
                    if (j == nh)
#pragma unroll
                        for (int v = 0; v < V; ++v) hv[j][v] = __ldg(p[SI_INIT] + v * a.in[SI_INIT].s2);
            }
        }
        issue(r0 + 2 * stride, stage);
        // this thread's maps, those of the threads before it in time, and the tile's
        float2 m[V], before[V];
        float2 tile = make_float2(1.0f, 0.0f);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            m[v] = tile_map<BACKWARD, TS>([&](int j) { return ga[j][v]; }, [&](int j) { return xv[j][v]; });
            before[v] = make_float2(1.0f, 0.0f);
#pragma unroll
            for (int d = COLS; d < 32; d *= 2) {
                const float2 b = make_float2(__shfl_up_sync(0xffffffffu, m[v].x, d), __shfl_up_sync(0xffffffffu, m[v].y, d));
                if (l >= d) m[v] = join(b, m[v]);
            }
            if (V > 1) {
                const float2 b = make_float2(__shfl_up_sync(0xffffffffu, m[v].x, COLS), __shfl_up_sync(0xffffffffu, m[v].y, COLS));
                if (sub > 0) before[v] = b;
                // lane l's map lies with the last of its threads, 32 - COLS + l / V, at v = l % V
                const float2 w = make_float2(__shfl_sync(0xffffffffu, m[v].x, 32 - COLS + l / V),
                                             __shfl_sync(0xffffffffu, m[v].y, 32 - COLS + l / V));
                if (l % V == v) tile = w;
            } else {
                tile = m[v];
            }
        }
        const float first = joiner.first(tile, c, base == begin, true);
        const bool last_step = base + stride >= end;
        if constexpr (PASS == MAPS) {
            joiner.gates_of_step(gates);
            const float s = apply(tile, first);
            if (last_step && lane0 + l < a.lanes && wt == W - 1) a.maps[at.seg * a.lanes + lane0 + l] = make_float2(gates, s);
            joiner.hand_on(s, last_step, true);
        } else {
            float s[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                s[v] = V > 1 ? __shfl_sync(0xffffffffu, first, col * V + v) : first;
                if (V > 1 && sub > 0) s[v] = apply(before[v], s[v]);
            }
            const int64_t step = BACKWARD ? -a.inner : a.inner;
            const int64_t y = (o * a.T + (BACKWARD ? a.T - 1 - r0 : r0)) * a.inner + i;
            float* ym = a.out[SO_MAIN] + y;
            float* yg = a.out[SO_GATE] + y;
            const int nm = a.out[SO_MAIN] ? n : 0, ng = want_gate ? n : 0;
#pragma unroll
            for (int j = 0; j < TS; ++j, ym += step, yg += step) {  // (past the end: gate 1, x 0, the state stays)
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
                if (j < ng) store_vec<V>(yg, dg, true);
            }
            // the thread of the last step has the last state as it was stored
            if (n > 0 && r0 + n == a.T && a.out[SO_LANE]) store_vec<V>(a.out[SO_LANE] + lane, s, false);
            float behind = s[0];  // the state behind the tile, of lane l
            if (V > 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float w = __shfl_sync(0xffffffffu, s[v], 32 - COLS + l / V);
                    if (l % V == v) behind = w;
                }
            }
            joiner.hand_on(behind, last_step, true);
        }
    }
    copies_wait_all();
}

// ---- time adjacent in memory ([.., T]): a warp's tile is 384 steps of one row, a run of 12
// adjacent steps per thread (an odd number of 16-byte vectors, so that the threads' runs lie
// in different banks), the runs' maps joined by shuffles.  Tiles move between global and
// shared memory in coalesced vectors, in and out.  Rows need not start on 16 bytes: vectors are
// cut at the row's own 16-byte boundaries (`shift` steps before its first one), so whole
// vectors move as 16 bytes and only ragged ends value by value.
constexpr int kRun = 12, kTile = 32 * kRun, kVectors = kTile / 4;

template <bool BACKWARD>
struct RowTile {
    float in[2][kArrays<BACKWARD>][kTile];
    float out[kTile];
    float before[2];  // backward: the state before the tile's first step in memory
    float pad[2];
};
template <bool BACKWARD>
constexpr size_t rows_smem() {
    return NW * sizeof(RowTile<BACKWARD>) + sizeof(Exchange<1>);
}

template <bool BACKWARD, int PASS>
__global__ void __launch_bounds__(NW * 32, BACKWARD ? 2 : 3) scan_rows_kernel(ScanArgs a) {
    constexpr int NA = kArrays<BACKWARD>;
    extern __shared__ __align__(16) unsigned char raw[];
    const Place at = place(a);
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31, W = a.W;
    const int wt = warp % W, wr = warp / W;
    RowTile<BACKWARD>& tile = reinterpret_cast<RowTile<BACKWARD>*>(raw)[warp];
    Exchange<1>& ex = *reinterpret_cast<Exchange<1>*>(raw + NW * sizeof(RowTile<BACKWARD>));
    const int64_t row = at.block * (NW / W) + wr;
    const bool live = row < a.lanes;
    const float* p[SI_COUNT];
#pragma unroll
    for (int k = 0; k < SI_COUNT; ++k) p[k] = a.in[k].p ? a.in[k].p + (live ? row : 0) * a.in[k].so : nullptr;
    const int64_t dst = (live ? row : 0) * a.T;
    const int shift = static_cast<int>(dst & 3);
    const int64_t vectors = (a.T + shift + 3) / 4;
    const bool want_gate = BACKWARD && PASS != MAPS && a.out[SO_GATE];
    // segments and tiles are counted in vectors of four; scan order r
    const int64_t begin = at.seg * a.seg_len, end = live ? min(vectors, begin + a.seg_len) : begin;
    const int64_t all_end = min((a.T + 6) / 4, begin + a.seg_len);  // the longest row's: all warps loop alike
    const int64_t stride = static_cast<int64_t>(at.size) * W * kVectors;
    const int64_t own = begin + (static_cast<int64_t>(at.rank) * W + wt) * kVectors;
    // the tile at r0: its first vector in memory and how many vectors it has; backward a tile that is
    // cut short keeps its high end
    auto tile_place = [&](int64_t r0, int64_t& v0) {
        const int n = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(kVectors), end - r0)));
        v0 = BACKWARD ? vectors - r0 - kVectors : r0;  // may be negative where n < kVectors
        return n;
    };
    auto issue = [&](int64_t r0, int stage) {
        int64_t v0;
        const int n = tile_place(r0, v0);
        if (n > 0) {
            const int lo = BACKWARD ? kVectors - n : 0;  // the vectors of the tile that exist: [lo, lo + n)
#pragma unroll
            for (int arr = 0; arr < NA; ++arr) {
                const int k = arr == 0 ? SI_GATE : arr == 1 ? SI_X : SI_H;
                if (arr == 1 && !p[SI_X]) continue;
                if (arr == 2 && !want_gate) continue;
#pragma unroll
                for (int q = 0; q < kVectors / 32; ++q) {
                    const int v = l + 32 * q;
                    if (v < lo || v >= lo + n) continue;
                    const int64_t t = 4 * (v0 + v) - shift;
                    const uint32_t to = smem_addr(&tile.in[stage][arr][4 * v]);
                    if ((a.vec >> k & 1) && t >= 0 && t + 3 < a.T) {
                        copy_async<16>(to, p[k] + t);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (t + j >= 0 && t + j < a.T) copy_async<4>(to + 4 * j, p[k] + (t + j) * a.in[k].st);
                    }
                }
            }
            if (want_gate && l == 0) {
                const int64_t t = 4 * (v0 + lo) - shift - 1;  // before the tile's first step in memory
                if (t >= 0) copy_async<4>(smem_addr(&tile.before[stage]), p[SI_H] + t * a.in[SI_H].st);
            }
        }
        copies_commit();
    };
    issue(own, 0);
    issue(own + stride, 1);
    if (at.size > 1) cg::this_cluster().sync();  // every CTA runs before another writes to it
    float c = live ? segment_state<PASS>(a, at.seg, row, p[SI_CARRY]) : 0.0f;
    if (a.T == 0) {
        copies_wait_all();
        if (live && wt == 0 && l == 0 && a.out[SO_LANE]) a.out[SO_LANE][row] = c;
        return;
    }
    Joiner<1> joiner{ex, at, W, wt, wr, warp, 0};
    float gates = 1.0f;
    const float init = want_gate && live && p[SI_INIT] ? __ldg(p[SI_INIT]) : 0.0f;
    const int run = (BACKWARD ? 31 - l : l) * kRun;  // this thread's run within the tile
    int stage = 0;
    for (int64_t base = begin; base < all_end; base += stride, stage ^= 1) {
        const int64_t r0 = own + (base - begin);
        int64_t v0;
        const int n = tile_place(r0, v0);
        const int lo = BACKWARD ? kVectors - n : 0;
        const int64_t t0 = 4 * v0 - shift + run;  // the run's first step in memory
        copies_wait_one();
        __syncwarp();
        float ga[kRun], xv[kRun], hv[BACKWARD ? kRun : 1];
#pragma unroll
        for (int j = 0; j < kRun; j += 4) {
            load_shared<4>(&tile.in[stage][0][run + j], ga + j);
            load_shared<4>(&tile.in[stage][1][run + j], xv + j);
        }
        if constexpr (BACKWARD) {
            if (want_gate) {  // the state before each step
                float h[kRun];
#pragma unroll
                for (int j = 0; j < kRun; j += 4) load_shared<4>(&tile.in[stage][2][run + j], h + j);
                hv[0] = run > 4 * lo ? tile.in[stage][2][run > 0 ? run - 1 : 0] : tile.before[stage];
#pragma unroll
                for (int j = 1; j < kRun; ++j) hv[j] = h[j - 1];
            }
        }
        // the row's ends: steps outside it leave the state as it is
        const bool whole = n == kVectors && t0 >= (BACKWARD ? 1 : 0) && t0 + kRun <= a.T && p[SI_X];
        if (!whole) {
#pragma unroll
            for (int j = 0; j < kRun; ++j) {
                const int v = (run + j) / 4;
                const bool inside = v >= lo && v < lo + n && t0 + j >= 0 && t0 + j < a.T;
                if (!inside) ga[j] = 1.0f;
                if (!inside || !p[SI_X]) xv[j] = 0.0f;
                if (BACKWARD && want_gate && run + j == 4 * lo) hv[BACKWARD ? j : 0] = tile.before[stage];
                if (BACKWARD && t0 + j == 0) hv[BACKWARD ? j : 0] = init;
            }
        }
        __syncwarp();
        issue(r0 + 2 * stride, stage);
        float2 q = tile_map<BACKWARD, kRun>([&](int j) { return ga[BACKWARD ? kRun - 1 - j : j]; },
                                            [&](int j) { return xv[BACKWARD ? kRun - 1 - j : j]; });
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const float2 b = make_float2(__shfl_up_sync(0xffffffffu, q.x, d), __shfl_up_sync(0xffffffffu, q.y, d));
            if (l >= d) q = join(b, q);
        }
        const float2 m = make_float2(__shfl_sync(0xffffffffu, q.x, 31), __shfl_sync(0xffffffffu, q.y, 31));
        float2 b = make_float2(__shfl_up_sync(0xffffffffu, q.x, 1), __shfl_up_sync(0xffffffffu, q.y, 1));
        float s = joiner.first(m, c, base == begin, l == 0);
        const bool last_step = base + stride >= all_end;
        float y = l > 0 ? apply(b, s) : s;
        if constexpr (PASS == MAPS) {
            joiner.gates_of_step(gates);
            s = apply(m, s);
            if (last_step && live && wt == W - 1 && l == 0) a.maps[at.seg * a.lanes + row] = make_float2(gates, s);
        } else {
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
#pragma unroll
                for (int j = 0; j < kRun; j += 4)
                    *reinterpret_cast<float4*>(&tile.out[run + j]) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                __syncwarp();
#pragma unroll
                for (int u = 0; u < kVectors / 32; ++u) {
                    const int k = l + 32 * u;
                    if (k < lo || k >= lo + n) continue;
                    const int64_t t = 4 * (v0 + k) - shift;
                    float f[4];
                    load_shared<4>(&tile.out[4 * k], f);
                    if (t >= 0 && t + 3 < a.T) {
                        store_vec<4>(out + dst + t, f, BACKWARD);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (t + j >= 0 && t + j < a.T) out[dst + t + j] = f[j];
                    }
                }
                __syncwarp();
            };
            if (a.out[SO_MAIN]) write(a.out[SO_MAIN], xv);
            if constexpr (BACKWARD) {
                if (want_gate) write(a.out[SO_GATE], hv);
            }
            s = __shfl_sync(0xffffffffu, y, 31);  // behind the tile's last run
            if (n > 0 && r0 + n == vectors && l == 0 && a.out[SO_LANE]) a.out[SO_LANE][row] = s;
        }
        joiner.hand_on(s, last_step, l == 0);
    }
    copies_wait_all();
}

// The widest vectors of lanes: every operand has adjacent lanes behind n1 whose vectors are
// aligned wherever they start (buffers start on 16 bytes), or is broadcast over them.
int widest(const ScanDesc& d) {
    for (int v = 4; v > 1; v /= 2) {
        bool ok = d.n2 % v == 0;
        for (int k = 0; k < SI_COUNT && ok; ++k) {
            const ScanStrides& s = d.in[k];  // (all 0 where absent)
            if (s.s2 == 0) continue;
            ok = s.s2 == 1 && s.so % v == 0 && s.st % v == 0 && s.s1 % v == 0 && s.off % v == 0;
        }
        if (ok) return v;
    }
    return 1;
}

// How a scan is cut: lanes per thread, warps along time, CTAs of a cluster along time, segments.
struct Cut {
    bool rows;
    int V = 1, W = 1, cluster = 1, segments = 1;
    int64_t seg_len = 0, blocks = 0;
};

Cut cut(const ScanDesc& d) {
    Cut c;
    const int64_t inner = d.n1 * d.n2, lanes = d.outer * inner;
    c.rows = inner == 1;
    if (!c.rows) c.V = widest(d);
    const int64_t len = c.rows ? (d.T + 6) / 4 : d.T;  // rows count time in vectors of four
    const int64_t tile = c.rows ? kVectors : kTileSteps, tiles = (len + tile - 1) / tile;
    while (c.W < NW && c.W < tiles) c.W *= 2;
    const int64_t groups = c.rows ? lanes : (lanes + 31) / 32;
    c.blocks = (groups + NW / c.W - 1) / (NW / c.W);
    // more CTAs along time while the card is not full and every CTA has a step of its own
    while (c.W == NW && c.cluster < 8 && c.blocks * c.cluster < 256 && c.cluster * c.W * tile * 2 <= len) c.cluster *= 2;
    c.seg_len = len > 0 ? len : 1;
    if (c.blocks * c.cluster < 128 && len > static_cast<int64_t>(c.cluster) * c.W * tile) {
        c.cluster = 1;
        const int64_t step = c.W * tile, most = (len + step - 1) / step;
        int64_t want = (296 + c.blocks - 1) / c.blocks;
        if (want > most) want = most;
        c.seg_len = ((len + want - 1) / want + step - 1) / step * step;
        c.segments = static_cast<int>((len + c.seg_len - 1) / c.seg_len);
    }
    return c;
}

template <auto Kernel>
cudaError_t launch_kernel(size_t smem, const Cut& c, const ScanArgs& a, cudaStream_t stream) {
    static std::atomic<uint64_t> ready{0};  // devices on which the kernel's shared memory limit is raised
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (!(ready.load() & bit)) {
        e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
        ready |= bit;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(c.blocks * c.segments * c.cluster));
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

template <bool BACKWARD, int PASS>
cudaError_t launch_pass(const Cut& c, const ScanArgs& a, cudaStream_t stream) {
    if (c.rows) return launch_kernel<scan_rows_kernel<BACKWARD, PASS>>(rows_smem<BACKWARD>(), c, a, stream);
    if (c.V == 4) return launch_kernel<scan_cols_kernel<BACKWARD, PASS, 4>>(cols_smem<BACKWARD>(), c, a, stream);
    if (c.V == 2) return launch_kernel<scan_cols_kernel<BACKWARD, PASS, 2>>(cols_smem<BACKWARD>(), c, a, stream);
    return launch_kernel<scan_cols_kernel<BACKWARD, PASS, 1>>(cols_smem<BACKWARD>(), c, a, stream);
}

template <bool BACKWARD>
cudaError_t launch_cut(const Cut& c, const ScanArgs& a, cudaStream_t stream) {
    if (c.segments == 1) return launch_pass<BACKWARD, ONLY>(c, a, stream);
    const cudaError_t e = launch_pass<BACKWARD, MAPS>(c, a, stream);
    return e != cudaSuccess ? e : launch_pass<BACKWARD, JOINED>(c, a, stream);
}

}  // namespace

int64_t scan_scratch_bytes(const ScanDesc& d) {
    const Cut c = cut(d);
    return c.segments > 1 ? c.segments * d.outer * d.n1 * d.n2 * static_cast<int64_t>(sizeof(float2)) : 0;
}

int scan_launch_count(const ScanDesc& d) {
    return d.outer * d.n1 * d.n2 == 0 ? 0 : cut(d).segments > 1 ? 2 : 1;
}

int launch_scan(const ScanDesc& d, const float* const* in, float* const* out, void* scratch, void* stream) {
    const int64_t lanes = d.outer * d.n1 * d.n2;
    if (lanes == 0) return 0;
    const Cut c = cut(d);
    if (c.blocks * c.segments * c.cluster > 0x7fffffff) return static_cast<int>(cudaErrorInvalidConfiguration);
    ScanArgs a;
    a.vec = 0;
    for (int k = 0; k < SI_COUNT; ++k) {
        const ScanStrides& s = d.in[k];
        a.in[k] = Operand{in[k] ? in[k] + s.off : nullptr, s.so, s.st, s.s1, s.s2};
        // rows: every row starts at the same place within 16 bytes as the result's
        if (c.rows ? s.st == 1 && s.off % 4 == 0 && (s.so - d.T) % 4 == 0 : s.s2 == 1) a.vec |= 1 << k;
    }
    for (int k = 0; k < SO_COUNT; ++k) a.out[k] = out[k];
    a.maps = static_cast<float2*>(scratch);
    a.lanes = lanes;
    a.inner = d.n1 * d.n2;
    a.n2 = d.n2;
    a.T = d.T;
    a.seg_len = c.seg_len;
    a.segments = c.segments;
    a.W = c.W;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return static_cast<int>(d.backward ? launch_cut<true>(c, a, st) : launch_cut<false>(c, a, st));
}

}  // namespace ttb
