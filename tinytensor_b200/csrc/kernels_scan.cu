// Gated linear recurrences for sm_100a.
//
//   forward    h[t] = gate[t]*h[t-1] + x[t],  h[-1] = init (0 when absent)
//   backward   u[t] = g[t] + c[t+1],  c[t] = gate[t]*u[t],  c[T] = upstream gradient of the
//              last state;  dx[t] = u[t],  dgate[t] = u[t]*h[t-1],  dinit = c[0]
//
// Both are a chain of maps c -> A*c + H, and maps compose: a run of steps is one map, found
// without knowing the state it starts from.  Every warp holds a tile of the time axis in
// registers, finds its tile's map, learns its first state by joining the maps of the tiles
// before it, and only then writes its states: one pass over the data, each value read once
// and written once, which is what bounds these kernels (forward 12 bytes a value, backward
// 20 with all gradients).  Tiles are joined in time order at three levels, so results do not
// depend on how CTAs are scheduled:
//   warps of a CTA        through shared memory, one block barrier a step;
//   CTAs of a cluster     through distributed shared memory, one cluster barrier a step,
//                         where there are too few lanes to fill the card;
//   segments of the axis  through device scratch, by a first launch that finds the segments'
//                         maps, where clusters are not enough (the data is read twice).
// Time runs in scan order r: t = r forward, t = T-1-r backward.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "program.hpp"

namespace cg = cooperative_groups;

namespace ttb {

namespace {

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
    int vec;          // line kernel: bit k = operand k can be read as float4
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

// The maps of a CTA's warps and of a cluster's CTAs, double-buffered: a buffer is written
// again two steps later, after a barrier that every reader passes behind its reads.
template <int NW, int LW>
struct Exchange {
    float2 warp[2][NW][LW];
    float2 cta[2][8][LW];  // [buffer][rank in the cluster]; clusters are cut with W = NW, one lane group a CTA
};

// Gives this warp the state its tile starts from and advances `c` (the state before the
// step's first tile, the same in all warps) past the step.  m: the map of the warp's tile.
template <int NW, int LW>
__device__ __forceinline__ float tile_state(Exchange<NW, LW>& ex, int buf, float2 m, float& c, int W, int warp, int l,
                                            int cluster_size, int rank) {
    const int wt = warp % W, wr = warp / W;
    ex.warp[buf][warp][l] = m;
    __syncthreads();
    float first = c;
    if (cluster_size > 1) {
        cg::cluster_group cl = cg::this_cluster();
        if (wt == 0) {
            float2 all = ex.warp[buf][warp][l];
            for (int w = 1; w < W; ++w) all = join(all, ex.warp[buf][wr * W + w][l]);
            for (int q = 0; q < cluster_size; ++q) cl.map_shared_rank(&ex, q)->cta[buf][rank][l] = all;
        }
        cl.sync();
        float s = c;
        for (int q = 0; q < cluster_size; ++q) {
            if (q == rank) first = s;
            s = apply(ex.cta[buf][q][l], s);
        }
        c = s;
        for (int w = 0; w < wt; ++w) first = apply(ex.warp[buf][wr * W + w][l], first);
    } else {
        float s = c;
        for (int w = 0; w < W; ++w) {
            if (w == wt) first = s;
            s = apply(ex.warp[buf][wr * W + w][l], s);
        }
        c = s;
    }
    return first;
}

// The state before segment `seg` and what it starts from otherwise.
template <int PASS>
__device__ __forceinline__ float segment_state(const ScanArgs& a, int seg, int64_t lane, const float* carry) {
    float c = 0.0f;
    if (PASS != MAPS && carry) c = __ldg(carry);
    if constexpr (PASS == JOINED)
        for (int s = 0; s < seg; ++s) c = apply(a.maps[s * a.lanes + lane], c);
    return c;
}

struct Place {
    int64_t block;  // of lanes
    int seg, rank, size;
};
__device__ __forceinline__ Place place(const ScanArgs& a) {
    Place p;
    cg::cluster_group cl = cg::this_cluster();
    p.size = static_cast<int>(cl.num_blocks());
    p.rank = static_cast<int>(cl.block_rank());
    const int64_t unit = blockIdx.x / p.size;
    p.seg = static_cast<int>(unit % a.segments);
    p.block = unit / a.segments;
    return p;
}

// ---- lanes side by side in memory ([.., T, lanes]): a warp takes 32 lanes and TS steps, a lane
// per thread, every step of it one coalesced 128-byte row per operand.
template <bool BACKWARD, int PASS, int TS, int NW>
__global__ void __launch_bounds__(NW * 32, 2) scan_cols_kernel(ScanArgs a) {
    __shared__ Exchange<NW, 32> ex;
    const Place at = place(a);
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31, W = a.W;
    const int wt = warp % W, wr = warp / W;
    const int64_t lane = (at.block * (NW / W) + wr) * 32 + l;
    const bool live = lane < a.lanes;
    const int64_t o = live ? lane / a.inner : 0, i = live ? lane % a.inner : 0, i1 = i / a.n2, i2 = i % a.n2;
    const float* p[SI_COUNT];
#pragma unroll
    for (int k = 0; k < SI_COUNT; ++k)
        p[k] = a.in[k].p ? a.in[k].p + o * a.in[k].so + i1 * a.in[k].s1 + i2 * a.in[k].s2 : nullptr;
    const int64_t dst = o * a.T * a.inner + i;
    float c = live ? segment_state<PASS>(a, at.seg, lane, p[SI_CARRY]) : 0.0f;
    float gates = 1.0f;  // MAPS: the segment's product of gates
    const int64_t begin = at.seg * a.seg_len, end = min(a.T, begin + a.seg_len);
    const bool want_gate = BACKWARD && PASS != MAPS && a.out[SO_GATE];
    int buf = 0;
    for (int64_t base = begin; base < end; base += static_cast<int64_t>(at.size) * W * TS, buf ^= 1) {
        const int64_t r0 = base + (static_cast<int64_t>(at.rank) * W + wt) * TS;
        const int n = live ? static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(TS), end - r0))) : 0;
        const int64_t t0 = BACKWARD ? a.T - 1 - r0 : r0, dt = BACKWARD ? -1 : 1;
        float ga[TS], xv[TS], hv[BACKWARD ? TS : 1];
        {
            const float* q = p[SI_GATE] + t0 * a.in[SI_GATE].st;
            const int64_t step = dt * a.in[SI_GATE].st;
#pragma unroll
            for (int j = 0; j < TS; ++j, q += step) ga[j] = j < n ? __ldg(q) : 1.0f;
        }
        {
            const float* q = p[SI_X] + t0 * a.in[SI_X].st;
            const int64_t step = dt * a.in[SI_X].st;
            const int nx = p[SI_X] ? n : 0;
#pragma unroll
            for (int j = 0; j < TS; ++j, q += step) xv[j] = j < nx ? __ldcs(q) : 0.0f;
        }
        if (BACKWARD) {
            const float* q = p[SI_H] + (t0 - 1) * a.in[SI_H].st;
            const int64_t step = dt * a.in[SI_H].st;
            const int nh = want_gate ? static_cast<int>(min(static_cast<int64_t>(n), t0)) : 0;  // t = 0 has init before it
#pragma unroll
            for (int j = 0; j < TS; ++j, q += step) hv[j] = j < nh ? __ldcs(q) : 0.0f;
            if (want_gate && nh < n && p[SI_INIT]) {
                const float first = __ldg(p[SI_INIT]);
#pragma unroll
                for (int j = 0; j < TS; ++j)
                    if (j == nh) hv[j] = first;
            }
        }
        float2 m = make_float2(ga[0], BACKWARD ? ga[0] * xv[0] : xv[0]);
#pragma unroll
        for (int j = 1; j < TS; ++j) {
            m.x = ga[j] == 0.0f ? 0.0f : m.x * ga[j];
            m.y = BACKWARD ? ga[j] * (xv[j] + m.y) : fmaf(ga[j], m.y, xv[j]);
        }
        float s = tile_state<NW, 32>(ex, buf, m, c, W, warp, l, at.size, at.rank);
        if constexpr (PASS == MAPS) {
            for (int w = 0; w < W; ++w) gates = join_gates(gates, ex.warp[buf][wr * W + w][l].x);
            continue;
        }
        int64_t y = dst + t0 * a.inner;
        const int64_t step = dt * a.inner;
        const int nm = a.out[SO_MAIN] ? n : 0, ng = want_gate ? n : 0;
#pragma unroll
        for (int j = 0; j < TS; ++j, y += step) {  // (past the end: gate 1, x 0, the state stays)
            if (BACKWARD) {
                const float u = xv[j] + s;
                if (j < nm) __stcs(a.out[SO_MAIN] + y, u);
                if (j < ng) __stcs(a.out[SO_GATE] + y, u * hv[j]);
                s = ga[j] * u;
            } else {
                s = fmaf(ga[j], s, xv[j]);
                if (j < nm) a.out[SO_MAIN][y] = s;
            }
        }
        // the thread of the last step has the last state as it was stored
        if (n > 0 && r0 + n == a.T && a.out[SO_LANE]) a.out[SO_LANE][lane] = s;
    }
    if (!live || wt != 0 || at.rank != 0) return;
    if (PASS == MAPS) a.maps[at.seg * a.lanes + lane] = make_float2(gates, c);
    else if (a.T == 0 && a.out[SO_LANE]) a.out[SO_LANE][lane] = c;
}

// ---- time adjacent in memory ([.., T]): a warp takes one row and K*128 steps, four adjacent
// steps per thread and chunk of 128; the threads' maps are joined by shuffles.  Rows need
// not start on 16 bytes: vectors are cut at the row's own 16-byte boundaries (`shift` steps
// before its first one), so whole vectors move as float4 and only ragged ends as scalars.
__device__ __forceinline__ void load4(const Operand& q, const float* p, bool vec, int64_t t, int64_t T, float none, float* v) {
    if (vec && t >= 0 && t + 3 < T) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(p + t));
        v[0] = f.x;
        v[1] = f.y;
        v[2] = f.z;
        v[3] = f.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = t + j >= 0 && t + j < T ? __ldg(p + (t + j) * q.st) : none;
    }
}

__device__ __forceinline__ void store4(float* p, int64_t t, int64_t T, const float* v) {
    if (t >= 0 && t + 3 < T) {
        *reinterpret_cast<float4*>(p + t) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (t + j >= 0 && t + j < T) p[t + j] = v[j];
    }
}

template <bool BACKWARD, int PASS, int K, int NW>
__global__ void __launch_bounds__(NW * 32, 2) scan_rows_kernel(ScanArgs a) {
    __shared__ Exchange<NW, 1> ex;
    const Place at = place(a);
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31, W = a.W;
    const int wt = warp % W, wr = warp / W;
    const int64_t row = at.block * (NW / W) + wr;
    const bool live = row < a.lanes;
    const float* p[SI_COUNT];
#pragma unroll
    for (int k = 0; k < SI_COUNT; ++k) p[k] = a.in[k].p ? a.in[k].p + (live ? row : 0) * a.in[k].so : nullptr;
    const int64_t dst = (live ? row : 0) * a.T;
    const int64_t shift = dst & 3, vectors = (a.T + shift + 3) / 4;
    float c = live ? segment_state<PASS>(a, at.seg, row, p[SI_CARRY]) : 0.0f;
    float gates = 1.0f;
    // segments and steps are counted in vectors of four
    const int64_t begin = at.seg * a.seg_len, end = live ? min(vectors, begin + a.seg_len) : begin;
    const int64_t steps = (min((a.T + 6) / 4, begin + a.seg_len) - begin);  // the longest row's: all warps loop alike
    const bool want_gate = BACKWARD && PASS != MAPS && a.out[SO_GATE];
    int buf = 0;
    for (int64_t base = 0; base < steps; base += static_cast<int64_t>(at.size) * W * K * 32, buf ^= 1) {
        const int64_t v0 = begin + base + (static_cast<int64_t>(at.rank) * W + wt) * K * 32 + l;
        float ga[K][4], xv[K][4];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t v = v0 + k * 32;
            const int64_t t = 4 * (BACKWARD ? vectors - 1 - v : v) - shift;
            const int64_t T = v < end ? a.T : 0;  // 0: nothing of this vector is read
            load4(a.in[SI_GATE], p[SI_GATE], a.vec >> SI_GATE & 1, t, T, 1.0f, ga[k]);
            if (p[SI_X]) load4(a.in[SI_X], p[SI_X], a.vec >> SI_X & 1, t, T, 0.0f, xv[k]);
            else xv[k][0] = xv[k][1] = xv[k][2] = xv[k][3] = 0.0f;
        }
        // per chunk: this thread's map, the map of the threads before it, the chunk's map
        float2 before[K], m = make_float2(1.0f, 0.0f);
        float2 chunk[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float2 q;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float g = ga[k][BACKWARD ? 3 - j : j], x = xv[k][BACKWARD ? 3 - j : j];
                if (j == 0) {
                    q = make_float2(g, BACKWARD ? g * x : x);
                } else {
                    q.x = g == 0.0f ? 0.0f : q.x * g;
                    q.y = BACKWARD ? g * (x + q.y) : fmaf(g, q.y, x);
                }
            }
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const float2 b = make_float2(__shfl_up_sync(0xffffffffu, q.x, d), __shfl_up_sync(0xffffffffu, q.y, d));
                if (l >= d) q = join(b, q);
            }
            chunk[k] = make_float2(__shfl_sync(0xffffffffu, q.x, 31), __shfl_sync(0xffffffffu, q.y, 31));
            const float2 b = make_float2(__shfl_up_sync(0xffffffffu, q.x, 1), __shfl_up_sync(0xffffffffu, q.y, 1));
            before[k] = l > 0 ? b : make_float2(1.0f, 0.0f);
            m = k == 0 ? chunk[0] : join(m, chunk[k]);
        }
        float s = tile_state<NW, 1>(ex, buf, m, c, W, warp, 0, at.size, at.rank);
        if constexpr (PASS == MAPS) {
            for (int w = 0; w < W; ++w) gates = join_gates(gates, ex.warp[buf][wr * W + w][0].x);
            continue;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t v = v0 + k * 32;
            const int64_t t = 4 * (BACKWARD ? vectors - 1 - v : v) - shift;
            const int64_t T = v < end ? a.T : 0;
            float y = apply(before[k], s);
            s = apply(chunk[k], s);
            float main[4], dg[4];
            if (BACKWARD) {
                float hv[4];
                if (want_gate) {
                    // h[t-1 .. t+2]: the vector at t, moved by one, and its predecessor
                    load4(a.in[SI_H], p[SI_H], a.vec >> SI_H & 1, t, T, 0.0f, hv);
                    hv[3] = hv[2];
                    hv[2] = hv[1];
                    hv[1] = hv[0];
                    hv[0] = t > 0 && t - 1 < T ? __ldg(p[SI_H] + (t - 1) * a.in[SI_H].st) : 0.0f;
                    const float first = t <= 0 && t > -4 && T > 0 && p[SI_INIT] ? __ldg(p[SI_INIT]) : 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (t + j == 0) hv[j] = first;
                }
#pragma unroll
                for (int j = 3; j >= 0; --j) {
                    main[j] = xv[k][j] + y;
                    if (want_gate) dg[j] = main[j] * hv[j];
                    y = ga[k][j] * main[j];
                }
                if (a.out[SO_MAIN]) store4(a.out[SO_MAIN] + dst, t, T, main);
                if (want_gate) store4(a.out[SO_GATE] + dst, t, T, dg);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) main[j] = y = fmaf(ga[k][j], y, xv[k][j]);
                if (a.out[SO_MAIN]) store4(a.out[SO_MAIN] + dst, t, T, main);
            }
            if (v == vectors - 1 && v < end && a.out[SO_LANE]) a.out[SO_LANE][row] = y;  // the last step's thread
        }
    }
    if (!live || wt != 0 || at.rank != 0 || l != 0) return;
    if (PASS == MAPS) a.maps[at.seg * a.lanes + row] = make_float2(gates, c);
    else if (a.T == 0 && a.out[SO_LANE]) a.out[SO_LANE][row] = c;
}

constexpr int kWarps = 16, kSteps = 16, kStepsBack = 8, kChunks = 4, kChunksBack = 2;

// How a scan is cut: warps along time, CTAs of a cluster along time, segments.
struct Cut {
    bool rows;
    int W = 1, cluster = 1, segments = 1;
    int64_t seg_len = 0, blocks = 0;
};

Cut cut(const ScanDesc& d) {
    Cut c;
    const int64_t inner = d.n1 * d.n2, lanes = d.outer * inner;
    c.rows = inner == 1;
    // time in units of what one warp holds
    const int64_t len = c.rows ? (d.T + 6) / 4 : d.T;
    const int64_t tile = c.rows ? 32 * (d.backward ? kChunksBack : kChunks) : d.backward ? kStepsBack : kSteps;
    const int64_t tiles = (len + tile - 1) / tile;
    while (c.W < kWarps && c.W < tiles) c.W *= 2;
    const int64_t groups = c.rows ? lanes : (lanes + 31) / 32;
    c.blocks = (groups + kWarps / c.W - 1) / (kWarps / c.W);
    // two CTAs fit an SM: more of them along time while the card is not full and every CTA
    // still has a step of its own
    while (c.W == kWarps && c.cluster < 8 && c.blocks * c.cluster < 192 && c.cluster * c.W * tile * 2 <= len) c.cluster *= 2;
    c.seg_len = len > 0 ? len : 1;
    if (c.blocks * c.cluster < 96 && len > static_cast<int64_t>(c.cluster) * c.W * tile) {
        c.cluster = 1;
        const int64_t step = c.W * tile, most = (len + step - 1) / step;
        int64_t want = (296 + c.blocks - 1) / c.blocks;
        if (want > most) want = most;
        c.seg_len = ((len + want - 1) / want + step - 1) / step * step;
        c.segments = static_cast<int>((len + c.seg_len - 1) / c.seg_len);
    }
    return c;
}

template <bool BACKWARD, int PASS>
cudaError_t launch_pass(const Cut& c, const ScanArgs& a, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(c.blocks * c.segments * c.cluster));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(c.cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (c.rows) return cudaLaunchKernelEx(&cfg, scan_rows_kernel<BACKWARD, PASS, BACKWARD ? kChunksBack : kChunks, kWarps>, a);
    return cudaLaunchKernelEx(&cfg, scan_cols_kernel<BACKWARD, PASS, BACKWARD ? kStepsBack : kSteps, kWarps>, a);
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
        // float4 where every row starts at the same place within 16 bytes as the result's
        if (a.in[k].p && s.st == 1 && reinterpret_cast<uintptr_t>(a.in[k].p) % 16 == 0 && (s.so - d.T) % 4 == 0)
            a.vec |= 1 << k;
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
