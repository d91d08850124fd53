// Log-probabilities of chosen tokens, the clipped policy loss and the preference loss over
// logits, forward and backward, for sm_100a.
//
// Per row of logits x[V] with token k:  m = max x,  s = sum exp(x - m),
//   p = x[k] - m - log s                                    (the token's log-probability)
//   dlogits[j] = c * ([j == k] - exp(x[j] - m)/s),  c = upstream gradient * d value / d p
//
// What bounds them is the logits: 4 bytes a value read, 4 written where the gradient is
// wanted.  A loss and its gradient are one kernel that reads a row once: its values stay in
// registers between the row's maximum and sum and the gradient's write.  A row that no CTA
// can hold is held by a cluster of up to 8, whose parts' (maximum, sum) are joined through
// distributed shared memory, one barrier a row; so are rows that are too few to fill the card.
// The preference loss's slope depends on all rows of its pair, so its gradient is a second
// pass, from the rows' m and s, in reverse order: the rows read last are still in L2.
// Row scalars (p, ratios, losses, c) are formed in double: one thread per row does it, and
// differences of log-probabilities decide on which side of a clip border a ratio lies.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "program.hpp"

namespace cg = cooperative_groups;

namespace ttb {

namespace {

constexpr int kMaxCluster = 8;  // portable cluster size

struct RowOperand {
    const float* p;  // null: absent
    int64_t s0, s1;
    __device__ float at(int64_t i0, int64_t i1) const { return __ldg(p + i0 * s0 + i1 * s1); }
};

struct TokenArgs {
    const float* logits;
    int64_t ls0, ls1;
    const int* tokens;
    int64_t ts0, ts1;
    RowOperand old, adv, ref, g;
    float* y;
    float* dlogits;
    float* stats;   // preference loss: per row {m, 1/s, p - ref}; null otherwise
    float* slopes;  // preference loss: per pair, upstream gradient * d loss / d S(0)
    int* status;
    int64_t rows, n1, V;
    int kind;
    float f0, f1, f2;
};

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN propagates
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Maximum and sum of exp(x - maximum) of part of a row; joins are exact in any order of the
// maxima, and sums are always joined in the same order.  An empty part is (-inf, 0).
struct Part {
    float m, s;
};

// exp(a - b) for the maxima of a part and a whole: 0 for a part of -inf alone, whose sum is 0 too
__device__ __forceinline__ float part_weight(float m, float whole) { return m == -INFINITY ? 0.0f : expf(m - whole); }

// Value and slope (d value / d p) of a row from its token's log-probability.
__device__ void row_value(const TokenArgs& a, int64_t i0, int64_t i1, double p, double& value, double& slope) {
    value = p;
    slope = 1.0;
    if (a.kind != TK_POLICY) return;
    const double adv = a.adv.at(i0, i1), r = exp(p - static_cast<double>(a.old.at(i0, i1)));
    const double lo = 1.0 - static_cast<double>(a.f0), hi = 1.0 + static_cast<double>(a.f1);
    const double plain = r * adv, held = (r < lo ? lo : r > hi ? hi : r) * adv;
    value = plain <= held ? -plain : -held;
    slope = plain <= held ? -plain : 0.0;
    if (plain != plain) value = slope = plain;  // NaN in the row or its numbers
    if (a.ref.p) {
        const double k = static_cast<double>(a.ref.at(i0, i1)) - p, e = exp(k), kl = a.f2;
        value += kl * (e - k - 1.0);
        slope += kl * (1.0 - e);
    }
}

// A row: its token, where its logits and its gradient lie, and how they lie within 16 bytes.
// Vectors are cut at the logits' 16-byte boundaries, `shift` values before the row's first.
struct Row {
    int64_t row, i0, i1;
    const float* x;
    float* dx;
    int token, shift;
    bool dx_vec;  // the gradient lies alike
    __device__ Row(const TokenArgs& a, int64_t r) : row(r), i0(r / a.n1), i1(r % a.n1) {
        if (a.rows <= 0x7fffffff) {
            i0 = static_cast<unsigned>(r) / static_cast<unsigned>(a.n1);
            i1 = static_cast<unsigned>(r) % static_cast<unsigned>(a.n1);
        }
        token = __ldg(a.tokens + i0 * a.ts0 + i1 * a.ts1);
        x = a.logits + i0 * a.ls0 + i1 * a.ls1;
        dx = a.dlogits ? a.dlogits + r * a.V : nullptr;
        shift = static_cast<int>(reinterpret_cast<uintptr_t>(x) / 4 % 4);
        dx_vec = static_cast<int>(reinterpret_cast<uintptr_t>(dx) / 4 % 4) == shift;
    }
};

// `once`: the value is not read again soon (evict it first).
__device__ __forceinline__ void load_vec(const float* x, int64_t j, int64_t V, bool once, float* v) {
    if (j >= 0 && j + 3 < V) {
        const float4* p = reinterpret_cast<const float4*>(x + j);
        const float4 f = once ? __ldcs(p) : __ldg(p);
        v[0] = f.x;
        v[1] = f.y;
        v[2] = f.z;
        v[3] = f.w;
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = j + u >= 0 && j + u < V ? __ldg(x + j + u) : -INFINITY;
    }
}
__device__ __forceinline__ void store_vec(float* x, int64_t j, int64_t V, bool vec, const float* v) {
    if (vec && j >= 0 && j + 3 < V) {
        __stcs(reinterpret_cast<float4*>(x + j), make_float4(v[0], v[1], v[2], v[3]));
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (j + u >= 0 && j + u < V) x[j + u] = v[u];
    }
}

// A row that is not computed: padding is 0, a token outside the vocabulary is NaN.  `first`:
// this thread writes the row's scalars; part / parts and tid / G share out the gradient.
__device__ void fill_row(const TokenArgs& a, const Row& r, bool first, int64_t from, int64_t step) {
    const float v = r.token < 0 ? 0.0f : __int_as_float(0x7fc00000);
    if (first) {
        if (r.token >= 0) *a.status = TT_STATUS_BAD_TOKEN;
        if (a.stats) a.stats[3 * r.row + 2] = v;
        else if (a.y) a.y[r.row] = v;
    }
    if (!r.dx || a.stats) return;
    const int out = static_cast<int>(reinterpret_cast<uintptr_t>(r.dx) / 4 % 4);
    const float f[4] = {v, v, v, v};
    for (int64_t q = from; 4 * q - out < a.V; q += step) store_vec(r.dx, 4 * q - out, a.V, true, f);
}

// The row's outputs besides the gradient, and the gradient's factor c, by one thread.
__device__ __forceinline__ float row_scalars(const TokenArgs& a, const Row& r, float xk, Part all, bool write) {
    if (a.stats) {
        if (write) {
            const double p = static_cast<double>(xk) - static_cast<double>(all.m) - log(static_cast<double>(all.s));
            a.stats[3 * r.row] = all.m;
            a.stats[3 * r.row + 1] = 1.0f / all.s;
            a.stats[3 * r.row + 2] = static_cast<float>(p - static_cast<double>(a.ref.at(r.i0, r.i1)));
        }
        return 0.0f;
    }
    const double p = static_cast<double>(xk) - static_cast<double>(all.m) - log(static_cast<double>(all.s));
    double value, slope;
    row_value(a, r.i0, r.i1, p, value, slope);
    if (write && a.y) a.y[r.row] = static_cast<float>(value);
    return r.dx ? static_cast<float>(slope * static_cast<double>(a.g.at(r.i0, r.i1))) : 0.0f;
}

// Sum / maximum over a CTA's threads (G a multiple of 32), the same in every thread.  sh: G/32
// floats that no other reduction of the kernel uses.
template <int G, bool MAX>
__device__ __forceinline__ float all_threads(float v, float* sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, w) : v + w;
    }
    if (G == 32) return v;
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < G / 32; ++w) v = MAX ? max_nan(v, sh[w]) : v + sh[w];
    return v;
}

// ---- rows held in registers: G threads (a warp, or a CTA of a cluster) hold up to 4*NV values
// each.  G = 32: 8 rows a CTA, a warp each.
template <int G, int NV, bool GRAD>
__global__ void __launch_bounds__(G == 32 ? 256 : G, G == 512 ? 2 : 4) token_held_kernel(TokenArgs a) {
    __shared__ float sh_max[G / 32], sh_sum[G / 32];
    __shared__ Part parts[kMaxCluster];
    __shared__ float sh_c;
    cg::cluster_group cl = cg::this_cluster();
    const int size = G == 32 ? 1 : static_cast<int>(cl.num_blocks()), rank = G == 32 ? 0 : static_cast<int>(cl.block_rank());
    const int tid = G == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t index = G == 32 ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x / size;
    if (G == 32 && index >= a.rows) return;
    const Row r(a, index);
    if (r.token < 0 || r.token >= a.V) {  // (the whole cluster leaves)
        fill_row(a, r, tid == 0 && rank == 0, rank * G + tid, size * G);
        return;
    }
    if (size > 1) cl.barrier_arrive();  // every CTA runs before another writes to it
    const float xk = __ldg(r.x + r.token);
    // this CTA's vectors: NV runs of G adjacent ones
    const int64_t j0 = 4 * (static_cast<int64_t>(rank) * NV * G + tid) - r.shift;
    float v[NV][4];
#pragma unroll
    for (int q = 0; q < NV; ++q) load_vec(r.x, j0 + 4 * q * G, a.V, GRAD, v[q]);
    Part all;
    all.m = v[0][0];
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int u = 0; u < 4; ++u) all.m = max_nan(all.m, v[q][u]);
    all.m = all_threads<G, true>(all.m, sh_max);
    const float own = all.m, from = own == -INFINITY ? 0.0f : own;
    all.s = 0.0f;
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int u = 0; u < 4; ++u) all.s += v[q][u] = expf(v[q][u] - from);
    all.s = all_threads<G, false>(all.s, sh_sum);
    if (size > 1) {
        cl.barrier_wait();
        if (tid < size) *cl.map_shared_rank(&parts[rank], tid) = all;
        cl.sync();
        float whole = -INFINITY, sum = 0.0f;
        for (int q = 0; q < size; ++q) whole = max_nan(whole, parts[q].m);
        for (int q = 0; q < size; ++q) sum += parts[q].s * part_weight(parts[q].m, whole);
        all.m = whole;
        all.s = sum;
    }
    if (!GRAD) {
        if (tid == 0 && rank == 0) row_scalars(a, r, xk, all, true);
        return;
    }
    float c;
    if (a.kind == TK_LOGPROB) {  // the gradient does not need p
        c = a.g.at(r.i0, r.i1);
        if (tid == 0 && rank == 0) row_scalars(a, r, xk, all, true);
    } else if (G == 32) {
        c = __shfl_sync(0xffffffffu, tid == 0 ? row_scalars(a, r, xk, all, true) : 0.0f, 0);
    } else {
        if (tid == 0) sh_c = row_scalars(a, r, xk, all, rank == 0);
        __syncthreads();
        c = sh_c;
    }
    // (all.m = NaN or -inf: the sum is NaN or 0 and makes the row NaN)
    const float scale = -c * (size > 1 ? part_weight(own, all.m) : 1.0f) / all.s;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int64_t j = j0 + 4 * q * G;
#pragma unroll
        for (int u = 0; u < 4; ++u) v[q][u] = v[q][u] * scale + (j + u == r.token ? c : 0.0f);
        store_vec(r.dx, j, a.V, r.dx_vec, v[q]);
    }
}

// ---- rows longer than a cluster can hold: every CTA reads its share twice, joining maximum and
// sum as it goes the first time (the second time most of it comes from L2).
constexpr int kStream = 512, kStreamVec = 4;

template <bool GRAD>
__global__ void __launch_bounds__(kStream, 2) token_stream_kernel(TokenArgs a) {
    __shared__ float sh_max[kStream / 32], sh_sum[kStream / 32];
    __shared__ Part parts[kMaxCluster];
    __shared__ float sh_c;
    cg::cluster_group cl = cg::this_cluster();
    const int size = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank()), tid = threadIdx.x;
    const Row r(a, blockIdx.x / size);
    if (r.token < 0 || r.token >= a.V) {
        fill_row(a, r, tid == 0 && rank == 0, rank * kStream + tid, size * kStream);
        return;
    }
    cl.barrier_arrive();
    const float xk = __ldg(r.x + r.token);
    const int64_t vectors = (a.V + r.shift + 3) / 4, share = (vectors + size - 1) / size;
    const int64_t begin = min(vectors, rank * share), end = min(vectors, begin + share);
    Part t{-INFINITY, 0.0f};
    for (int64_t q0 = begin + tid; q0 < end; q0 += kStreamVec * kStream) {
        float v[kStreamVec][4];
#pragma unroll
        for (int q = 0; q < kStreamVec; ++q) load_vec(r.x, 4 * (q0 + q * kStream) - r.shift, q0 + q * kStream < end ? a.V : 0, false, v[q]);
        float m = t.m;
#pragma unroll
        for (int q = 0; q < kStreamVec; ++q)
#pragma unroll
            for (int u = 0; u < 4; ++u) m = max_nan(m, v[q][u]);
        const float from = m == -INFINITY ? 0.0f : m;
        t.s *= part_weight(t.m, from);
#pragma unroll
        for (int q = 0; q < kStreamVec; ++q)
#pragma unroll
            for (int u = 0; u < 4; ++u) t.s += expf(v[q][u] - from);
        t.m = m;
    }
    Part all;
    all.m = all_threads<kStream, true>(t.m, sh_max);
    all.s = all_threads<kStream, false>(t.s * part_weight(t.m, all.m), sh_sum);
    cl.barrier_wait();
    if (tid < size) *cl.map_shared_rank(&parts[rank], tid) = all;
    cl.sync();
    float whole = -INFINITY, sum = 0.0f;
    for (int q = 0; q < size; ++q) whole = max_nan(whole, parts[q].m);
    for (int q = 0; q < size; ++q) sum += parts[q].s * part_weight(parts[q].m, whole);
    if (tid == 0) sh_c = row_scalars(a, r, xk, Part{whole, sum}, rank == 0);
    if (!GRAD) return;
    __syncthreads();
    const float c = sh_c, scale = -c / sum;
    for (int64_t q = end - 1 - tid; q >= begin; q -= kStream) {
        float v[4];
        const int64_t j = 4 * q - r.shift;
        load_vec(r.x, j, a.V, true, v);
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = expf(v[u] - whole) * scale + (j + u == r.token ? c : 0.0f);
        store_vec(r.dx, j, a.V, r.dx_vec, v);
    }
}

// ---- preference loss: one CTA per pair: z = beta*(S(0) - S(1)), the loss and its slope.
constexpr int kPair = 256;
__global__ void __launch_bounds__(kPair) preference_pair_kernel(TokenArgs a) {
    __shared__ double sh[kPair / 32];
    const int64_t n = blockIdx.x, T = a.n1 / 2;
    double v = 0.0;
    for (int64_t t = threadIdx.x; t < T; t += kPair) {
        const float* st = a.stats + 3 * (n * a.n1 + t);
        v += static_cast<double>(st[2]) - static_cast<double>(st[3 * T + 2]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < kPair / 32; ++w) v += sh[w];
    const double beta = a.f0, eps = a.f1, z = beta * v;
    const double e = exp(-fabs(z)), soft = log1p(e);  // soft = -log sigmoid(|z|)
    // (eps = 0 drops its term: an impossible rejected answer has z = inf and loss 0)
    if (a.y) a.y[n] = static_cast<float>(soft + (z < 0.0 ? -z * (1.0 - eps) : z == z && eps == 0.0 ? 0.0 : z * eps));
    if (a.slopes) {
        const double up = 1.0 / (1.0 + e), down = e / (1.0 + e);  // sigmoid(|z|), sigmoid(-|z|)
        const double pos = z < 0.0 ? down : up, neg = z < 0.0 ? up : down;
        a.slopes[n] = static_cast<float>(static_cast<double>(a.g.at(n, 0)) * beta * (eps * pos - (1.0 - eps) * neg));
    }
}

// The preference loss's gradient from the rows' stats: a CTA takes kGradVec*kGrad vectors of a row.
constexpr int kGrad = 256, kGradVec = 4;
__global__ void __launch_bounds__(kGrad) preference_grad_kernel(TokenArgs a, int per_row) {
    const Row r(a, a.rows - 1 - blockIdx.x / per_row);
    const int64_t q0 = static_cast<int64_t>(blockIdx.x % per_row) * kGradVec * kGrad + threadIdx.x;
    if (r.token < 0 || r.token >= a.V) {
        const float f = r.token < 0 ? 0.0f : __int_as_float(0x7fc00000), v[4] = {f, f, f, f};
#pragma unroll
        for (int q = 0; q < kGradVec; ++q) store_vec(r.dx, 4 * (q0 + q * kGrad) - r.shift, a.V, r.dx_vec, v);
        return;
    }
    float v[kGradVec][4];
#pragma unroll
    for (int q = 0; q < kGradVec; ++q) load_vec(r.x, 4 * (q0 + q * kGrad) - r.shift, a.V, true, v[q]);
    const float m = __ldg(a.stats + 3 * r.row), slope = __ldg(a.slopes + r.i0), c = r.i1 < a.n1 / 2 ? slope : -slope;
    const float scale = -c * __ldg(a.stats + 3 * r.row + 1);
#pragma unroll
    for (int q = 0; q < kGradVec; ++q) {
        const int64_t j = 4 * (q0 + q * kGrad) - r.shift;
#pragma unroll
        for (int u = 0; u < 4; ++u) v[q][u] = expf(v[q][u] - m) * scale + (j + u == r.token ? c : 0.0f);
        store_vec(r.dx, j, a.V, r.dx_vec, v[q]);
    }
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

template <class Kernel>
cudaError_t launch_rows(Kernel kernel, int64_t blocks, int threads, int cluster, const TokenArgs& a, cudaStream_t stream) {
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int G, bool GRAD>
cudaError_t launch_held(int nv, int64_t blocks, int cluster, const TokenArgs& a, cudaStream_t stream) {
    const int threads = G == 32 ? 256 : G;
    if (nv <= 1) return launch_rows(token_held_kernel<G, 1, GRAD>, blocks, threads, cluster, a, stream);
    if (nv <= 2) return launch_rows(token_held_kernel<G, 2, GRAD>, blocks, threads, cluster, a, stream);
    if (nv <= 4) return launch_rows(token_held_kernel<G, 4, GRAD>, blocks, threads, cluster, a, stream);
    return launch_rows(token_held_kernel<G, 8, GRAD>, blocks, threads, cluster, a, stream);
}

template <bool GRAD>
cudaError_t launch_row_kernel(const TokenArgs& a, cudaStream_t stream) {
    const int64_t vectors = (a.V + 6) / 4;  // at most, wherever a row starts
    if (vectors <= 32 * 8)
        return launch_held<32, GRAD>(static_cast<int>((vectors + 31) / 32), (a.rows + 7) / 8, 1, a, stream);
    if (vectors > static_cast<int64_t>(kMaxCluster) * 512 * 8)
        return launch_rows(token_stream_kernel<GRAD>, a.rows * kMaxCluster, kStream, kMaxCluster, a, stream);
    const int G = vectors > kMaxCluster * 256 * 8 ? 512 : 256;
    // as many CTAs as hold the row, and more while rows do not fill the card
    int cluster = static_cast<int>((vectors + G * 8 - 1) / (G * 8));
    while (cluster < kMaxCluster && a.rows * cluster < 296 && cluster * G < vectors) ++cluster;
    const int nv = static_cast<int>((vectors + cluster * G - 1) / (cluster * G));
    return G == 512 ? launch_held<512, GRAD>(nv, a.rows * cluster, cluster, a, stream)
                    : launch_held<256, GRAD>(nv, a.rows * cluster, cluster, a, stream);
}

}  // namespace

int64_t token_scratch_bytes(const TokenDesc& d) {
    return d.kind == TK_PREFERENCE ? align256(d.n0 * d.n1 * 12) + align256(d.n0 * 4) : 0;
}

int token_launch_count(const TokenDesc& d) {
    const int rows = d.n0 * d.n1 > 0 ? 1 : 0;
    return d.kind == TK_PREFERENCE ? rows * (d.grad ? 2 : 1) + (d.n0 > 0 ? 1 : 0) : rows;
}

int launch_token(const TokenDesc& d, const void* const* in, float* y, float* dlogits, void* scratch, int* status,
                 void* stream) {
    auto f = [&](int k) { return in[k] ? static_cast<const float*>(in[k]) + d.off[k] : nullptr; };
    TokenArgs a;
    a.logits = f(TI_LOGITS);
    a.ls0 = d.s0[TI_LOGITS];
    a.ls1 = d.s1[TI_LOGITS];
    a.tokens = static_cast<const int*>(in[TI_TOKENS]) + d.off[TI_TOKENS];
    a.ts0 = d.s0[TI_TOKENS];
    a.ts1 = d.s1[TI_TOKENS];
    auto operand = [&](int k) { return RowOperand{f(k), d.s0[k], d.s1[k]}; };
    a.old = operand(TI_OLD);
    a.adv = operand(TI_ADVANTAGE);
    a.ref = operand(TI_REF);
    a.g = operand(TI_GRAD);
    a.y = y;
    a.dlogits = dlogits;
    const bool pref = d.kind == TK_PREFERENCE;
    a.stats = pref ? static_cast<float*>(scratch) : nullptr;
    a.slopes = pref && dlogits ? reinterpret_cast<float*>(static_cast<char*>(scratch) + align256(d.n0 * d.n1 * 12)) : nullptr;
    a.status = status;
    a.rows = d.n0 * d.n1;
    a.n1 = d.n1;
    a.V = d.V;
    a.kind = d.kind;
    a.f0 = d.f[0];
    a.f1 = d.f[1];
    a.f2 = d.f[2];
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.rows > 0) {
        const cudaError_t e = dlogits && !pref ? launch_row_kernel<true>(a, st) : launch_row_kernel<false>(a, st);
        if (e != cudaSuccess) return static_cast<int>(e);
    }
    if (pref && d.n0 > 0) {
        if (d.n0 > 0x7fffffff) return static_cast<int>(cudaErrorInvalidConfiguration);
        preference_pair_kernel<<<static_cast<unsigned>(d.n0), kPair, 0, st>>>(a);
        if (dlogits && a.rows > 0) {
            const int64_t per_row = ((a.V + 6) / 4 + kGradVec * kGrad - 1) / (kGradVec * kGrad);
            if (a.rows * per_row > 0x7fffffff) return static_cast<int>(cudaErrorInvalidConfiguration);
            preference_grad_kernel<<<static_cast<unsigned>(a.rows * per_row), kGrad, 0, st>>>(a, static_cast<int>(per_row));
        }
    }
    return static_cast<int>(cudaGetLastError());
}

}  // namespace ttb
