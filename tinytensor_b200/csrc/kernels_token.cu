// Log-probabilities of chosen tokens, the clipped policy loss and the preference loss over
// logits, forward and backward, for sm_100a.
//
// Per row of logits x[V] with token k:  m = max x,  s = sum exp(x - m),
//   p = x[k] - m - log s                                    (the token's log-probability)
//   dlogits[j] = c * ([j == k] - exp(x[j] - m)/s),  c = upstream gradient * d value / d p
// Row scalars (p, ratios, losses, c) are formed in double: one thread per row does it, and
// differences of log-probabilities decide on which side of a clip border a ratio lies.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "program.hpp"

namespace ttb {

namespace {

constexpr int kThreads = 256;

struct RowOperand {
    const float* p;  // null: absent
    int64_t s0, s1;
    __device__ float at(int64_t i0, int64_t i1) const { return p[i0 * s0 + i1 * s1]; }
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
    int64_t n0, n1, V;
    int kind;
    float f0, f1, f2;
};

struct MaxOp {
    static __device__ float of(float a, float b) {  // NaN propagates
        return a > b || a != a ? a : b;
    }
};
struct SumOp {
    static __device__ float of(float a, float b) { return a + b; }
};

template <class Op>
__device__ float block_all(float v, float* sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = Op::of(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) v = Op::of(v, sh[w]);
    return v;
}

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

// One CTA per row: maximum, sum, the row's value, the row's gradient.
__global__ void __launch_bounds__(kThreads) token_row_kernel(TokenArgs a) {
    __shared__ float sh[kThreads / 32];
    __shared__ float bc;
    const int64_t row = blockIdx.x, i0 = row / a.n1, i1 = row % a.n1;
    const int token = a.tokens[i0 * a.ts0 + i1 * a.ts1];
    const bool bad = token >= a.V;
    if (bad && threadIdx.x == 0) *a.status = TT_STATUS_BAD_TOKEN;
    float* dx = a.dlogits ? a.dlogits + row * a.V : nullptr;
    const float nan = __int_as_float(0x7fc00000);
    if (token < 0 || bad) {
        if (threadIdx.x == 0) {
            if (a.stats) a.stats[3 * row + 2] = bad ? nan : 0.0f;
            else if (a.y) a.y[row] = bad ? nan : 0.0f;
        }
        if (dx && !a.stats)
            for (int64_t j = threadIdx.x; j < a.V; j += kThreads) dx[j] = bad ? nan : 0.0f;
        return;
    }
    const float* x = a.logits + i0 * a.ls0 + i1 * a.ls1;
    float m = -INFINITY;
    for (int64_t j = threadIdx.x; j < a.V; j += kThreads) m = MaxOp::of(m, x[j]);
    m = block_all<MaxOp>(m, sh);
    float s = 0.0f;
    for (int64_t j = threadIdx.x; j < a.V; j += kThreads) s += expf(x[j] - m);
    s = block_all<SumOp>(s, sh);
    if (threadIdx.x == 0) {
        const double p = static_cast<double>(x[token]) - static_cast<double>(m) - log(static_cast<double>(s));
        if (a.stats) {
            a.stats[3 * row] = m;
            a.stats[3 * row + 1] = 1.0f / s;
            a.stats[3 * row + 2] = static_cast<float>(p - static_cast<double>(a.ref.at(i0, i1)));
        } else {
            double value, slope;
            row_value(a, i0, i1, p, value, slope);
            if (a.y) a.y[row] = static_cast<float>(value);
            if (dx) bc = static_cast<float>(slope * static_cast<double>(a.g.at(i0, i1)));
        }
    }
    if (!dx || a.stats) return;
    __syncthreads();
    const float c = bc, scale = -c / s;
    for (int64_t j = threadIdx.x; j < a.V; j += kThreads) dx[j] = expf(x[j] - m) * scale + (j == token ? c : 0.0f);
}

// One CTA per pair: z = beta*(S(0) - S(1)), the loss and its slope.
__global__ void __launch_bounds__(kThreads) preference_pair_kernel(TokenArgs a) {
    __shared__ double sh[kThreads];
    const int64_t n = blockIdx.x, T = a.n1 / 2;
    double v = 0.0;
    for (int64_t t = threadIdx.x; t < T; t += kThreads) {
        const float* st = a.stats + 3 * (n * a.n1 + t);
        v += static_cast<double>(st[2]) - static_cast<double>(st[3 * T + 2]);
    }
    sh[threadIdx.x] = v;
    __syncthreads();
    for (int w = kThreads / 2; w > 0; w >>= 1) {
        if (threadIdx.x < w) sh[threadIdx.x] += sh[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x != 0) return;
    const double beta = a.f0, eps = a.f1, z = beta * sh[0];
    const double soft = log1p(exp(-fabs(z)));  // -log sigmoid(|z|)
    // (eps = 0 drops its term: an impossible rejected answer has z = inf and loss 0)
    if (a.y) a.y[n] = static_cast<float>(soft + (z < 0.0 ? -z * (1.0 - eps) : z == z && eps == 0.0 ? 0.0 : z * eps));
    if (a.slopes) {
        const double e = exp(-fabs(z)), up = 1.0 / (1.0 + e), down = e / (1.0 + e);  // sigmoid(|z|), sigmoid(-|z|)
        const double pos = z < 0.0 ? down : up, neg = z < 0.0 ? up : down;
        a.slopes[n] = static_cast<float>(static_cast<double>(a.g.at(n, 0)) * beta * (eps * pos - (1.0 - eps) * neg));
    }
}

// One CTA per row of the preference loss's gradient.
__global__ void __launch_bounds__(kThreads) preference_grad_kernel(TokenArgs a) {
    const int64_t row = blockIdx.x, i0 = row / a.n1, i1 = row % a.n1;
    const int token = a.tokens[i0 * a.ts0 + i1 * a.ts1];
    float* dx = a.dlogits + row * a.V;
    if (token < 0 || token >= a.V) {
        const float v = token < 0 ? 0.0f : __int_as_float(0x7fc00000);
        for (int64_t j = threadIdx.x; j < a.V; j += kThreads) dx[j] = v;
        return;
    }
    const float* x = a.logits + i0 * a.ls0 + i1 * a.ls1;
    const float m = a.stats[3 * row], c = i1 < a.n1 / 2 ? a.slopes[i0] : -a.slopes[i0];
    const float scale = -c * a.stats[3 * row + 1];
    for (int64_t j = threadIdx.x; j < a.V; j += kThreads) dx[j] = expf(x[j] - m) * scale + (j == token ? c : 0.0f);
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

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
    a.stats = d.kind == TK_PREFERENCE ? static_cast<float*>(scratch) : nullptr;
    a.slopes = d.kind == TK_PREFERENCE && dlogits
                   ? reinterpret_cast<float*>(static_cast<char*>(scratch) + align256(d.n0 * d.n1 * 12)) : nullptr;
    a.status = status;
    a.n0 = d.n0;
    a.n1 = d.n1;
    a.V = d.V;
    a.kind = d.kind;
    a.f0 = d.f[0];
    a.f1 = d.f[1];
    a.f2 = d.f[2];
    const int64_t rows = d.n0 * d.n1;
    if (rows > 0x7fffffff) return static_cast<int>(cudaErrorInvalidConfiguration);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows > 0) token_row_kernel<<<static_cast<unsigned>(rows), kThreads, 0, st>>>(a);
    if (d.kind == TK_PREFERENCE && d.n0 > 0) {
        preference_pair_kernel<<<static_cast<unsigned>(d.n0), kThreads, 0, st>>>(a);
        if (dlogits && rows > 0) preference_grad_kernel<<<static_cast<unsigned>(rows), kThreads, 0, st>>>(a);
    }
    return static_cast<int>(cudaGetLastError());
}

}  // namespace ttb
