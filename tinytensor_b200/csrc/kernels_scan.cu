// Gated linear recurrences for sm_100a.
//
//   forward    h[t] = gate[t]*h[t-1] + x[t],  h[-1] = init (0 when absent)
//   backward   u[t] = g[t] + c[t+1],  c[t] = gate[t]*u[t],  c[T] = upstream gradient of the
//              last state;  dx[t] = u[t],  dgate[t] = u[t]*h[t-1],  dinit = c[0]
#include <cuda_runtime.h>

#include <cstdint>

#include "program.hpp"

namespace ttb {

namespace {

struct Operand {
    const float* p;  // null: absent
    int64_t so, st, s1, s2;
};

struct ScanArgs {
    Operand in[SI_COUNT];
    float* out[SO_COUNT];
    int64_t outer, T, n1, n2;
};

// One thread per lane walks the time axis.
template <bool BACKWARD>
__global__ void __launch_bounds__(256) scan_lane_kernel(ScanArgs a) {
    const int64_t inner = a.n1 * a.n2, lane = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (lane >= a.outer * inner) return;
    const int64_t o = lane / inner, i = lane % inner, i1 = i / a.n2, i2 = i % a.n2;
    const float* p[SI_COUNT];
    for (int k = 0; k < SI_COUNT; ++k)
        p[k] = a.in[k].p ? a.in[k].p + o * a.in[k].so + i1 * a.in[k].s1 + i2 * a.in[k].s2 : nullptr;
    const int64_t at = o * a.T * inner + i;  // this lane's first result
    float c = p[SI_CARRY] ? *p[SI_CARRY] : 0.0f;
    if (!BACKWARD) {
        for (int64_t t = 0; t < a.T; ++t) {
            c = fmaf(p[SI_GATE][t * a.in[SI_GATE].st], c, p[SI_X][t * a.in[SI_X].st]);
            if (a.out[SO_MAIN]) a.out[SO_MAIN][at + t * inner] = c;
        }
    } else {
        for (int64_t t = a.T; t-- > 0;) {
            const float u = (p[SI_X] ? p[SI_X][t * a.in[SI_X].st] : 0.0f) + c;
            if (a.out[SO_MAIN]) a.out[SO_MAIN][at + t * inner] = u;
            if (a.out[SO_GATE]) {
                const float before = t > 0 ? p[SI_H][(t - 1) * a.in[SI_H].st] : p[SI_INIT] ? *p[SI_INIT] : 0.0f;
                a.out[SO_GATE][at + t * inner] = u * before;
            }
            c = p[SI_GATE][t * a.in[SI_GATE].st] * u;
        }
    }
    if (a.out[SO_LANE]) a.out[SO_LANE][lane] = c;
}

}  // namespace

int scan_launch_count(const ScanDesc& d) { return d.outer * d.n1 * d.n2 > 0 ? 1 : 0; }

int launch_scan(const ScanDesc& d, const float* const* in, float* const* out, void* stream) {
    const int64_t lanes = d.outer * d.n1 * d.n2;
    if (lanes == 0) return 0;
    ScanArgs a;
    for (int k = 0; k < SI_COUNT; ++k) {
        const ScanStrides& s = d.in[k];
        a.in[k] = Operand{in[k] ? in[k] + s.off : nullptr, s.so, s.st, s.s1, s.s2};
    }
    for (int k = 0; k < SO_COUNT; ++k) a.out[k] = out[k];
    a.outer = d.outer;
    a.T = d.T;
    a.n1 = d.n1;
    a.n2 = d.n2;
    const int64_t blocks = (lanes + 255) / 256;
    if (blocks > 0x7fffffff) return static_cast<int>(cudaErrorInvalidConfiguration);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d.backward) scan_lane_kernel<true><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a);
    else scan_lane_kernel<false><<<static_cast<unsigned>(blocks), 256, 0, st>>>(a);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace ttb
