// The norm of a training step's gradients as partial sums, and the factor that clipping derives from them (grad_clip.hip); the
// optimizer step of a clipped update reads the partial sums itself (train_kernels.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sr {

constexpr int GRAD_PARTS = 4096;    // partial sums of a list of n pieces: at most GRAD_PARTS + n
constexpr uint32_t GRAD_PIECE = 1u << 29;   // elements of a piece: longer tensors are several pieces

// a run of `n` <= GRAD_PIECE dense elements of enum sr_type `type`
struct GradPiece {
    const void* src;
    uint32_t n, type;
};

// elements of one partial sum, so that `total` elements make at most GRAD_PARTS full ones
uint32_t grad_chunk(int64_t total);
inline int64_t grad_chunks(uint32_t n, uint32_t chunk) { return ((int64_t)n + chunk - 1) / chunk; }
// parts[i] = sum of squares of chunk i; piece after piece, the chunks of a piece in order.  At most 160 pieces.
hipError_t launch_grad_partials(const GradPiece* pieces, int n, uint32_t chunk, double* parts, hipStream_t s);

// the same of one vector, however long; *nparts: how many partial sums there are (at most FLAT_PARTS)
constexpr int FLAT_PARTS = GRAD_PARTS + 64;
hipError_t launch_flat_partials(const float* g, int64_t n, double* parts, int* nparts, hipStream_t s);

// What a kernel needs to know the norm of scaled gradients: two runs of partial sums (the second may be empty) and their scales
struct ClipArgs {
    const double* parts;
    int n0, n1;                     // parts[0 .. n0) carry scale s0, parts[n0 .. n0 + n1) carry s1
    float s0, s1, max_norm;
    float* norm;                    // written by workgroup 0
};

// What a gradient is multiplied by: f, then 2^e.  e is 0 but where the product is below fp32's normal range (gradients near its upper
// end and a small bound, for instance: 1e6 elements of 1e38 and a bound of 1), which one fp32 factor would hold with a few bits or not
// at all; f is then in [0.5, 1).
struct GradScale {
    float f;
    int e;
    __device__ __forceinline__ float operator()(float g) const { return ldexpf(g * f, e); }
};

// All 256 threads of a workgroup: `scale` times the factor that brings the gradients' norm down to max_norm, 1 where it is not above it
// (or NaN).  Every workgroup adds the partial sums in the same order, so all have the same bits.
__device__ __forceinline__ GradScale clip_factor(const ClipArgs& c, float scale, double* lds4) {
    double s = 0.0;
    const double q0 = (double)c.s0 * c.s0, q1 = (double)c.s1 * c.s1;
#pragma unroll 8
    for (int i = threadIdx.x; i < c.n0 + c.n1; i += 256) s += c.parts[i] * (i < c.n0 ? q0 : q1);
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) lds4[threadIdx.x >> 6] = s;
    __syncthreads();
    const double norm = sqrt((lds4[0] + lds4[1]) + (lds4[2] + lds4[3]));
    if (blockIdx.x == 0 && threadIdx.x == 0 && c.norm) *c.norm = (float)norm;
    const double factor = norm > (double)c.max_norm ? (double)c.max_norm / norm : 1.0;
    constexpr float least = 1.17549435e-38f;
    const float f = (float)factor * scale;
    if ((float)factor >= least && fabsf(f) >= least) return {f, 0};
    const double p = factor * (double)scale;      // the factor alone may be out of range where the product is not
    if (p == 0.0 || fabs(p) >= (double)least) return {(float)p, 0};
    int e;
    const double m = frexp(p, &e);
    return {(float)m, e};
}

}  // namespace sr
