// The global norm of many gradients and clipping by it (include/sr_hip.h: sr_tensors_*, sr_op_grad_norm, sr_op_clip_grads):
//
//   norm = scale * sqrt(sum over all tensors and elements of g^2),   g' = g * scale * (max_norm / norm if norm > max_norm else 1)
//
// Bound by HBM: the norm reads every gradient once, clipping reads it again (from the 256 MB last-level cache where it is still
// there) and writes it once.  The squares are added in 64 bits: an fp32 square overflows above 1.8e19 and vanishes below 1e-23, a
// 64-bit one does neither, and beside the loads the conversions and products cost nothing.  A tensor is cut into chunks, a workgroup
// takes one chunk and leaves one partial sum; chunks grow with the whole list so that there are about 2048 of them at most, which
// every workgroup of the clipping launch adds up by itself in one fixed order (2048 doubles from L2) -- no atomics, no third
// launch, the same bits on every run.  The chunk table travels in the kernel arguments: nothing is uploaded, and a captured
// graph holds its own copy.
#include "grad_clip.h"
#include "op_host.h"
#include "row_math.h"

#include <algorithm>
#include <new>

using namespace sr;
using namespace srh;

namespace {

// 224 x (8 + 4 + 4 + 1) and 152 x (16 + 4 + 4 + 1) bytes of the 4 KiB of kernel arguments
constexpr int NORM_MAX = 224, SCALE_MAX = 152;

template <int MAX>
struct Pieces {
    uint32_t n[MAX], first[MAX];    // elements of a piece, its first chunk in this launch
    uint8_t type[MAX];
    int count;
    uint32_t chunk;

    // the piece that owns chunk b of this launch
    __device__ __forceinline__ int find(uint32_t b) const {
        int lo = 0, hi = count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= b) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    }
};

struct NormTable {
    const void* src[NORM_MAX];
    Pieces<NORM_MAX> p;
};
struct ScaleTable {
    const void* src[SCALE_MAX];
    void* dst[SCALE_MAX];
    Pieces<SCALE_MAX> p;
};

__device__ __forceinline__ double block_sum(double s, double* lds4) {
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) lds4[threadIdx.x >> 6] = s;
    __syncthreads();
    return (lds4[0] + lds4[1]) + (lds4[2] + lds4[3]);
}

// sum of squares of n elements by 256 threads: 16-byte loads, 4 in flight
template <typename T>
__device__ __forceinline__ double sum_squares(const T* p, uint32_t n) {
    constexpr int V = 16 / sizeof(T);
    double s[2] = {0.0, 0.0};
    const uint32_t nv = n / V;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < nv; i += 256) {
        float v[V];
        load_vec<T, V>(p + (size_t)i * V, v);
#pragma unroll
        for (int k = 0; k < V; ++k) s[k & 1] = fma((double)v[k], (double)v[k], s[k & 1]);
    }
    const uint32_t t = nv * V + threadIdx.x;
    if (t < n) s[0] = fma((double)(float)p[t], (double)(float)p[t], s[0]);   // fewer than V elements are left
    return s[0] + s[1];
}

__global__ void __launch_bounds__(256) grad_partials_kernel(const NormTable t, double* __restrict__ parts) {
    __shared__ double lds4[4];
    const int e = t.p.find(blockIdx.x);
    const uint32_t at = (blockIdx.x - t.p.first[e]) * t.p.chunk, n = min(t.p.chunk, t.p.n[e] - at);
    double s;
    if (t.p.type[e] == SR_T_F32) s = sum_squares((const float*)t.src[e] + at, n);
    else if (t.p.type[e] == SR_T_BF16) s = sum_squares((const bf16_t*)t.src[e] + at, n);
    else s = sum_squares((const f16_t*)t.src[e] + at, n);
    s = block_sum(s, lds4);
    if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

// workgroup 0: the norm of everything; the others: one tensor a wave
constexpr int EACH_MAX = 900;
struct EachTable {
    uint32_t first[EACH_MAX + 1];   // partial sums of the tensors of this launch
    int count;
};
__global__ void __launch_bounds__(256) grad_norm_kernel(const EachTable t, const double* __restrict__ parts, int nparts, float scale,
                                                        float* __restrict__ norm, float* __restrict__ each) {
    __shared__ double lds4[4];
    if (blockIdx.x == 0) {
        if (!norm) return;
        double s = 0.0;
        for (int i = threadIdx.x; i < nparts; i += 256) s += parts[i];
        s = block_sum(s, lds4);
        if (threadIdx.x == 0) *norm = (float)(sqrt(s) * (double)scale);
        return;
    }
    const int i = ((int)blockIdx.x - 1) * 4 + (threadIdx.x >> 6);
    if (i >= t.count) return;
    double s = 0.0;
    for (uint32_t k = t.first[i] + (threadIdx.x & 63); k < t.first[i + 1]; k += 64) s += parts[k];
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) each[i] = (float)(sqrt(s) * (double)scale);
}

template <typename T>
__device__ __forceinline__ void scale_run(const T* src, T* dst, uint32_t n, float f) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t nv = n / V;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < nv; i += 256) {
        float v[V];
        load_vec<T, V>(src + (size_t)i * V, v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] *= f;
        store_vec<T, V>(dst + (size_t)i * V, v);
    }
    const uint32_t t = nv * V + threadIdx.x;
    if (t < n) dst[t] = (T)((float)src[t] * f);
}

__global__ void __launch_bounds__(256) grad_scale_kernel(const ScaleTable t, const ClipArgs c) {
    __shared__ double lds4[4];
    const float f = clip_factor(c, lds4) * c.s0;
    const int e = t.p.find(blockIdx.x);
    if (f == 1.f && t.src[e] == t.dst[e]) return;   // in place and nothing to do
    const uint32_t at = (blockIdx.x - t.p.first[e]) * t.p.chunk, n = min(t.p.chunk, t.p.n[e] - at);
    if (t.p.type[e] == SR_T_F32) scale_run((const float*)t.src[e] + at, (float*)t.dst[e] + at, n, f);
    else if (t.p.type[e] == SR_T_BF16) scale_run((const bf16_t*)t.src[e] + at, (bf16_t*)t.dst[e] + at, n, f);
    else scale_run((const f16_t*)t.src[e] + at, (f16_t*)t.dst[e] + at, n, f);
}

// an empty list has no chunks, but still a norm
__global__ void grad_zero_norm_kernel(float* norm) { *norm = 0.f; }

}  // namespace

namespace sr {

uint32_t grad_chunk(int64_t total) {
    const int64_t unit = 8192;
    return (uint32_t)(std::max<int64_t>(1, (total + GRAD_PARTS * unit - 1) / (GRAD_PARTS * unit)) * unit);
}

hipError_t launch_grad_partials(const GradPiece* pieces, int n, uint32_t chunk, double* parts, hipStream_t s) {
    NormTable t;
    for (int i = 0; i < n;) {
        uint32_t blocks = 0;
        int k = 0;
        for (; i < n && k < NORM_MAX; ++i) {
            if (!pieces[i].n) continue;
            t.src[k] = pieces[i].src, t.p.n[k] = pieces[i].n, t.p.first[k] = blocks, t.p.type[k] = (uint8_t)pieces[i].type;
            blocks += (uint32_t)grad_chunks(pieces[i].n, chunk);
            ++k;
        }
        if (!k) break;
        t.p.count = k, t.p.chunk = chunk;
        grad_partials_kernel<<<blocks, 256, 0, s>>>(t, parts);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        parts += blocks;
    }
    return hipSuccess;
}

}  // namespace sr

// ------------------------------------------------------------------------------------------------- C ABI
struct sr_tensors {
    int device = 0;
    std::vector<sr_tensor_desc> list;
    std::vector<GradPiece> pieces;
    std::vector<uint32_t> first;             // first partial sum of every tensor, and their number
    std::vector<std::pair<const char*, const char*>> sorted;   // byte ranges by address
    uint32_t chunk = 0;
    bool overlap = false;                    // two tensors share memory
};

#define GC_TRY(call)          \
    do {                      \
        const int rc_ = call; \
        if (rc_) return rc_;  \
    } while (0)

namespace {

size_t workspace_of(const sr_tensors* t) { return std::max<size_t>(t->first.back(), 1) * sizeof(double); }

int check_call(const sr_tensors* t, float scale, const float* d_norm, const float* d_norms, const void* ws, size_t ws_bytes, const char* who) {
    if (!t) return fail(nullptr, SR_ERR_ARG, "%s: the tensor list is NULL", who);
    if (!(scale > 0.f && scale < 3e38f)) return fail(nullptr, SR_ERR_ARG, "%s: scale must be positive and finite", who);
    if (!ws || (uintptr_t)ws % 8) return fail(nullptr, SR_ERR_ARG, "%s: the workspace is NULL or not aligned to 8 bytes", who);
    if (ws_bytes < workspace_of(t))
        return fail(nullptr, SR_ERR_ARG, "%s: the workspace holds %zu bytes, this list needs %zu", who, ws_bytes, workspace_of(t));
    if (!d_norm || (uintptr_t)d_norm % 4 || (uintptr_t)d_norms % 4) return fail(nullptr, SR_ERR_ARG, "%s: d_norm is NULL or not aligned", who);
    const Region w = {(const char*)ws, 1, 0, (int64_t)workspace_of(t)}, a = {(const char*)d_norm, 1, 0, 4}, b = {(const char*)d_norms, 1, 0, (int64_t)t->list.size() * 4};
    if (!disjoint(w, a) || !disjoint(w, b) || !disjoint(a, b)) return fail(nullptr, SR_ERR_ARG, "%s: the norms and the workspace overlap", who);
    return SR_OK;
}

// does any tensor of `t` touch [p, p + bytes)?
bool touches(const sr_tensors* t, const void* p, size_t bytes) {
    const char *b = (const char*)p, *e = b + bytes;
    if (!p || !bytes) return false;
    for (const auto& r : t->sorted)
        if (r.first < e && b < r.second) return true;
    return false;
}

int launched(hipError_t e, const char* what) {
    return e == hipSuccess ? SR_OK : fail(nullptr, SR_ERR_HIP, "launch %s: %s", what, hipGetErrorString(e));
}

}  // namespace

extern "C" {

int sr_tensors_create(sr_tensors** out, int device, int n, const sr_tensor_desc* tensors) {
    const char* who = "sr_tensors_create";
    if (!out) return fail(nullptr, SR_ERR_ARG, "%s: out is NULL", who);
    *out = nullptr;
    if (n < 0 || (n && !tensors)) return fail(nullptr, SR_ERR_ARG, "%s: bad tensor list", who);
    if (device < 0) return fail(nullptr, SR_ERR_ARG, "%s: device %d out of range", who, device);
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
        const sr_tensor_desc& d = tensors[i];
        const int b = type_bytes(d.type);
        if (!b) return fail(nullptr, SR_ERR_ARG, "%s: tensor %d: unknown type", who, i);
        if (d.count < 0 || d.count > ((int64_t)1 << 40)) return fail(nullptr, SR_ERR_ARG, "%s: tensor %d: count must be 0 .. 2^40", who, i);
        if (d.count && (!d.data || (uintptr_t)d.data % b)) return fail(nullptr, SR_ERR_ARG, "%s: tensor %d is NULL or not aligned to its elements", who, i);
        total += d.count;
        if (total > ((int64_t)1 << 40)) return fail(nullptr, SR_ERR_ARG, "%s: more than 2^40 elements", who);
    }
    sr_tensors* t = nullptr;
    try {
        t = new sr_tensors;
        t->device = device;
        t->list.assign(tensors, tensors + n);
        t->chunk = grad_chunk(total);
        uint32_t parts = 0;
        t->first.push_back(0);
        for (const sr_tensor_desc& d : t->list) {
            const int b = type_bytes(d.type);
            for (int64_t at = 0; at < d.count; at += GRAD_PIECE) {
                const uint32_t m = (uint32_t)std::min<int64_t>(d.count - at, GRAD_PIECE);
                t->pieces.push_back({(const char*)d.data + at * b, m, (uint32_t)d.type});
                parts += (uint32_t)grad_chunks(m, t->chunk);
            }
            t->first.push_back(parts);
            if (d.count) t->sorted.emplace_back((const char*)d.data, (const char*)d.data + d.count * b);
        }
        std::sort(t->sorted.begin(), t->sorted.end());
        for (size_t i = 1; i < t->sorted.size(); ++i) t->overlap |= t->sorted[i].first < t->sorted[i - 1].second;
    } catch (const std::bad_alloc&) {
        delete t;
        return fail(nullptr, SR_ERR_ARG, "%s: out of host memory", who);
    }
    *out = t;
    return SR_OK;
}

int sr_tensors_destroy(sr_tensors* t) {
    delete t;
    return SR_OK;
}

int sr_tensors_workspace(const sr_tensors* t, size_t* bytes) {
    if (!t || !bytes) return fail(nullptr, SR_ERR_ARG, "NULL argument");
    *bytes = workspace_of(t);
    return SR_OK;
}

int sr_op_grad_norm(const sr_tensors* t, float scale, float* d_norm, float* d_norms, void* workspace, size_t workspace_bytes,
                    void* hip_stream) {
    const char* who = "sr_op_grad_norm";
    GC_TRY(check_call(t, scale, d_norm, d_norms, workspace, workspace_bytes, who));
    const size_t n = t->list.size();
    if (touches(t, workspace, workspace_of(t)) || touches(t, d_norm, 4) || touches(t, d_norms, n * 4))
        return fail(nullptr, SR_ERR_ARG, "%s: an output or the workspace overlaps a tensor", who);
    OnDevice on;
    GC_TRY(on.enter(t->device));
    hipStream_t st = (hipStream_t)hip_stream;
    double* parts = (double*)workspace;
    GC_TRY(launched(launch_grad_partials(t->pieces.data(), (int)t->pieces.size(), t->chunk, parts, st), who));
    EachTable e;
    size_t at = 0;
    do {
        e.count = d_norms ? (int)std::min<size_t>(n - at, EACH_MAX) : 0;
        for (int i = 0; i <= e.count; ++i) e.first[i] = t->first[at + i];
        grad_norm_kernel<<<1 + (e.count + 3) / 4, 256, 0, st>>>(e, parts, (int)t->first.back(), scale, at ? nullptr : d_norm, d_norms + at);
        GC_TRY(launched(hipGetLastError(), who));
        at += e.count;
    } while (d_norms && at < n);
    return SR_OK;
}

int sr_op_clip_grads(const sr_tensors* t, const sr_tensors* out, float max_norm, float scale, float* d_norm, void* workspace,
                     size_t workspace_bytes, void* hip_stream) {
    const char* who = "sr_op_clip_grads";
    GC_TRY(check_call(t, scale, d_norm, nullptr, workspace, workspace_bytes, who));
    if (!(max_norm > 0.f)) return fail(nullptr, SR_ERR_ARG, "%s: max_norm must be positive", who);
    if (!out) out = t;
    if (out->overlap) return fail(nullptr, SR_ERR_ARG, "%s: two of the tensors to write share memory", who);
    if (out != t) {
        if (out->device != t->device || out->list.size() != t->list.size())
            return fail(nullptr, SR_ERR_ARG, "%s: the two lists differ in device or length", who);
        for (size_t i = 0; i < t->list.size(); ++i)
            if (out->list[i].count != t->list[i].count || out->list[i].type != t->list[i].type)
                return fail(nullptr, SR_ERR_ARG, "%s: tensor %zu differs in count or type between the lists", who, i);
        // what is written is the gradient itself (then no other gradient may share its memory) or touches no gradient; both
        // lists go by address
        bool in_place = false;
        size_t a = 0;
        for (const auto& w : out->sorted) {
            while (a < t->sorted.size() && t->sorted[a].second <= w.first) ++a;
            for (size_t k = a; k < t->sorted.size() && t->sorted[k].first < w.second; ++k) {
                if (t->sorted[k].second <= w.first) continue;
                if (t->sorted[k] != w || t->overlap) return fail(nullptr, SR_ERR_ARG, "%s: a tensor to write overlaps another gradient", who);
                in_place = true;
            }
        }
        for (size_t i = 0; in_place && i < t->list.size(); ++i) {
            const sr_tensor_desc& w = out->list[i];
            if (!w.count || w.data == t->list[i].data) continue;
            const std::pair<const char*, const char*> r((const char*)w.data, (const char*)w.data + w.count * type_bytes(w.type));
            if (std::binary_search(t->sorted.begin(), t->sorted.end(), r))
                return fail(nullptr, SR_ERR_ARG, "%s: a tensor to write is another gradient", who);
        }
    }
    if (touches(t, workspace, workspace_of(t)) || touches(t, d_norm, 4) || (out != t && (touches(out, workspace, workspace_of(t)) || touches(out, d_norm, 4))))
        return fail(nullptr, SR_ERR_ARG, "%s: the norm or the workspace overlaps a tensor", who);
    OnDevice on;
    GC_TRY(on.enter(t->device));
    hipStream_t st = (hipStream_t)hip_stream;
    double* parts = (double*)workspace;
    const int n = (int)t->pieces.size();
    if (!n) {
        grad_zero_norm_kernel<<<1, 1, 0, st>>>(d_norm);
        return launched(hipGetLastError(), who);
    }
    GC_TRY(launched(launch_grad_partials(t->pieces.data(), n, t->chunk, parts, st), who));
    ClipArgs c = {parts, (int)t->first.back(), 0, scale, 0.f, max_norm, d_norm};
    ScaleTable s;
    for (int i = 0; i < n;) {
        uint32_t blocks = 0;
        int k = 0;
        for (; i < n && k < SCALE_MAX; ++i, ++k) {
            const GradPiece& p = t->pieces[i];
            s.src[k] = p.src, s.dst[k] = const_cast<void*>(out->pieces[i].src), s.p.n[k] = p.n, s.p.first[k] = blocks, s.p.type[k] = (uint8_t)p.type;
            blocks += (uint32_t)grad_chunks(p.n, t->chunk);
        }
        s.p.count = k, s.p.chunk = t->chunk;
        grad_scale_kernel<<<blocks, 256, 0, st>>>(s, c);
        GC_TRY(launched(hipGetLastError(), who));
        c.norm = nullptr;
    }
    return SR_OK;
}

}  // extern "C"
