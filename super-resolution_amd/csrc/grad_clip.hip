// The global norm of many gradients and clipping by it (include/sr_hip.h: sr_tensors_*, sr_op_grad_norm, sr_op_clip_grads):
//
//   norm = scale * sqrt(sum over all tensors and elements of g^2),   g' = g * scale * (max_norm / norm if norm > max_norm else 1)
//
// Bound by HBM: the norm reads every gradient once, clipping reads it again (from the 256 MB last-level cache where it is still
// there) and writes it once.  The squares are added in 64 bits: an fp32 square overflows above 1.8e19 and vanishes below 1e-23, a
// 64-bit one does neither, and beside the loads the conversions and products cost nothing (250 M bf16 elements: 86 us, 5.8 TB/s).
// A tensor is cut into chunks, a workgroup takes one chunk and leaves one partial sum; chunks grow with the whole list so that there
// are about 4096 of them at most (and one a tensor), added up in one fixed order: no atomics, the same bits on every run.  Every
// workgroup of the clipping launch does that by itself where they are few, which saves a launch.
#include "grad_clip.h"
#include "op_host.h"
#include "row_math.h"

#include <algorithm>
#include <mutex>
#include <new>

using namespace sr;
using namespace srh;

namespace {

// Where a workgroup finds its chunk.  A list of up to TABLE pieces travels in the kernel arguments (24 bytes a piece of their
// 4 KiB): nothing is uploaded, and a captured graph holds its own copy.  Longer ones have a record for every chunk in device memory,
// so that a pass is one launch whatever the number of tensors: in memory of the list where sr_tensors_upload has left them, or in
// the workspace, where a launch for every TABLE pieces (4.7 us each, mostly the way of the arguments) writes them first.  Clipping
// 60 M elements in 700 tensors took 188 us with a launch for every 224 or 152 pieces.
constexpr int TABLE = 160;
// From 128 MB on, half of the last-level cache, clipped gradients are stored past the caches: their next reader would find the first
// of them gone anyway, and the following pass over the gradients does not wait for them to be written back (60 M elements of three
// types: 106 -> 84 us, 100 M bf16: 128 -> 106; 250 M bf16 at odd addresses: 315 -> 322; 5 M fp32 would gain 1 us and lose it to the
// next reader).
constexpr int64_t PAST_CACHES = 128 << 20;
// From this many partial sums on, a launch of one workgroup joins them before the clipping one (2 us): each of that one's workgroups
// would read them all, which grows with the square (us without / with, to other tensors: 24 M fp32 in 2929 sums 46.6 / 48.4, 33 M in
// 4028 sums 64.7 / 63.6, 33 M bf16 39.2 / 36.4, 10,000 tensors of 1000 fp32 64 / 31, 60,000 of 100 1541 / 118).
constexpr uint32_t JOIN_FROM = 3600;

struct Piece {
    const void* src;
    void* dst;
    uint32_t n, first;              // elements, with the type in the two highest bits; the piece's first chunk
};
struct Table {
    Piece e[TABLE];
    int count;
    uint32_t chunk;
};
static_assert(sizeof(Table) + sizeof(ClipArgs) + 64 <= 4096, "kernel arguments");

struct Record {
    const char* p;
    uint32_t n, type;
};
struct Records {
    const Record *src, *dst;
};

struct Chunk {
    const char* src;
    char* dst;
    uint32_t n, type;
};
__device__ __forceinline__ Chunk chunk_of(const Piece& e, uint32_t b, uint32_t chunk) {
    const uint32_t at = (b - e.first) * chunk, n = e.n & 0x3fffffffu, type = e.n >> 30;
    const size_t bytes = (size_t)at * (type == SR_T_F32 ? 4 : 2);
    return {(const char*)e.src + bytes, (char*)e.dst + bytes, min(chunk, n - at), type};
}
__device__ __forceinline__ Chunk chunk_of(const Table& t, uint32_t b) {
    // the last piece that does not start behind chunk b: every lane of the wave compares a few
    int before = 0;
#pragma unroll
    for (int i = 0; i < (TABLE + 63) / 64; ++i) {
        const int k = i * 64 + (threadIdx.x & 63);
        before += __popcll(__ballot(k < t.count && t.e[k < TABLE ? k : 0].first <= b));
    }
    return chunk_of(t.e[__builtin_amdgcn_readfirstlane(before) - 1], b, t.chunk);
}
__device__ __forceinline__ Chunk chunk_of(const Records& t, uint32_t b) {
    const Record s = t.src[b];
    return {s.p, (char*)t.dst[b].p, s.n, s.type};
}

__global__ void __launch_bounds__(64) grad_records_kernel(const Table t, Record* __restrict__ src, Record* __restrict__ dst) {
    const Piece e = t.e[blockIdx.x];
    const uint32_t chunks = ((e.n & 0x3fffffffu) + t.chunk - 1) / t.chunk;
    for (uint32_t i = threadIdx.x; i < chunks; i += 64) {
        const Chunk c = chunk_of(e, e.first + i, t.chunk);
        src[e.first + i] = {c.src, c.n, c.type};
        dst[e.first + i] = {c.dst, c.n, c.type};
    }
}

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

template <typename TABLE_T>
__global__ void __launch_bounds__(256) grad_partials_kernel(const TABLE_T t, double* __restrict__ parts) {
    __shared__ double lds4[4];
    const Chunk c = chunk_of(t, blockIdx.x);
    double s;
    if (c.type == SR_T_F32) s = sum_squares((const float*)c.src, c.n);
    else if (c.type == SR_T_BF16) s = sum_squares((const bf16_t*)c.src, c.n);
    else s = sum_squares((const f16_t*)c.src, c.n);
    s = block_sum(s, lds4);
    if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

// workgroup 0: the norm of everything; the others: a tensor each
constexpr int EACH_MAX = 900;
struct EachTable {
    uint32_t first[EACH_MAX + 1];   // partial sums of the tensors of this launch
};
struct EachRecords {
    const uint32_t* first;
};
template <typename TABLE_T>
__global__ void __launch_bounds__(256) grad_norm_kernel(const TABLE_T t, const double* __restrict__ parts, uint32_t nparts, float scale,
                                                        float* __restrict__ norm, float* __restrict__ each) {
    __shared__ double lds4[4];
    const int i = (int)blockIdx.x - 1;
    if (i < 0 && !norm) return;
    const uint32_t k0 = i < 0 ? 0 : t.first[i], k1 = i < 0 ? nparts : t.first[i + 1];
    double s = 0.0;
#pragma unroll 16
    for (uint32_t k = k0 + threadIdx.x; k < k1; k += 256) s += parts[k];
    s = block_sum(s, lds4);
    if (threadIdx.x == 0) *(i < 0 ? norm : each + i) = (float)(sqrt(s) * (double)scale);
}

template <bool NT, typename T>
__device__ __forceinline__ void scale_run(const T* src, T* dst, uint32_t n, GradScale f) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t nv = n / V;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < nv; i += 256) {
        float v[V];
        load_vec<T, V>(src + (size_t)i * V, v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = f(v[k]);
        if (NT) store_vec_nt<T, V>(dst + (size_t)i * V, v);
        else store_vec<T, V>(dst + (size_t)i * V, v);
    }
    const uint32_t t = nv * V + threadIdx.x;
    if (t < n) dst[t] = (T)f((float)src[t]);
}

template <bool NT, typename TABLE_T>
__global__ void __launch_bounds__(256) grad_scale_kernel(const TABLE_T t, const ClipArgs a) {
    __shared__ double lds4[4];
    const Chunk c = chunk_of(t, blockIdx.x);
    const GradScale f = clip_factor(a, a.s0, lds4);
    if (f.f == 1.f && f.e == 0 && c.src == c.dst) return;   // in place and nothing to do
    if (c.type == SR_T_F32) scale_run<NT>((const float*)c.src, (float*)c.dst, c.n, f);
    else if (c.type == SR_T_BF16) scale_run<NT>((const bf16_t*)c.src, (bf16_t*)c.dst, c.n, f);
    else scale_run<NT>((const f16_t*)c.src, (f16_t*)c.dst, c.n, f);
}

// all partial sums to one behind them
__global__ void __launch_bounds__(1024) grad_join_kernel(double* __restrict__ parts, uint32_t n) {
    __shared__ double lds[16];
    double s = 0.0;
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < n; i += 1024) s += parts[i];
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 16; ++w) s += lds[w];
    parts[n] = s;
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
    Table t;
    uint32_t blocks = 0;
    int k = 0;
    for (int i = 0; i < n; ++i) {
        if (!pieces[i].n) continue;
        if (k == TABLE) return hipErrorInvalidValue;
        t.e[k++] = {pieces[i].src, nullptr, pieces[i].n | pieces[i].type << 30, blocks};
        blocks += (uint32_t)grad_chunks(pieces[i].n, chunk);
    }
    if (!k) return hipSuccess;
    t.count = k, t.chunk = chunk;
    grad_partials_kernel<<<blocks, 256, 0, s>>>(t, parts);
    return hipGetLastError();
}

hipError_t launch_flat_partials(const float* g, int64_t n, double* parts, int* nparts, hipStream_t s) {
    GradPiece p[64];
    const uint32_t chunk = grad_chunk(n);
    int k = 0;
    *nparts = 0;
    for (int64_t at = 0; at < n; at += GRAD_PIECE, ++k) {
        if (k == 64) return hipErrorInvalidValue;
        p[k] = {g + at, (uint32_t)std::min<int64_t>(n - at, GRAD_PIECE), SR_T_F32};
        *nparts += (int)grad_chunks(p[k].n, chunk);
    }
    return launch_grad_partials(p, k, chunk, parts, s);
}

}  // namespace sr

// ------------------------------------------------------------------------------------------------- C ABI
struct sr_tensors {
    int device = 0;
    std::vector<sr_tensor_desc> list;
    std::vector<Piece> pieces;               // dst: the tensor itself
    std::vector<uint32_t> first;             // first partial sum of every tensor, and their number
    std::vector<std::pair<const char*, const char*>> sorted;   // byte ranges by address
    uint32_t chunk = 0;
    int64_t bytes = 0;
    bool overlap = false;                    // two tensors share memory
    Record* d_records = nullptr;             // of every chunk (sr_tensors_upload), behind them `first`
};

#define GC_TRY(call)          \
    do {                      \
        const int rc_ = call; \
        if (rc_) return rc_;  \
    } while (0)

namespace {

// Records of lists that are gone.  They are freed by the next upload on their device: hipFree waits for the calls that may still read
// them, and would end a capture that happens to be under way where a list goes out of scope.
std::mutex g_retired_mu;
std::vector<std::pair<int, Record*>> g_retired;

// workspace: the partial sums; for a list that does not fit the kernel arguments, the records of both sides
size_t parts_bytes(const sr_tensors* t) { return ((size_t)t->first.back() + 1) * sizeof(double); }
size_t workspace_of(const sr_tensors* t) {
    return parts_bytes(t) + (t->pieces.size() > TABLE ? 2 * t->first.back() * sizeof(Record) : 0);
}

// The kernel arguments for pieces [at, at + count) of t, written to out's tensors
void fill(Table& a, const sr_tensors* t, const sr_tensors* out, size_t at) {
    a.count = (int)std::min<size_t>(t->pieces.size() - at, TABLE);
    a.chunk = t->chunk;
    for (int i = 0; i < a.count; ++i) {
        a.e[i] = t->pieces[at + i];
        a.e[i].dst = out->pieces[at + i].dst;
    }
}

// Does a call on `st` go by what sr_tensors_upload left of the lists?  A captured one does not: a graph may outlive the list.
hipError_t uploaded(const sr_tensors* t, const sr_tensors* out, hipStream_t st, bool* yes) {
    *yes = false;
    if (!t->d_records || !out->d_records) return hipSuccess;
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    const hipError_t e = hipStreamIsCapturing(st, &capture);
    *yes = capture == hipStreamCaptureStatusNone;
    return e;
}

// Partial sums of the whole list, and with `c` the scaled gradients
hipError_t launch_list(const sr_tensors* t, const sr_tensors* out, void* ws, const ClipArgs* c, hipStream_t st) {
    const uint32_t blocks = t->first.back();
    if (!blocks) return hipSuccess;
    auto run = [&](const auto& table) {
        double* parts = (double*)ws;
        grad_partials_kernel<<<blocks, 256, 0, st>>>(table, parts);
        if (!c) return hipGetLastError();
        ClipArgs a = *c;
        if (blocks > JOIN_FROM) {
            grad_join_kernel<<<1, 1024, 0, st>>>(parts, blocks);
            a.parts = parts + blocks, a.n0 = 1;
        }
        if (t->bytes > PAST_CACHES) grad_scale_kernel<true><<<blocks, 256, 0, st>>>(table, a);
        else grad_scale_kernel<false><<<blocks, 256, 0, st>>>(table, a);
        return hipGetLastError();
    };
    bool have;
    const hipError_t e = uploaded(t, out, st, &have);
    if (e != hipSuccess) return e;
    Records r = {t->d_records, out->d_records};
    if (have) return run(r);
    Table a;
    if (t->pieces.size() <= TABLE) {
        fill(a, t, out, 0);
        return run(a);
    }
    Record *src = (Record*)((char*)ws + parts_bytes(t)), *dst = src + blocks;
    for (size_t at = 0; at < t->pieces.size(); at += TABLE) {
        fill(a, t, out, at);
        grad_records_kernel<<<a.count, 64, 0, st>>>(a, src, dst);
    }
    r = {src, dst};
    return run(r);
}

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
                t->pieces.push_back({(const char*)d.data + at * b, (char*)d.data + at * b, m | (uint32_t)d.type << 30, parts});
                parts += (uint32_t)grad_chunks(m, t->chunk);
            }
            t->first.push_back(parts);
            t->bytes += d.count * b;
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

int sr_tensors_upload(sr_tensors* t) {
    const char* who = "sr_tensors_upload";
    if (!t) return fail(nullptr, SR_ERR_ARG, "%s: the tensor list is NULL", who);
    OnDevice on;
    GC_TRY(on.enter(t->device));
    {
        std::lock_guard<std::mutex> lock(g_retired_mu);
        auto gone = std::remove_if(g_retired.begin(), g_retired.end(), [&](const std::pair<int, Record*>& r) {
            return r.first == t->device && hipFree(r.second) == hipSuccess;
        });
        g_retired.erase(gone, g_retired.end());
    }
    const size_t n = t->first.back();
    if (t->d_records || !n) return SR_OK;
    try {
        std::vector<Record> r;
        r.reserve(n);
        for (const Piece& p : t->pieces) {
            const uint32_t all = p.n & 0x3fffffffu, type = p.n >> 30;
            for (uint32_t at = 0; at < all; at += t->chunk)
                r.push_back({(const char*)p.src + (size_t)at * type_bytes((int)type), std::min(t->chunk, all - at), type});
        }
        Record* d = nullptr;
        HIPCHK(nullptr, hipMalloc((void**)&d, n * sizeof(Record) + t->first.size() * 4));
        hipError_t e = hipMemcpy(d, r.data(), n * sizeof(Record), hipMemcpyHostToDevice);
        if (e == hipSuccess) e = hipMemcpy(d + n, t->first.data(), t->first.size() * 4, hipMemcpyHostToDevice);
        if (e != hipSuccess) {
            (void)hipFree(d);
            return fail(nullptr, SR_ERR_HIP, "%s: hipMemcpy failed: %s", who, hipGetErrorString(e));
        }
        t->d_records = d;
    } catch (const std::bad_alloc&) {
        return fail(nullptr, SR_ERR_ARG, "%s: out of host memory", who);
    }
    return SR_OK;
}

int sr_tensors_destroy(sr_tensors* t) {
    if (!t) return SR_OK;
    if (t->d_records) {
        std::lock_guard<std::mutex> lock(g_retired_mu);
        try {
            g_retired.emplace_back(t->device, t->d_records);
        } catch (const std::bad_alloc&) {    // they stay until the process ends
        }
    }
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
    GC_TRY(launched(launch_list(t, t, workspace, nullptr, st), who));
    bool have;
    GC_TRY(launched(uploaded(t, t, st, &have), who));
    if (have) {
        const EachRecords e = {(const uint32_t*)(t->d_records + t->first.back())};
        grad_norm_kernel<<<1 + (d_norms ? (int)n : 0), 256, 0, st>>>(e, parts, t->first.back(), scale, d_norm, d_norms);
        return launched(hipGetLastError(), who);
    }
    EachTable e;
    size_t at = 0;
    do {
        const int count = d_norms ? (int)std::min<size_t>(n - at, EACH_MAX) : 0;
        for (int i = 0; i <= count; ++i) e.first[i] = t->first[at + i];
        grad_norm_kernel<<<1 + count, 256, 0, st>>>(e, parts, t->first.back(), scale, at ? nullptr : d_norm, d_norms + at);
        GC_TRY(launched(hipGetLastError(), who));
        at += count;
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
    if (t->pieces.empty()) {
        grad_zero_norm_kernel<<<1, 1, 0, st>>>(d_norm);
        return launched(hipGetLastError(), who);
    }
    const ClipArgs c = {(const double*)workspace, (int)t->first.back(), 0, scale, 0.f, max_norm, d_norm};
    return launched(launch_list(t, out, workspace, &c, st), who);
}

}  // extern "C"
