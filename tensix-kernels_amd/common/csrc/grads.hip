// grads.hip: the global norm of a model's gradients and clipping by it for MI355X (gfx950), behind include/grads.h.
//
// A launch takes up to 128 tensors of any sizes and types, whose addresses and sizes are its arguments, so that nothing about them
// goes through memory first. They are cut into chunks of 8192 values, which a grid of at most 2048 workgroups takes in turn (of
// gr_squares all are on the card at once, of gr_clip, whose lanes hold more registers, 1280); each leaves one sum of squares. The next
// launch adds those up in every workgroup for itself (16 KB at most a launch of them, which the caches hold), in one order, and is the
// clip itself, or one workgroup for the norm alone: no atomics, two launches for 128 tensors. Of many launches' sums one workgroup adds
// up all first (gr_total). The clip takes the chunks the other way round, the last ones read first, which the 256 MB cache behind the L2s
// still holds.
//
// Bound by memory: one read, and for a clip a second and one write. 252 M bf16 values in 145 tensors, two launches of 70 and 16 us (5.9
// TB/s) and 4 for the norm; 283 M float32 values clipped 189 us for the squares (6.0 TB/s) and 416 for the rest (5.5; a large copy
// reaches 4.9). 18 tensors of 190 k values: two launches, 5.5 and 1.7 us, less than the host's 19.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "dense_reader.h"
#include "grads.h"

#pragma clang fp contract(off)

namespace {

constexpr int CHUNK = 8192, LANES = 256;  // values
constexpr int MOST = DR_GRADS_LIST;        // tensors a launch: its arguments fit 4 KB
constexpr int GRID = 2048;                 // 8 workgroups a CU of gr_squares (60 registers a lane), 5 of gr_clip (92) at once
static_assert(GRID * 8 == DR_GRADS_LIST_BYTES, "the header's bytes");

struct List {
    const void* in[MOST];
    void* out[MOST];
    long long size[MOST];
    uint32_t end[MOST];  // chunks of the tensors up to and with this one
    uint8_t kind[MOST];  // type, out's type << 2, whether both lie at multiples of 16 bytes << 4
    int count;
    uint32_t chunks;
};
static_assert(sizeof(List) <= 4000, "a launch's arguments fit 4 KB");

// a chunk's tensor (all lanes look, 64 tensors at a time), and the chunk within it
__device__ __forceinline__ int tensor_of(const List& a, uint32_t chunk, uint32_t& within) {
    const int lane = threadIdx.x & 63;
    int t = 0;
#pragma unroll
    for (int i = 0; i < MOST; i += 64) t += __popcll(__ballot(i + lane < a.count && a.end[i + lane] <= chunk));
    t = __builtin_amdgcn_readfirstlane(t);
    within = chunk - (t ? a.end[t - 1] : 0);
    return t;
}

template <int TYPE>
__device__ __forceinline__ float one(const void* p, long long i) {
    if constexpr (TYPE == DR_GRADS_F32) return reinterpret_cast<const float*>(p)[i];
    else if constexpr (TYPE == DR_GRADS_BF16) return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
    else return (float)reinterpret_cast<const _Float16*>(p)[i];
}

// N values of a lane: 16 bytes of the wider type, so that the lanes' lie one after another, loads and stores
template <int TYPE, int N>
struct Some {
    typedef __attribute__((__vector_size__(N * (TYPE == DR_GRADS_F32 ? 4 : 2)))) uint8_t raw;
    typedef __attribute__((__vector_size__(N * sizeof(float)))) float floats;
    raw v;
    __device__ __forceinline__ void load(const void* p, long long i) {
        v = *reinterpret_cast<const raw*>(reinterpret_cast<const char*>(p) + i * (TYPE == DR_GRADS_F32 ? 4 : 2));
    }
    __device__ __forceinline__ floats get() const {
        if constexpr (TYPE == DR_GRADS_F32) return __builtin_bit_cast(floats, v);
        else if constexpr (TYPE == DR_GRADS_BF16) {
            typedef __attribute__((__vector_size__(N * sizeof(__bf16)))) __bf16 halves;
            return __builtin_convertvector(__builtin_bit_cast(halves, v), floats);
        } else {
            typedef __attribute__((__vector_size__(N * sizeof(_Float16)))) _Float16 halves;
            return __builtin_convertvector(__builtin_bit_cast(halves, v), floats);
        }
    }
    // (past the caches: what is read again by this call should stay there)
    static __device__ __forceinline__ void store(void* p, long long i, floats v) {
        raw* o = reinterpret_cast<raw*>(reinterpret_cast<char*>(p) + i * (TYPE == DR_GRADS_F32 ? 4 : 2));
        if constexpr (TYPE == DR_GRADS_F32) __builtin_nontemporal_store(__builtin_bit_cast(raw, v), o);
        else if constexpr (TYPE == DR_GRADS_BF16) {
            typedef __attribute__((__vector_size__(N * sizeof(__bf16)))) __bf16 halves;
            __builtin_nontemporal_store(__builtin_bit_cast(raw, __builtin_convertvector(v, halves)), o);
        } else {
            typedef __attribute__((__vector_size__(N * sizeof(_Float16)))) _Float16 halves;
            __builtin_nontemporal_store(__builtin_bit_cast(raw, __builtin_convertvector(v, halves)), o);
        }
    }
};

template <int TYPE>
__device__ __forceinline__ void put(void* p, long long i, float v) {
    if constexpr (TYPE == DR_GRADS_F32) reinterpret_cast<float*>(p)[i] = v;
    else if constexpr (TYPE == DR_GRADS_BF16) reinterpret_cast<__bf16*>(p)[i] = (__bf16)v;
    else reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
}

// The sum of the workgroup's lanes, to all of them, in one order.
__device__ __forceinline__ double block_sum(double s) {
    __shared__ double parts[LANES / 64];
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = s;
    __syncthreads();
    return (parts[0] + parts[1]) + (parts[2] + parts[3]);
}

template <int TYPE>
__device__ __forceinline__ double squares(const void* p, int n, bool vec) {
    const int tid = threadIdx.x;
    constexpr int N = TYPE == DR_GRADS_F32 ? 4 : 8, VECS = CHUNK / (N * LANES);
    typedef Some<TYPE, N> Values;
    double s = 0., t = 0.;
    auto add = [&](const Values& x) {
        const auto v = x.get();
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            s = __builtin_fma((double)v[e], (double)v[e], s);
            t = __builtin_fma((double)v[e + 1], (double)v[e + 1], t);
        }
    };
    int from = 0;
    if (vec && n == CHUNK) {
        Values v[VECS];
#pragma unroll
        for (int j = 0; j < VECS; ++j) v[j].load(p, N * (j * LANES + tid));
#pragma unroll
        for (int j = 0; j < VECS; ++j) add(v[j]);
        from = n;
    } else if (vec) {
        for (int i = tid; i < n / N; i += LANES) {
            Values v;
            v.load(p, N * i);
            add(v);
        }
        from = n / N * N;
    }
#pragma unroll 8
    for (int i = from + tid; i < n; i += LANES) {
        const double v = one<TYPE>(p, i);
        s = __builtin_fma(v, v, s);
    }
    return s + t;
}

__device__ __forceinline__ const char* at(const void* p, int type, long long i) {
    return reinterpret_cast<const char*>(p) + i * (type == DR_GRADS_F32 ? 4 : 2);
}

__global__ __launch_bounds__(LANES) void gr_squares(const List a, double* sums) {
    double s = 0.;
    for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
        uint32_t within;
        const int t = tensor_of(a, c, within), kind = a.kind[t], type = kind & 3;
        const long long first = (long long)within * CHUNK;
        const int n = (int)min((long long)CHUNK, a.size[t] - first);
        const void* p = at(a.in[t], type, first);
        const bool vec = kind & 16;
        if (type == DR_GRADS_F32) s += squares<DR_GRADS_F32>(p, n, vec);
        else if (type == DR_GRADS_BF16) s += squares<DR_GRADS_BF16>(p, n, vec);
        else s += squares<DR_GRADS_F16>(p, n, vec);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// the sums' sum, the same in every workgroup, and its square root
__device__ __forceinline__ double sum_of(const double* sums, int count) {
    double s = 0.;
#pragma unroll 8
    for (int i = threadIdx.x; i < count; i += LANES) s += sums[i];
    return block_sum(s);
}

__device__ __forceinline__ double norm_of(const double* sums, int count) { return sqrt(sum_of(sums, count)); }

__global__ __launch_bounds__(LANES) void gr_norm(const double* sums, int count, float* norm) {
    const double v = norm_of(sums, count);
    if (threadIdx.x == 0) *norm = (float)v;
}

// Of several launches the sums' sum, in the place of the first: the clip's launches, as many, would each add up all of them in every
// workgroup. From ADDED (launches times sums) on: 384 tensors of 16 chunks 72 us with it and 76 without, 1024 193 and
// 255, 8192 1.7 and 8.3 ms; but 384 of 3 chunks 37.4 and 36.4, 256 of one 20.4 and 19.1 us.
constexpr long long ADDED = 8192;
__global__ __launch_bounds__(LANES) void gr_total(double* sums, int count) {
    const double s = sum_of(sums, count);
    if (threadIdx.x == 0) *sums = s;  // (all have read theirs: block_sum's barrier)
}

template <int TYPE, int OUT>
__device__ __forceinline__ void scale(const void* p, void* o, int n, bool vec, float f) {
    constexpr int N = TYPE == DR_GRADS_F32 || OUT == DR_GRADS_F32 ? 4 : 8, VECS = CHUNK / (N * LANES);
    const int tid = threadIdx.x;
    int from = 0;
    if (vec && n == CHUNK) {
        Some<TYPE, N> v[VECS];
#pragma unroll
        for (int j = 0; j < VECS; ++j) v[j].load(p, N * (j * LANES + tid));
#pragma unroll
        for (int j = 0; j < VECS; ++j) Some<OUT, N>::store(o, N * (j * LANES + tid), v[j].get() * f);
        return;
    }
    if (vec) {
        for (int i = tid; i < n / N; i += LANES) {
            Some<TYPE, N> v;
            v.load(p, N * i);
            Some<OUT, N>::store(o, N * i, v.get() * f);
        }
        from = n / N * N;
    }
#pragma unroll 8
    for (int i = from + tid; i < n; i += LANES) put<OUT>(o, i, one<TYPE>(p, i) * f);
}

template <int TYPE>
__device__ __forceinline__ void scale(const void* p, void* o, int out, int n, bool vec, float f) {
    if (out == DR_GRADS_F32) scale<TYPE, DR_GRADS_F32>(p, o, n, vec, f);
    else if (out == DR_GRADS_BF16) scale<TYPE, DR_GRADS_BF16>(p, o, n, vec, f);
    else scale<TYPE, DR_GRADS_F16>(p, o, n, vec, f);
}

// sums: of `count` workgroups, or NULL: the norm is there
__global__ __launch_bounds__(LANES) void gr_clip(const List a, const double* sums, int count, float* norm, double max_norm) {
    const double v = sums ? norm_of(sums, count) : (double)*norm;
    if (sums && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    const double q = max_norm / (v + 1e-6);
    // (a NaN of the norm stays one; no limit clips nothing, whatever else the norm is)
    const float f = q >= 1. || (max_norm == __builtin_inf() && v == v) ? 1.f : (float)q;
    for (uint32_t i = blockIdx.x; i < a.chunks; i += gridDim.x) {
        uint32_t within;
        const int t = tensor_of(a, a.chunks - 1 - i, within), kind = a.kind[t], type = kind & 3, out = kind >> 2 & 3;
        if (f == 1.f && a.in[t] == a.out[t]) continue;  // (they are there)
        const long long first = (long long)within * CHUNK;
        const int n = (int)min((long long)CHUNK, a.size[t] - first);
        const void* p = at(a.in[t], type, first);
        void* o = const_cast<char*>(at(a.out[t], out, first));
        const bool vec = kind & 16;
        if (type == DR_GRADS_F32) scale<DR_GRADS_F32>(p, o, out, n, vec, f);
        else if (type == DR_GRADS_BF16) scale<DR_GRADS_BF16>(p, o, out, n, vec, f);
        else scale<DR_GRADS_F16>(p, o, out, n, vec, f);
    }
}

// --- the host -----------------------------------------------------------------------------------------------------------

constexpr int WIDTH[] = {4, 2, 2};

bool type_ok(int t) { return t >= 0 && t <= 2; }

bool list_ok(const dr_grads* a, bool clip) {
    if (a == nullptr || a->count < 0 || a->count > (1 << 20)) return false;
    if (a->count && (!a->in || !a->sizes || !a->types || (clip && (!a->out || !a->out_types)))) return false;
    long long all = 0;
    for (int i = 0; i < a->count; ++i) {
        if (a->sizes[i] < 0 || a->sizes[i] > (1ll << 40) || !type_ok(a->types[i]) || (clip && !type_ok(a->out_types[i]))) return false;
        all += a->sizes[i];
        if (all > (1ll << 40)) return false;
        if (a->sizes[i] && (!a->in[i] || reinterpret_cast<uintptr_t>(a->in[i]) % WIDTH[a->types[i]])) return false;
        if (clip && a->sizes[i] &&
            (!a->out[i] || reinterpret_cast<uintptr_t>(a->out[i]) % WIDTH[a->out_types[i]] ||
             (a->out[i] == a->in[i] && a->out_types[i] != a->types[i])))
            return false;
    }
    return true;
}

struct Span {
    uintptr_t lo, hi;
    int id;
    bool out;
};

// Whether no out shares memory with any other tensor's in or out or with the norm, nor with its own in but all of it (swept by
// address). -1: no memory.
int apart(const dr_grads* a) {
    Span* s = new (std::nothrow) Span[2 * (size_t)a->count + 1];
    if (!s) return -1;
    int n = 0;
    const uintptr_t norm = reinterpret_cast<uintptr_t>(a->norm);  // (read or written while the others are)
    s[n++] = Span{norm, norm + 4, -1, !a->given};
    for (int i = 0; i < a->count; ++i) {
        if (!a->sizes[i]) continue;
        const uintptr_t in = reinterpret_cast<uintptr_t>(a->in[i]), out = reinterpret_cast<uintptr_t>(a->out[i]);
        s[n++] = Span{out, out + a->sizes[i] * WIDTH[a->out_types[i]], i, true};
        if (in != out) s[n++] = Span{in, in + a->sizes[i] * WIDTH[a->types[i]], i, false};  // (in place: as the out)
    }
    std::sort(s, s + n, [](const Span& x, const Span& y) { return x.lo < y.lo; });
    uintptr_t outs = 0, ins = 0;  // where the last out, and the last in, ends
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
        ok = s[i].lo >= outs && (!s[i].out || s[i].lo >= ins);
        // (of two that begin at one place the first could be the in)
        if (i + 1 < n && s[i + 1].lo == s[i].lo && (s[i].out || s[i + 1].out)) ok = false;
        uintptr_t& end = s[i].out ? outs : ins;
        if (s[i].hi > end) end = s[i].hi;
    }
    delete[] s;
    return ok;
}

// the next tensors of a launch, from `i` on and before `to`; false: none left
bool fill(const dr_grads* a, bool clip, int& i, int to, List& l) {
    l.count = 0, l.chunks = 0;
    for (; i < to && l.count < MOST; ++i) {
        const long long n = a->sizes[i], chunks = (n + CHUNK - 1) / CHUNK;
        if (!n) continue;
        const int k = l.count++;
        l.in[k] = a->in[i];
        l.out[k] = clip ? a->out[i] : nullptr;
        l.size[k] = n;
        l.chunks += (uint32_t)chunks;  // (2^40 values are 2^27)
        l.end[k] = l.chunks;
        const bool vec = reinterpret_cast<uintptr_t>(a->in[i]) % 16 == 0 && (!clip || reinterpret_cast<uintptr_t>(a->out[i]) % 16 == 0);
        l.kind[k] = (uint8_t)(a->types[i] | (clip ? a->out_types[i] << 2 : 0) | vec << 4);
    }
    return l.count > 0;
}

int groups(uint32_t chunks) { return (int)std::min<uint32_t>(chunks, GRID); }

// the sums' launches, how many; how many sums there are
int squares_of(const dr_grads* a, hipStream_t st, int& lists) {
    List l;
    int count = 0;
    lists = 0;
    for (int i = 0; fill(a, false, i, a->count, l); ++lists) {
        const int g = groups(l.chunks);
        hipLaunchKernelGGL(gr_squares, dim3(g), dim3(LANES), 0, st, l, reinterpret_cast<double*>(a->workspace) + count);
        count += g;
    }
    return count;
}

bool call_ok(const dr_grads* a) {
    return a->norm && reinterpret_cast<uintptr_t>(a->norm) % 4 == 0 &&
           (a->workspace_bytes >= dr_grads_workspace_bytes(a) && (a->workspace_bytes == 0 || (a->workspace && reinterpret_cast<uintptr_t>(a->workspace) % 8 == 0)));
}

}  // namespace

extern "C" int64_t dr_grads_workspace_bytes(const dr_grads* a) {
    if (!list_ok(a, false)) return -1;
    List l;
    int64_t bytes = 0;
    for (int i = 0; fill(a, false, i, a->count, l);) bytes += 8ll * groups(l.chunks);
    return bytes;
}

extern "C" int dr_grads_norm(const dr_grads* a) {
    if (!list_ok(a, false) || !call_ok(a)) return DR_EINVAL;
    const hipStream_t st = reinterpret_cast<hipStream_t>(a->stream);
    int lists;
    const int count = squares_of(a, st, lists);
    hipLaunchKernelGGL(gr_norm, dim3(1), dim3(LANES), 0, st, reinterpret_cast<const double*>(a->workspace), count, a->norm);
    return hipGetLastError() == hipSuccess ? DR_OK : DR_EHIP;
}

extern "C" int dr_grads_clip(const dr_grads* a) {
    if (!list_ok(a, true) || !(a->max_norm >= 0.) || !a->norm || reinterpret_cast<uintptr_t>(a->norm) % 4 || (!a->given && !call_ok(a)))
        return DR_EINVAL;
    const int ok = apart(a);
    if (ok <= 0) return ok < 0 ? DR_EHIP : DR_EINVAL;
    const hipStream_t st = reinterpret_cast<hipStream_t>(a->stream);
    double* sums = reinterpret_cast<double*>(a->workspace);
    int lists = 0, count = a->given ? 0 : squares_of(a, st, lists);
    if (lists > 1 && (long long)lists * count >= ADDED) {
        hipLaunchKernelGGL(gr_total, dim3(1), dim3(LANES), 0, st, sums, count);
        count = 1;
    }
    bool any = false;
    for (int to = a->count; to > 0;) {  // (the last tensors first: they were read last)
        int from = to;
        for (int k = 0; from > 0 && k < MOST; k += a->sizes[from] != 0) --from;
        List l;
        int i = from;
        if (fill(a, true, i, to, l)) {
            hipLaunchKernelGGL(gr_clip, dim3(groups(l.chunks)), dim3(LANES), 0, st, l, a->given ? nullptr : sums, count, a->norm, a->max_norm);
            any = true;
        }
        to = from;
    }
    if (!any && !a->given) hipLaunchKernelGGL(gr_norm, dim3(1), dim3(LANES), 0, st, sums, 0, a->norm);
    return hipGetLastError() == hipSuccess ? DR_OK : DR_EHIP;
}
