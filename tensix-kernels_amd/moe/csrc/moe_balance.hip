// moe_balance.hip: the router's balance loss, each expert's count and the gradient of the logits on MI355X (gfx950), behind
// dr_moe_balance (include/moe.h).
//
// A row lies over L lanes (16 up to 256 experts, a wavefront beyond), each with runs of four experts, so that a load takes 16
// bytes a lane, a wavefront works on four rows at once, and a row's softmax or sigmoids and their sum are a few register
// operations and a butterfly of log2(L) steps. The sums over rows stay in registers until the wavefront's rows are done.
//   balance_sum_k   a workgroup's rows: the sum of p and the counts (LDS), written for the workgroup
//   balance_grad_k  every workgroup joins the workgroups' sums for itself, in order (cheaper than a launch of its own in
//                   between while they are few; balance_slice_k otherwise), then the logits' gradient of its rows, p computed
//                   again; balance_join_k: the join alone. After a call that kept the counts (DR_BALANCE_BACKWARD) there is nothing to
//                   join, and balance_grad_k is all that runs
//   balance_one_k   all of it by one workgroup, a batch of few rows or one of many batches: one launch and no memory between
//                   (32 rows x 32 experts: 4.8 us in a graph, two launches 8; called eagerly 12 and 16, the host's)
// What bounds it: the logits read twice and the gradient written once; at a few rows the launches.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe.h"

#pragma clang fp contract(off)

namespace {

constexpr int T = 512;      // lanes a workgroup
constexpr int W = T / 64;
constexpr int MAXE = 1024;  // experts

struct Bal {
    dr_balance a;
    float2* sums;         // [batch][groups][E] sum of p, count (its bits)
    int* live;            // [batch][groups] rows that count
    int groups;           // workgroups a batch
    const float2* in;     // [batch][parts][E], [batch][parts]: the sums to be joined, the workgroups' own or (parts 1) what
    const int* in_live;   //     balance_slice_k made of them
    int parts;
    int vec;              // the logits' rows can be read 16 bytes at a time
    int gvec;             // and dlogits' written so
    int given;            // the gradient alone: a.kept holds the rows that count and the counts
};

template <int CONTROL>
__device__ __forceinline__ float turned(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CONTROL, 0xF, 0xF, true));
}
template <int L, typename F>
__device__ __forceinline__ float over(float v, F&& f) {
    v = f(v, turned<0xB1>(v));   // quad_perm 1 0 3 2
    v = f(v, turned<0x4E>(v));   // quad_perm 2 3 0 1
    v = f(v, turned<0x141>(v));  // row_half_mirror
    v = f(v, turned<0x140>(v));  // row_mirror
#pragma unroll
    for (int o = 16; o < L; o <<= 1) v = f(v, __shfl_xor(v, o));
    return v;
}
template <int L>
__device__ __forceinline__ float sum_over(float v) {
    return over<L>(v, [](float a, float b) { return a + b; });
}
template <int L>
__device__ __forceinline__ float max_over(float v) {
    return over<L>(v, [](float a, float b) { return fmaxf(a, b); });
}

// a row's logits: value 4 i + c is expert 4 (l + L i) + c; past the experts -inf
template <int L, int N>
__device__ __forceinline__ void row_load(const Bal& b, long long row, int l, float (&z)[4 * N]) {
    const float* at = b.a.logits + row * b.a.ld_logits;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = 4 * (l + L * i);
        if (b.vec && e + 4 <= b.a.experts) {
            const float4 v = *reinterpret_cast<const float4*>(at + e);
            z[4 * i] = v.x, z[4 * i + 1] = v.y, z[4 * i + 2] = v.z, z[4 * i + 3] = v.w;
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) z[4 * i + c] = e + c < b.a.experts ? at[e + c] : -INFINITY;
        }
    }
}

// What a row takes from memory, asked for before the row ahead of it is worked on (two rows ahead: the same, within 3 %). Past
// the batch's last row that one again: every lane takes part in the butterflies.
template <int N>
struct Row {
    float z[4 * N];
    uint32_t id;  // lane l's slot
    uint8_t on;
};
template <int L, int N, bool IDS>
__device__ __forceinline__ void row_get(const Bal& b, int batch, int r, int l, Row<N>& to) {
    const dr_balance& a = b.a;
    const long long row = (long long)batch * a.rows + min(r, a.rows - 1);
    row_load<L, N>(b, row, l, to.z);
    if constexpr (IDS) {
        to.id = 0xFFFFFFFFu;
        if (l < a.k) {
            const long long at = row * a.ld_ids + l;
            to.id = a.ids32 ? reinterpret_cast<const uint32_t*>(a.ids)[at] : reinterpret_cast<const uint16_t*>(a.ids)[at];
        }
    }
    to.on = a.mask ? a.mask[row] : 1;
}

// the row's p from its logits, in place (0 past the experts); a row of no expert above -inf has p 0. down: 1 less the sigmoid,
// as a product, which keeps its accuracy where the sigmoid nears 1.
template <int L, int N, bool SIG>
__device__ __forceinline__ void row_p(float (&p)[4 * N], float (&down)[SIG ? 4 * N : 1]) {
    float total = 0.f;
    if constexpr (SIG) {
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) {
            const float x = __expf(-p[i]);
            p[i] = __builtin_amdgcn_rcpf(1.f + x);
            down[i] = x == INFINITY ? 1.f : x * p[i];
            total += p[i];
        }
    } else {
        float top = p[0];
#pragma unroll
        for (int i = 1; i < 4 * N; ++i) top = fmaxf(top, p[i]);
        top = max_over<L>(top);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) {
            p[i] = __expf(p[i] - base);
            total += p[i];
        }
    }
    total = sum_over<L>(total);
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) p[i] *= inv;
}

// a workgroup's rows in LDS: cnt, and by wavefront the sum of p and the rows that count
template <int L, int N>
struct Sums {
    int cnt[L * 4 * N];
    float p[W][L * 4 * N];
    int rows[W];
};

template <int L, int N, bool SIG>
__device__ __forceinline__ void sum_rows(const Bal& b, int g, int batch, Sums<L, N>& S) {
    constexpr int R = T / L;  // rows at once
    const dr_balance& a = b.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l = tid % L;
    for (int e = tid; e < a.experts; e += T) S.cnt[e] = 0;
    __syncthreads();
    float sum[4 * N];
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) sum[i] = 0.f;
    int n = 0;
    const int step = b.groups * R;
    Row<N> next;
    row_get<L, N, true>(b, batch, g * R + tid / L, l, next);
    for (int r = g * R + tid / L; r - tid / L < a.rows; r += step) {
        Row<N> now = next;
        row_get<L, N, true>(b, batch, r + step, l, next);
        const bool on = r < a.rows && now.on;
        float down[SIG ? 4 * N : 1];
        row_p<L, N, SIG>(now.z, down);
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) sum[i] += on ? now.z[i] : 0.f;
        n += on;
        if (on && now.id < (uint32_t)a.experts) atomicAdd(&S.cnt[now.id], 1);
    }
    // the wavefront's rows, then the workgroup's, in order
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
#pragma unroll
        for (int o = L; o < 64; o <<= 1) sum[i] += __shfl_xor(sum[i], o);
    }
#pragma unroll
    for (int o = L; o < 64; o <<= 1) n += __shfl_xor(n, o);
    if (lane < L) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            *reinterpret_cast<float4*>(&S.p[wave][4 * (l + L * i)]) =
                make_float4(sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]);
    }
    if (lane == 0) S.rows[wave] = n;
    __syncthreads();
}

template <int L, int N, bool SIG>
__global__ __launch_bounds__(T) void balance_sum_k(const Bal b) {
    __shared__ __attribute__((aligned(16))) Sums<L, N> S;
    const dr_balance& a = b.a;
    const int tid = threadIdx.x, g = blockIdx.x % b.groups, batch = blockIdx.x / b.groups;
    sum_rows<L, N, SIG>(b, g, batch, S);
    for (int e = tid; e < a.experts; e += T) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += S.p[w][e];
        b.sums[(long long)blockIdx.x * a.experts + e] = make_float2(v, __int_as_float(S.cnt[e]));
    }
    if (tid == 0) {
        int v = 0;
        for (int w = 0; w < W; ++w) v += S.rows[w];
        b.live[blockIdx.x] = v;
    }
}

struct Joined {
    float p[MAXE], f[MAXE];  // the sums of p; counts, then E count / counts
    float2 part[T];          // experts by slices of the workgroups
    float red[W];
    int tot[W], live[W];
};

// A batch's sums (J.p, J.f) and the lane's share of its rows that count to f; 1 / those rows is returned. write: the counts, the
// loss and what a backward takes too.
__device__ __forceinline__ float finish(const Bal& b, int batch, bool write, int rows, Joined& J) {
    const dr_balance& a = b.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int total = 0, *kept = write && a.kept ? a.kept + (long long)batch * (1 + a.experts) : nullptr;
    for (int e = tid; e < a.experts; e += T) {
        const int c = __float_as_int(J.f[e]);
        total += c;
        if (write) a.counts[(long long)batch * a.experts + e] = c;
        if (kept) kept[1 + e] = c;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) rows += __shfl_xor(rows, o), total += __shfl_xor(total, o);
    if (lane == 0) J.live[wave] = rows, J.tot[wave] = total;
    __syncthreads();
    rows = total = 0;
    for (int w = 0; w < W; ++w) rows += J.live[w], total += J.tot[w];
    if (kept && tid == 0) *kept = rows;
    const float per = rows ? 1.f / (float)rows : 0.f;
    float loss = 0.f;
    for (int e = tid; e < a.experts; e += T) {
        const float f = total ? (float)a.experts * ((float)__float_as_int(J.f[e]) / (float)total) : 0.f;
        J.f[e] = f;
        loss += f * (J.p[e] * per);
    }
    if (write) {
        loss = sum_over<64>(loss);
        if (lane == 0) J.red[wave] = loss;
    }
    __syncthreads();
    if (write && tid == 0) {
        for (int w = 1; w < W; ++w) loss += J.red[w];
        a.loss[batch] = loss;
    }
    return per;
}

// f from the rows and counts that an earlier call kept; no sums of p, which the gradient does not need
__device__ __forceinline__ float given(const Bal& b, int batch, Joined& J) {
    const int tid = threadIdx.x, *kept = b.a.kept + (long long)batch * (1 + b.a.experts);
    for (int e = tid; e < b.a.experts; e += T) {
        J.p[e] = 0.f;
        J.f[e] = __int_as_float(kept[1 + e]);
    }
    return finish(b, batch, false, tid == 0 ? *kept : 0, J);
}

// the batch's sums over its parts, finished
__device__ __forceinline__ float join(const Bal& b, int batch, bool write, Joined& J) {
    const dr_balance& a = b.a;
    const int tid = threadIdx.x;
    const long long at = (long long)batch * b.parts;
    int pw = 32;  // experts at a time, by T / pw slices of the workgroups
    while (pw < a.experts && pw < T) pw *= 2;
    const int e0 = tid & (pw - 1), sl = tid / pw, slices = T / pw;
    for (int e = e0; e - e0 < a.experts; e += pw) {
        float p = 0.f;
        int c = 0;
        if (e < a.experts) {
#pragma unroll 16
            for (int g = sl; g < b.parts; g += slices) {
                const float2 v = b.in[(at + g) * a.experts + e];
                p += v.x;
                c += __float_as_int(v.y);
            }
        }
        J.part[tid] = make_float2(p, __int_as_float(c));
        __syncthreads();
        if (sl == 0 && e < a.experts) {
            for (int i = 1; i < slices; ++i) {
                const float2 v = J.part[i * pw + e0];
                p += v.x;
                c += __float_as_int(v.y);
            }
            J.p[e] = p;
            J.f[e] = __int_as_float(c);
        }
        __syncthreads();
    }
    int rows = 0;
    for (int g = tid; g < b.parts; g += T) rows += b.in_live[at + g];
    return finish(b, batch, write, rows, J);
}

// the workgroups' sums of 64 experts of a batch, an eighth of the workgroups a wavefront
__global__ __launch_bounds__(T) void balance_slice_k(const Bal b, float2* sums, int* live) {
    __shared__ float2 part[W][64];
    __shared__ int rows[W];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E = b.a.experts;
    const int slices = (E + 63) / 64, batch = blockIdx.x / slices, slice = blockIdx.x % slices, e = 64 * slice + lane;
    const long long at = (long long)batch * b.groups;
    float p = 0.f;
    int c = 0;
    if (e < E) {
#pragma unroll 16
        for (int g = wave; g < b.groups; g += W) {
            const float2 v = b.sums[(at + g) * E + e];
            p += v.x;
            c += __float_as_int(v.y);
        }
    }
    part[wave][lane] = make_float2(p, __int_as_float(c));
    int n = 0;
    if (slice == 0)
        for (int g = tid; g < b.groups; g += T) n += b.live[at + g];
#pragma unroll
    for (int o = 32; o; o >>= 1) n += __shfl_xor(n, o);
    if (lane == 0) rows[wave] = n;
    __syncthreads();
    if (wave == 0 && e < E) {
#pragma unroll
        for (int w = 1; w < W; ++w) p += part[w][lane].x, c += __float_as_int(part[w][lane].y);
        sums[(long long)batch * E + e] = make_float2(p, __int_as_float(c));
    }
    if (slice == 0 && tid == 0) {
        for (int w = 1; w < W; ++w) n += rows[w];
        live[batch] = n;
    }
}

__global__ __launch_bounds__(T) void balance_join_k(const Bal b) {
    __shared__ Joined J;
    join(b, blockIdx.x, true, J);
}

// the gradient of a workgroup's rows; next: the first of them, asked for before the sums are joined
template <int L, int N, bool SIG>
__device__ __forceinline__ void grad_rows(const Bal& b, int g, int batch, float per, Row<N>& next, const Joined& J) {
    constexpr int R = T / L;
    const dr_balance& a = b.a;
    const int tid = threadIdx.x, l = tid % L, step = b.groups * R;
    const float scale = (a.g ? a.g[batch] : 1.f) * per;
    float f[4 * N];
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
        const int e = 4 * (l + L * (i / 4)) + i % 4;
        f[i] = e < a.experts ? J.f[e] : 0.f;
    }
    for (int r = g * R + tid / L; r - tid / L < a.rows; r += step) {
        Row<N> now = next;
        row_get<L, N, false>(b, batch, r + step, l, next);
        float (&p)[4 * N] = now.z, down[SIG ? 4 * N : 1];
        row_p<L, N, SIG>(p, down);
        float mean = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) mean += p[i] * f[i];
        mean = sum_over<L>(mean);
        if (r >= a.rows) continue;
        float* d = a.dlogits + ((long long)batch * a.rows + r) * a.ld_dlogits;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = 4 * (l + L * i);
            float o[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int q = 4 * i + c;
                o[c] = now.on ? scale * (SIG ? p[q] * down[SIG ? q : 0] : p[q]) * (f[q] - mean) : 0.f;
            }
            if (b.gvec && e + 4 <= a.experts) {
                *reinterpret_cast<float4*>(d + e) = make_float4(o[0], o[1], o[2], o[3]);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (e + c < a.experts) d[e + c] = o[c];
            }
        }
        for (int e = a.experts + l; e < a.width; e += L) d[e] = 0.f;
    }
}

template <int L, int N, bool SIG>
__global__ __launch_bounds__(T) void balance_grad_k(const Bal b) {
    __shared__ Joined J;
    const int g = blockIdx.x % b.groups, batch = blockIdx.x / b.groups;
    Row<N> next;
    row_get<L, N, false>(b, batch, g * (T / L) + threadIdx.x / L, threadIdx.x % L, next);
    const float per = b.given ? given(b, batch, J) : join(b, batch, g == 0, J);
    grad_rows<L, N, SIG>(b, g, batch, per, next, J);
}

template <int L, int N, bool SIG>
__global__ __launch_bounds__(T) void balance_one_k(const Bal b, int gradient) {
    __shared__ __attribute__((aligned(16))) Sums<L, N> S;
    __shared__ Joined J;
    const int tid = threadIdx.x, batch = blockIdx.x;
    sum_rows<L, N, SIG>(b, 0, batch, S);
    Row<N> next;
    if (gradient) row_get<L, N, false>(b, batch, tid / L, tid % L, next);
    for (int e = tid; e < b.a.experts; e += T) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += S.p[w][e];
        J.p[e] = v;
        J.f[e] = __int_as_float(S.cnt[e]);
    }
    const float per = finish(b, batch, true, tid < W ? S.rows[tid] : 0, J);
    if (gradient) grad_rows<L, N, SIG>(b, 0, batch, per, next, J);
}

// Workgroups a batch, and whether their sums are joined by a launch of its own: as many workgroups as the rows fill, but no more
// than all the CUs take in one round (65536 rows x 128 experts: 26.1 us, 33.3 by 128 workgroups; two rounds and four are slower
// too, 16384 x 1024 48 and 63 to 43). Every workgroup of the gradient reads all of a batch's sums, which a launch of its own saves
// where they are more than 256 KB: 16384 rows x 1024 experts 43 us (67 without), 8192 x 256 15.9 (19.5); at 8 batches of 4096 x
// 256, 64 KB each, 25.8 (23.4 without). Up to twice a workgroup's rows one takes all (64 rows x 32 experts 6.2 us, 8.1 in two
// launches; 128 rows 9.6 and 8.1). Times in a graph.
struct Split {
    int groups;
    bool slices;
};
constexpr int JOINED = 32768;  // sums of 8 bytes that every workgroup may read
Split split_of(const dr_balance* a) {
    const int at_once = a->experts <= 256 ? T / 16 : T / 64;
    const int fit = (a->rows + at_once - 1) / at_once;
    if (fit <= 2) return {1, false};
    const int most = a->batch < 256 ? 256 / a->batch : 1, groups = fit < most ? fit : most;
    return {groups, groups * a->experts > JOINED};
}

bool valid(const dr_balance* a, int what) {
    return a != nullptr && ((what >= 1 && what <= 3) || what == DR_BALANCE_BACKWARD) && a->batch >= 1 && a->batch <= (1 << 16) && a->rows >= 1 &&
           (long long)a->batch * a->rows < (1ll << 30) && a->experts >= 1 && a->experts <= MAXE && a->k >= 1 && a->k <= 16 &&
           (long long)a->rows * a->k < (1ll << 31) &&  // (the counts are int32)
           a->width >= a->experts && a->ld_logits >= a->width && a->ld_ids >= a->k && (a->kind == 0 || a->kind == 1);
}

long long up256(long long v) { return (v + 255) & ~255ll; }

template <int L, int N, bool SIG>
void run(const Bal& b, int what, hipStream_t st) {
    if (b.given) {
        hipLaunchKernelGGL((balance_grad_k<L, N, SIG>), dim3(b.groups * b.a.batch), dim3(T), 0, st, b);
        return;
    }
    if (b.groups == 1) {
        hipLaunchKernelGGL((balance_one_k<L, N, SIG>), dim3(b.a.batch), dim3(T), 0, st, b, what & DR_BALANCE_GRAD);
        return;
    }
    const dim3 grid(b.groups * b.a.batch);
    hipLaunchKernelGGL((balance_sum_k<L, N, SIG>), grid, dim3(T), 0, st, b);
    if (b.parts == 1)
        hipLaunchKernelGGL(balance_slice_k, dim3(b.a.batch * ((b.a.experts + 63) / 64)), dim3(T), 0, st, b,
                           const_cast<float2*>(b.in), const_cast<int*>(b.in_live));
    if (what & DR_BALANCE_GRAD) hipLaunchKernelGGL((balance_grad_k<L, N, SIG>), grid, dim3(T), 0, st, b);
    else hipLaunchKernelGGL(balance_join_k, dim3(b.a.batch), dim3(T), 0, st, b);
}

template <int L, int N>
void run_kind(const Bal& b, int what, hipStream_t st) {
    if (b.a.kind) run<L, N, true>(b, what, st);
    else run<L, N, false>(b, what, st);
}

}  // namespace

extern "C" int64_t dr_moe_balance_workspace_bytes(const dr_balance* a, int what) {
    if (!valid(a, what)) return -1;
    if (what == DR_BALANCE_BACKWARD) return 0;
    const Split s = split_of(a);
    const long long w = s.groups > 1 ? (long long)a->batch * (s.groups + s.slices) : 0;
    return up256(w * a->experts * 8) + up256(w * 4);
}

extern "C" int dr_moe_balance(const dr_balance* a, int what) {
    if (!valid(a, what)) return DR_EINVAL;
    const long long need = dr_moe_balance_workspace_bytes(a, what);
    auto aligned = [](const void* p, uintptr_t to) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % to == 0; };
    const bool given = what == DR_BALANCE_BACKWARD, grad = given || what & DR_BALANCE_GRAD;
    if (!aligned(a->logits, 4) ||
        (!given && (!aligned(a->ids, a->ids32 ? 4 : 2) || !aligned(a->loss, 4) || !aligned(a->counts, 4))) ||
        ((given || a->kept) && !aligned(a->kept, 4)) || (need > 0 && !aligned(a->workspace, 256)) ||
        a->workspace_bytes < need || (grad && (!aligned(a->dlogits, 4) || a->ld_dlogits < a->width)))
        return DR_EINVAL;
    Bal b{};
    b.a = *a;
    const Split s = split_of(a);
    b.groups = s.groups;
    b.given = given;
    b.vec = aligned(a->logits, 16) && a->ld_logits % 4 == 0;
    b.gvec = grad && aligned(a->dlogits, 16) && a->ld_dlogits % 4 == 0;
    const long long w = (long long)a->batch * b.groups;  // (the slices' sums behind the workgroups')
    b.sums = reinterpret_cast<float2*>(a->workspace);
    b.live = reinterpret_cast<int*>(reinterpret_cast<char*>(a->workspace) + up256((w + s.slices * a->batch) * a->experts * 8));
    b.in = s.slices ? b.sums + w * a->experts : b.sums;
    b.in_live = s.slices ? b.live + w : b.live;
    b.parts = s.slices ? 1 : b.groups;
    const hipStream_t st = reinterpret_cast<hipStream_t>(a->stream);
    if (a->experts <= 64) run_kind<16, 1>(b, what, st);
    else if (a->experts <= 128) run_kind<16, 2>(b, what, st);
    else if (a->experts <= 256) run_kind<16, 4>(b, what, st);
    else if (a->experts <= 512) run_kind<64, 2>(b, what, st);
    else run_kind<64, 4>(b, what, st);
    return hipGetLastError() == hipSuccess ? DR_OK : DR_EHIP;
}
