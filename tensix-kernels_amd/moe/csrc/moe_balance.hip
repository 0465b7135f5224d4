// moe_balance.hip: the router's balance loss, each expert's count and the gradient of the logits on MI355X (gfx950), behind
// dr_moe_balance (include/moe.h). A wavefront holds a row's experts (lane l: l, l + 64, ..), so a row's softmax or sigmoids
// and their sum are a few register operations and one butterfly, and the sums over rows stay in registers until the
// wavefront's rows are done.
//   balance_sum_k   a workgroup's rows: the sum of p and the counts (LDS), written for the workgroup
//   balance_join_k  a batch's workgroups' sums in order: counts, f, loss
//   balance_grad_k  the logits' gradient, p computed again
// What bounds it: the logits read twice and the gradient written once; at a few rows the launches.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe.h"

#pragma clang fp contract(off)

namespace {

constexpr int W = 4;         // wavefronts a workgroup
constexpr int MAXE = 1024;   // experts

struct Bal {
    dr_balance a;
    float* psum;   // [batch][groups][E]
    int* csum;     // [batch][groups][E]
    int* rsum;     // [batch][groups] rows that count
    float* f;      // [batch][E]: E count / counts
    float* per;    // [batch]: 1 / rows that count
    int groups;    // workgroups a batch
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// p of a row, lane's experts l + 64 i (0 past the experts); s (sigmoid): the sigmoids. A row of no expert above -inf has
// p 0 (softmax).
template <int N>
__device__ __forceinline__ void row_p(const dr_balance& a, const float* z, int lane, float (&p)[N], float (&s)[N]) {
    if (a.kind == 0) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = lane + 64 * i;
            p[i] = e < a.experts ? z[e] : -INFINITY;
            top = fmaxf(top, p[i]);
        }
        top = wave_max(top);
        const float base = top == -INFINITY ? 0.f : top;
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            p[i] = expf(p[i] - base);
            total += p[i];
        }
        total = wave_sum(total);
        const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] *= inv, s[i] = 0.f;
    } else {
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = lane + 64 * i;
            s[i] = e < a.experts ? 1.f / (1.f + expf(-z[e])) : 0.f;
            total += s[i];
        }
        total = wave_sum(total);
        const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = s[i] * inv;
    }
}

__device__ __forceinline__ bool counts(const dr_balance& a, long long row) { return a.mask == nullptr || a.mask[row] != 0; }

template <int N>
__global__ __launch_bounds__(64 * W) void balance_sum_k(const Bal b) {
    __shared__ int cnt[MAXE];
    __shared__ float ps[W][64 * N];
    __shared__ int rows[W];
    const dr_balance& a = b.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int g = blockIdx.x % b.groups, batch = blockIdx.x / b.groups;
    for (int e = tid; e < a.experts; e += 64 * W) cnt[e] = 0;
    __syncthreads();
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.f;
    int n = 0;
    for (int r = g * W + wave; r < a.rows; r += b.groups * W) {
        const long long row = (long long)batch * a.rows + r;
        if (!counts(a, row)) continue;
        ++n;
        float p[N], s[N];
        row_p<N>(a, a.logits + row * a.ld_logits, lane, p, s);
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] += p[i];
        if (lane < a.k) {
            const long long at = row * a.ld_ids + lane;
            const uint32_t id = a.ids32 ? reinterpret_cast<const uint32_t*>(a.ids)[at] : reinterpret_cast<const uint16_t*>(a.ids)[at];
            if (id < (uint32_t)a.experts) atomicAdd(&cnt[id], 1);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) ps[wave][lane + 64 * i] = sum[i];
    if (lane == 0) rows[wave] = n;
    __syncthreads();
    const long long at = (long long)blockIdx.x * a.experts;
    for (int e = tid; e < a.experts; e += 64 * W) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += ps[w][e];
        b.psum[at + e] = v;
        b.csum[at + e] = cnt[e];
    }
    if (tid == 0) {
        int v = 0;
        for (int w = 0; w < W; ++w) v += rows[w];
        b.rsum[blockIdx.x] = v;
    }
}

__global__ __launch_bounds__(1024) void balance_join_k(const Bal b) {
    __shared__ float red[16];
    __shared__ int tot[16], live[16];
    const dr_balance& a = b.a;
    const int e = threadIdx.x, lane = e & 63, wave = e >> 6, waves = blockDim.x >> 6;
    const long long at = (long long)blockIdx.x * b.groups;
    float p = 0.f;
    int c = 0, r = 0;
    if (e < a.experts)
        for (int g = 0; g < b.groups; ++g) {
            p += b.psum[(at + g) * a.experts + e];
            c += b.csum[(at + g) * a.experts + e];
        }
    for (int g = e; g < b.groups; g += blockDim.x) r += b.rsum[at + g];
    int cs = c, rs = r;
#pragma unroll
    for (int o = 32; o; o >>= 1) cs += __shfl_xor(cs, o), rs += __shfl_xor(rs, o);
    if (lane == 0) tot[wave] = cs, live[wave] = rs;
    __syncthreads();
    int total = 0, rows = 0;
    for (int w = 0; w < waves; ++w) total += tot[w], rows += live[w];
    const float f = total ? (float)a.experts * ((float)c / (float)total) : 0.f, per = rows ? 1.f / (float)rows : 0.f;
    const float l = wave_sum(f * (p * per));
    if (lane == 0) red[wave] = l;
    __syncthreads();
    if (e < a.experts) {
        a.counts[(long long)blockIdx.x * a.experts + e] = c;
        b.f[(long long)blockIdx.x * a.experts + e] = f;
    }
    if (e == 0) {
        float loss = 0.f;
        for (int w = 0; w < waves; ++w) loss += red[w];
        a.loss[blockIdx.x] = loss;
        b.per[blockIdx.x] = per;
    }
}

template <int N>
__global__ __launch_bounds__(64 * W) void balance_grad_k(const Bal b) {
    const dr_balance& a = b.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int g = blockIdx.x % b.groups, batch = blockIdx.x / b.groups;
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = lane + 64 * i < a.experts ? b.f[(long long)batch * a.experts + lane + 64 * i] : 0.f;
    const float scale = (a.g ? a.g[batch] : 1.f) * b.per[batch];
    for (int r = g * W + wave; r < a.rows; r += b.groups * W) {
        const long long row = (long long)batch * a.rows + r;
        float* d = a.dlogits + row * a.ld_dlogits;
        float p[N], s[N], o[N];
        if (counts(a, row)) {
            row_p<N>(a, a.logits + row * a.ld_logits, lane, p, s);
            float mean = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) mean += p[i] * f[i];
            mean = wave_sum(mean);
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = scale * (a.kind ? p[i] * (1.f - s[i]) : p[i]) * (f[i] - mean);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane + 64 * i < a.experts) d[lane + 64 * i] = o[i];
        for (int e = a.experts + lane; e < a.width; e += 64) d[e] = 0.f;
    }
}

// workgroups a batch: every CU a few, no more than its rows fill
int groups_of(const dr_balance* a) {
    const int fit = (a->rows + W - 1) / W, most = (1024 + a->batch - 1) / a->batch;
    return fit < most ? fit : most;
}

bool valid(const dr_balance* a, int what) {
    return a != nullptr && what >= 1 && what <= 3 && a->batch >= 1 && a->batch <= (1 << 16) && a->rows >= 1 &&
           (long long)a->batch * a->rows < (1ll << 31) && a->experts >= 1 && a->experts <= MAXE && a->k >= 1 && a->k <= 16 &&
           a->width >= a->experts && a->ld_logits >= a->width && a->ld_ids >= a->k && (a->kind == 0 || a->kind == 1);
}

long long up256(long long v) { return (v + 255) & ~255ll; }

template <int N>
void run(const Bal& b, int what, hipStream_t st) {
    const dim3 grid(b.groups * b.a.batch);
    hipLaunchKernelGGL(balance_sum_k<N>, grid, dim3(64 * W), 0, st, b);
    hipLaunchKernelGGL(balance_join_k, dim3(b.a.batch), dim3((b.a.experts + 63) & ~63), 0, st, b);
    if (what & DR_BALANCE_GRAD) hipLaunchKernelGGL(balance_grad_k<N>, grid, dim3(64 * W), 0, st, b);
}

}  // namespace

extern "C" int64_t dr_moe_balance_workspace_bytes(const dr_balance* a, int what) {
    if (!valid(a, what)) return -1;
    const long long w = (long long)a->batch * groups_of(a);
    return 2 * up256(w * a->experts * 4) + up256(w * 4) + up256((long long)a->batch * a->experts * 4) + up256((long long)a->batch * 4);
}

extern "C" int dr_moe_balance(const dr_balance* a, int what) {
    if (!valid(a, what)) return DR_EINVAL;
    auto aligned = [](const void* p, uintptr_t to) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % to == 0; };
    if (!aligned(a->logits, 4) || !aligned(a->ids, a->ids32 ? 4 : 2) || !aligned(a->loss, 4) || !aligned(a->counts, 4) ||
        !aligned(a->workspace, 256) || a->workspace_bytes < dr_moe_balance_workspace_bytes(a, what) ||
        ((what & DR_BALANCE_GRAD) && (!aligned(a->dlogits, 4) || a->ld_dlogits < a->width)))
        return DR_EINVAL;
    Bal b{};
    b.a = *a;
    b.groups = groups_of(a);
    char* ws = reinterpret_cast<char*>(a->workspace);
    const long long w = (long long)a->batch * b.groups;
    b.psum = reinterpret_cast<float*>(ws);
    ws += up256(w * a->experts * 4);
    b.csum = reinterpret_cast<int*>(ws);
    ws += up256(w * a->experts * 4);
    b.rsum = reinterpret_cast<int*>(ws);
    ws += up256(w * 4);
    b.f = reinterpret_cast<float*>(ws);
    ws += up256((long long)a->batch * a->experts * 4);
    b.per = reinterpret_cast<float*>(ws);
    const hipStream_t st = reinterpret_cast<hipStream_t>(a->stream);
    const int n = (a->experts + 63) / 64;
    if (n <= 1) run<1>(b, what, st);
    else if (n <= 2) run<2>(b, what, st);
    else if (n <= 4) run<4>(b, what, st);
    else if (n <= 8) run<8>(b, what, st);
    else run<16>(b, what, st);
    return hipGetLastError() == hipSuccess ? DR_OK : DR_EHIP;
}
