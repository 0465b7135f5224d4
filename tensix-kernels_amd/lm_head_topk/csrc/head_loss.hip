// head_loss.hip: the LM head's losses and their gradients for MI355X (gfx950), behind include/lm_head.h.
//
// Three products carry the work, all of one tiled MFMA kernel (hl_gemm), whose operands lie in memory either along the
// summed dimension or across it (read through the LDS transpose read), so that nothing is transposed in memory:
//   z  [v][n]  = head . x^T      summed over dim;    the softmax's statistics, or dz, are its epilogue
//   dhead [v][d] = dz^T . x      summed over rows;   x and dz across
//   dx [n][d]  = dz . head       summed over v;      head across
// A call is a few launches: the entries (ids checked, the teacher's softmax), the rows that count gathered into a
// contiguous x (rows left out cost nothing and whatever they hold enters no sum), z with each wavefront's maximum and sum
// of a row, their merge into lse and loss; backward, piece by piece of the vocabulary, dz from z computed again, the
// entries' own dz, dhead's rows, dx's sum so far.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dense_reader.h"
#include "lm_head.h"

#pragma clang fp contract(off)

namespace {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4;
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

constexpr int BK = 64;                     // k a step
constexpr uint32_t PAST = 0x80000000u;     // a buffer offset past every record: the load gives zeros
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ uint32_t cvt2(float lo, float hi) {  // to bf16, to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}

__device__ __forceinline__ f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The wavefront's LDS reads done and all but its newest VM loads landed, then the workgroup's barrier.
template <int VM>
__device__ __forceinline__ void step_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((VM & 15) | (7 << 4) | ((VM >> 4) << 14));  // vmcnt(VM) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// --- the tiled product ------------------------------------------------------------------------------------------------

enum Epi { EPI_STATS, EPI_DZ, EPI_DHEAD, EPI_DX };

struct Gemm {
    const uint16_t *A, *B;  // D[m][n] = sum over k of A[m][k] B[n][k]; an operand lies [rows][k] or (across) [k][rows]
    long long lda, ldb;
    int m, n, k;            // (k: of a [rows][k] operand a multiple of 8)
    int ka;                 // the k rows that an A across has (past them zeros)
    const int* live;        // the rows that count: n of z and dx, k of dhead
    int tm, tn, splits, steps;  // tiles; K splits of `steps` steps each
    // z's epilogues
    float sc;               // z to the exponent of 2: log2(e) / T
    int v0;                 // z's row 0 is the vocabulary's v0
    const int* idx;         // row that counts -> row, or NULL: itself
    const float* lse;       // [rows]
    const float* gs;        // [rows that count] g over the largest
    f32x2* part;            // [m / TM][n] maximum and sum
    long long ld_part;
    const int* ids;         // [rows][1 << kp] entries, -1 none
    int kp, kn;
    float* zt;              // [rows][kn]
    // outputs
    uint16_t* out;          // dz [n][ld_out], dhead [n = v][ld_out]
    float* acc;             // dx sums [splits][n][ld_out]
    long long ld_out, acc_stride;
    int add;                // dx: onto the sums so far
    const float* scale;     // dhead: the factor taken out of dz
};

// One operand's tile of ROWS x BK values in LDS: 16-byte chunks, laid out so that neither the loads straight from memory
// (64 chunks in a row a wavefront) nor the fragments' reads meet in a bank.
template <int ROWS, bool T, int NT>
struct Tile {
    static constexpr int N = ROWS * 8 / NT;  // chunks a lane loads
    uint32_t off[N];

    // row r's chunk c (8 k) at 8 r + (c ^ (r / 2 % 8)); across: k's chunk c (8 rows), in pairs (32 bytes) shifted by k
    static __device__ __forceinline__ int turn(int k) { return ROWS >= 128 ? 2 * (k & 3) : ROWS == 64 ? 2 * ((k >> 1) & 1) : 0; }

    __device__ __forceinline__ void init(int tid, long long ld, int left) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int s = i * NT + tid;
            if constexpr (T) {
                constexpr int C = ROWS / 8;
                const int k = s / C, c = s % C, src = ((((c >> 1) ^ turn(k))) << 1) | (c & 1);
                off[i] = 8 * src < left ? (uint32_t)(k * (uint32_t)ld * 2u) + 16u * src : PAST;
            } else {
                const int r = s >> 3, c = (s & 7) ^ ((r >> 1) & 7);
                off[i] = (uint32_t)(r * (uint32_t)ld * 2u) + 16u * c;
            }
        }
    }
    // base: the tile's first value of this step; rows: its rows (across: the step's k) in memory; left: its k (across:
    // its rows) in memory
    __device__ __forceinline__ void load(const uint16_t* base, long long ld, int rows, int left, uint4* lds, int tid) const {
        const long long bytes = rows > 0 && left > 0 ? ((long long)(rows - 1) * ld + ((left + 7) & ~7)) * 2 : 0;
        const __amdgpu_buffer_rsrc_t r =
            __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)(bytes < 0x7FFFFFFF ? bytes : 0x7FFFFFFF), 0x00020000);
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint32_t o = off[i];
            if constexpr (!T) {
                if (left < BK) {  // (the last step of a ragged k)
                    const int s = i * NT + tid, rr = s >> 3, c = (s & 7) ^ ((rr >> 1) & 7);
                    if (8 * c >= left) o = PAST;
                }
            }
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(lds + i * NT + 64 * wave), 16, o, 0, 0, 0);
        }
    }
    // lane's 8 values of row r0 + lane % 32, k = 16 u + 8 (lane / 32) ..
    static __device__ __forceinline__ uint4 frag(const uint4* lds, int r0, int u, int lane) {
        if constexpr (T) {
            constexpr int C = ROWS / 8;
            const int h = lane >> 5, half = (lane >> 4) & 1, i = lane & 15;
            uint2 q[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int k = 16 * u + 8 * h + 4 * p + (i >> 2);
                const int pair = ((r0 >> 4) + half) ^ turn(k);
                const uint16_t* at = reinterpret_cast<const uint16_t*>(lds + k * C + 2 * pair) + 4 * (i & 3);
                q[p] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at));
            }
            return make_uint4(q[0].x, q[0].y, q[1].x, q[1].y);
        } else {
            const int r = lane & 31, h = lane >> 5;
            return lds[(r0 + r) * 8 + ((2 * u + h) ^ ((r >> 1) & 7))];
        }
    }
};

// workgroups go to the XCDs in turn; each XCD takes a run of tiles, in groups of GM row tiles by all column tiles, so that
// what runs at once on an XCD shares rows and columns in its L2
__device__ __forceinline__ void tile_of(const Gemm& a, int& mt, int& nt, int& split) {
    const int total = a.tm * a.tn * a.splits, xcd = blockIdx.x & 7;
    int w = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
    split = w / (a.tm * a.tn);
    w -= split * a.tm * a.tn;
    constexpr int GM = 4;
    const int g = w / (GM * a.tn), first = g * GM, gm = min(GM, a.tm - first);
    w -= g * GM * a.tn;
    nt = w / gm;
    mt = first + w - nt * gm;
}

template <int BM, int BN, int WM, int WN, bool AT, bool BT, int EPI>
__global__ __launch_bounds__(64 * WM * WN) void hl_gemm(const Gemm a) {
    constexpr int NT = 64 * WM * WN, TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
    constexpr int CH = (BM + BN) * 8;  // chunks a stage
    __shared__ uint4 s0[CH], s1[CH];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    int mt, nt, split;
    tile_of(a, mt, nt, split);
    const int m0 = mt * BM, n0 = nt * BN;
    const int live = a.live ? *a.live : (EPI == EPI_DHEAD ? a.k : a.n);
    const int n_end = EPI == EPI_DHEAD ? a.n : live, k_end = EPI == EPI_DHEAD ? live : a.k;
    const int ka = EPI == EPI_DHEAD ? live : a.ka;
    if (n0 >= n_end) return;
    const int step0 = split * a.steps, steps = min(a.steps, (k_end + BK - 1) / BK - step0);

    Tile<BM, AT, NT> ta;
    Tile<BN, BT, NT> tb;
    ta.init(tid, a.lda, a.m - m0);
    tb.init(tid, a.ldb, n_end - n0);
    auto load = [&](int s, uint4* b) {
        const long long k0 = (long long)(step0 + s) * BK;
        if constexpr (AT) ta.load(a.A + k0 * a.lda + m0, a.lda, min(BK, ka - (int)k0), a.m - m0, b, tid);
        else ta.load(a.A + m0 * a.lda + k0, a.lda, min(BM, a.m - m0), k_end - (int)k0, b, tid);
        if constexpr (BT) tb.load(a.B + k0 * a.ldb + n0, a.ldb, min(BK, k_end - (int)k0), n_end - n0, b + BM * 8, tid);
        else tb.load(a.B + n0 * a.ldb + k0, a.ldb, min(BN, n_end - n0), k_end - (int)k0, b + BM * 8, tid);
    };
    f32x16 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    auto sum = [&](const uint4* b) {
#pragma unroll
        for (int u = 0; u < BK / 16; ++u) {
            uint4 fa[MI], fb[NI];
#pragma unroll
            for (int j = 0; j < NI; ++j) fb[j] = Tile<BN, BT, NT>::frag(b + BM * 8, wn * TN + 32 * j, u, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i) fa[i] = Tile<BM, AT, NT>::frag(b, wm * TM + 32 * i, u, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = mfma32(fa[i], fb[j], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);  // (one u's fragments at a time: the registers hold no more)
        }
    };
    // (in pairs of steps: one past the last is zeros, as are the loads past the end into a stage that nothing reads. A
    // last step of its own behind a branch would have the compiler copy every accumulator.)
    if (steps > 0) load(0, s0);
    for (int s = 0; s < steps; s += 2) {
        step_barrier<0>();
        load(s + 1, s1);
        sum(s0);
        step_barrier<0>();
        load(s + 2, s0);
        sum(s1);
    }
    step_barrier<0>();  // (the last loads landed: they write this workgroup's LDS)

    // lane: columns n = n0 + wn TN + 32 j + lane % 32, rows m0 + wm TM + 32 i + 8 g + 4 (lane / 32) + 0 .. 3 in words 4 g ..
    const int r = lane & 31, h = lane >> 5;
    const int mw = m0 + wm * TM;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        const int n = n0 + wn * TN + 32 * j + r;
        if constexpr (EPI == EPI_STATS) {
            const int left = a.m - mw;  // vocabulary rows of this wavefront
            if (left < TM) {
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        acc[i][j][e] = 32 * i + 8 * (e >> 2) + 4 * h + (e & 3) < left ? acc[i][j][e] : -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, acc[i][j][e]);
            top = fmaxf(top, __shfl_xor(top, 32));
            const float base = top == -INFINITY ? 0.f : top * a.sc;
            float total = 0.f;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) total += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], a.sc, -base));
            total += __shfl_xor(total, 32);
            if (h == 0 && n < n_end) a.part[(long long)(mt * WM + wm) * a.ld_part + n] = f32x2{top == -INFINITY ? top : base, total};
            // the entries that lie here: the wavefront's sums of these 32 rows through its own LDS
            f32x4* mine = reinterpret_cast<f32x4*>(wave < (WM * WN + 1) / 2 ? s0 : s1) + (wave % ((WM * WN + 1) / 2)) * 8 * TM;
            static_assert((WM * WN + 1) / 2 * 8 * TM <= CH, "a wavefront's sums of 32 rows fit its part of a stage");
            const int count = 32 << a.kp, nb = n0 + wn * TN + 32 * j;
            auto entry = [&](int e, long long& row) {  // its row of mw .., or -1
                const int nn = nb + (e >> a.kp);
                if (e >= count || nn >= n_end) return -1;
                row = a.idx ? a.idx[nn] : nn;
                const int d = a.ids[(row << a.kp) + (e & ((1 << a.kp) - 1))] - mw;
                return (unsigned)d < (unsigned)min(TM, left) ? d : -1;
            };
            long long row = 0;
            bool any = a.kp >= 4;
            for (int e = lane; !any && e - lane < count; e += 64) any = __ballot(entry(e, row) >= 0) != 0;
            if (any) {
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        mine[r * (TM / 4) + ((8 * i + 2 * g + h) ^ (r & 7))] =
                            f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                __builtin_amdgcn_wave_barrier();
                for (int e = lane; e - lane < count; e += 64) {
                    const int d = entry(e, row), t = e >> a.kp;
                    if (d >= 0) a.zt[row * a.kn + (e & ((1 << a.kp) - 1))] = mine[t * (TM / 4) + ((d >> 2) ^ (t & 7))][d & 3];
                }
                __builtin_amdgcn_wave_barrier();
            }
        } else if constexpr (EPI == EPI_DZ) {
            if (n >= n_end) continue;
            const float l2 = a.lse[a.idx ? a.idx[n] : n] * LOG2E, gs = a.gs[n];
            const int left = a.m - mw;
            uint16_t* o = a.out + n * a.ld_out + mw;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int v = 32 * i + 8 * g + 4 * h;
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        p[e] = v + e < left ? gs * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][4 * g + e], a.sc, -l2)) : 0.f;
                    *reinterpret_cast<uint2*>(o + v) = make_uint2(cvt2(p[0], p[1]), cvt2(p[2], p[3]));
                }
        } else if constexpr (EPI == EPI_DHEAD) {
            if (n >= n_end) continue;
            const float s = *a.scale;
            uint16_t* o = a.out + n * a.ld_out + mw;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * i + 8 * g + 4 * h;
                    if (mw + d < a.m)
                        *reinterpret_cast<uint2*>(o + d) =
                            make_uint2(cvt2(acc[i][j][4 * g] * s, acc[i][j][4 * g + 1] * s),
                                       cvt2(acc[i][j][4 * g + 2] * s, acc[i][j][4 * g + 3] * s));
                }
        } else {
            if (n >= n_end) continue;
            float* o = a.acc + split * a.acc_stride + n * a.ld_out + mw;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * i + 8 * g + 4 * h;
                    if (mw + d < a.m) {
                        f32x4 v = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                        f32x4* p = reinterpret_cast<f32x4*>(o + d);
                        if (a.add) v += *p;
                        *p = v;
                    }
                }
        }
    }
}

// --- entries, rows that count, merges -----------------------------------------------------------------------------------

struct Prep {
    dr_head_loss a;
    int kp;        // log2 of the entries' stride
    int* ids;      // [rows][1 << kp], -1: not held
    float* q;      // [rows][1 << kp] (a teacher's)
    float* ent;    // [rows] sum q log q (a teacher's)
    int* idx;      // [rows] row that counts -> row
    int* pos;      // [rows] row -> row that counts, -1: left out
    int* live;     // rows that count
    float* scale;  // the largest |g| of them, over T
    float* gs;     // [rows that count]
    uint16_t* xc;  // [rows that count][dim], or NULL: x where it lies
    int fwd, back;
};

__device__ __forceinline__ int entry_id(const dr_head_loss& a, int row, int j) {
    const long long at = (long long)row * a.ld_ids + j;
    const long long id = a.ids64 ? reinterpret_cast<const long long*>(a.ids)[at] : reinterpret_cast<const int*>(a.ids)[at];
    return id >= 0 && id < a.valid ? (int)id : -1;
}

// the entries of a row: 1 << kp lanes a row
__global__ __launch_bounds__(256) void hl_entries(const Prep p) {
    const int e = blockIdx.x * 256 + threadIdx.x, row = e >> p.kp, w = 1 << p.kp, j = e & (w - 1);
    const bool in = row < p.a.rows && j < p.a.k;
    int id = in ? entry_id(p.a, row, j) : -1;
    if (p.a.vals) {
        float v = in ? p.a.vals[(long long)row * p.a.ld_vals + j] / p.a.temperature : -INFINITY;
        if (v == -INFINITY) id = -1;
        if (id < 0) v = -INFINITY;
        float top = v;
        for (int o = w >> 1; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        const float d = id < 0 ? 0.f : v - top;
        const float x = id < 0 ? 0.f : __expf(d);
        float total = x;
        for (int o = w >> 1; o; o >>= 1) total += __shfl_xor(total, o);
        const float q = id < 0 ? 0.f : x / total;
        float ent = q == 0.f ? 0.f : q * (d - __logf(total));
        for (int o = w >> 1; o; o >>= 1) ent += __shfl_xor(ent, o);
        if (row < p.a.rows) {
            p.q[e] = q;
            if (j == 0) p.ent[row] = ent;
        }
    }
    if (row < p.a.rows) {
        p.ids[e] = id;
        if (in && id < 0 && p.fwd) p.a.logits[(long long)row * p.a.k + j] = 0.f;
        const unsigned long long held = __ballot(id >= 0);
        const int lane = threadIdx.x & 63;
        const unsigned long long mine = w == 64 ? held : (held >> (lane & ~(w - 1))) & ((1ull << w) - 1);
        if (j == 0) p.pos[row] = mine ? 0 : -1;
    }
}

// the rows that count, in order: each workgroup counts those before its own
__global__ __launch_bounds__(256) void hl_count(const Prep p) {
    __shared__ int part[256];
    __shared__ float gpart[256];
    const int tid = threadIdx.x, per = (p.a.rows + 255) / 256;
    const int r0 = min(tid * per, p.a.rows), r1 = min(r0 + per, p.a.rows);
    int c = 0;
    float gm = 0.f;
    for (int r = r0; r < r1; ++r)
        if (p.pos[r] >= 0) {
            ++c;
            const float g = p.a.g ? fabsf(p.a.g[r]) : 1.f;
            gm = fmaxf(gm, g);
        }
    part[tid] = c;
    gpart[tid] = gm;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < tid; ++i) before += part[i];
    float top = 0.f;
    for (int i = 0; i < 256; ++i) top = fmaxf(top, gpart[i]);
    if (tid == 255) {
        *p.live = before + c;
        *p.scale = top / p.a.temperature;
    }
    const float inv = top > 0.f ? 1.f / top : 0.f;
    for (int r = r0; r < r1; ++r)
        if (p.pos[r] >= 0) {
            p.pos[r] = before;
            p.idx[before] = r;
            if (p.back) p.gs[before] = (p.a.g ? p.a.g[r] : 1.f) == top ? 1.f : (p.a.g ? p.a.g[r] : 1.f) * inv;
            ++before;
        }
}

__global__ __launch_bounds__(256) void hl_gather(const Prep p) {
    const int n = blockIdx.x;
    if (n >= *p.live) return;
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.a.x) + p.idx[n] * p.a.ldx);
    uint4* dst = reinterpret_cast<uint4*>(p.xc + (long long)n * p.a.dim);
    for (int c = threadIdx.x; c < p.a.dim / 8; c += 256) dst[c] = src[c];
}

struct Merge {
    const f32x2* part;
    long long ld;
    int parts, rows, k, kp, gather;
    const int *pos;
    const float *q, *ent;
    float inv_t;
    float *loss, *lse;
    const float* zt;
};

// TB rows a workgroup, 256 / TB slices of the parts each
template <int TB>
__global__ __launch_bounds__(256) void hl_merge(const Merge p) {
    __shared__ float ms[256], ss[256];
    const int tid = threadIdx.x, t = tid % TB, sl = tid / TB, row = blockIdx.x * TB + t;
    int n = row < p.rows ? p.pos[row] : -1;
    if (n >= 0 && !p.gather) n = row;
    float m = -INFINITY, s = 0.f;
    if (n >= 0)
        for (int i = sl; i < p.parts; i += 256 / TB) {
            const f32x2 v = p.part[i * p.ld + n];
            if (v[0] == -INFINITY) continue;
            const float top = fmaxf(m, v[0]);
            if (top == m) s += v[1] * __builtin_amdgcn_exp2f(v[0] - top);
            else s = s * __builtin_amdgcn_exp2f(m - top) + v[1], m = top;
        }
    ms[tid] = m;
    ss[tid] = s;
    __syncthreads();
    if (sl) return;
    for (int i = 1; i < 256 / TB; ++i) {
        const float v = ms[i * TB + t], w = ss[i * TB + t];
        const float top = fmaxf(m, v);
        if (top == -INFINITY) continue;
        s = s * __builtin_amdgcn_exp2f(m - top) + w * __builtin_amdgcn_exp2f(v - top);
        m = top;
    }
    if (row >= p.rows) return;
    float lse = 0.f, loss = 0.f;
    if (n >= 0) {
        lse = (m + __builtin_amdgcn_logf(s)) * LN2;
        if (p.q) {
            float c = 0.f;
            for (int j = 0; j < p.k; ++j) {
                const float q = p.q[((long long)row << p.kp) + j];
                if (q != 0.f) c += q * (lse - p.zt[(long long)row * p.k + j] * p.inv_t);
            }
            loss = p.ent[row] + c;
        } else {
            loss = lse - p.zt[row];
        }
    }
    p.lse[row] = lse;
    p.loss[row] = loss;
}

struct Fix {
    const int *live, *idx, *ids;
    const float *q, *lse, *zt, *gs;
    int k, kp, v0, v1;
    float sc;
    uint16_t* dz;
    long long ld;
};

// the entries' own dz: p less the entries' q of that id
__global__ __launch_bounds__(256) void hl_fix(const Fix p) {
    const int e = blockIdx.x * 256 + threadIdx.x, n = e >> p.kp, w = 1 << p.kp, j = e & (w - 1);
    const bool in = n < *p.live;
    const long long row = in ? p.idx[n] : 0;
    const int id = in ? p.ids[(row << p.kp) + j] : -1;
    const float q = id < 0 ? 0.f : p.q ? p.q[(row << p.kp) + j] : 1.f;
    float all = 0.f;
    for (int i = 0; i < w; ++i) {
        const int oid = __shfl(id, i, w);
        const float oq = __shfl(q, i, w);
        if (oid == id) all += oq;
    }
    if (id < p.v0 || id >= p.v1) return;
    const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(p.zt[row * p.k + j], p.sc, -p.lse[row] * LOG2E));
    p.dz[n * p.ld + (id - p.v0)] = (uint16_t)cvt2(p.gs[n] * (pr - all), 0.f);
}

struct Finish {
    const float* acc;
    long long stride, ld;
    int splits, rows, dim;
    const int* pos;
    const float* scale;
    uint16_t* dx;
    long long ld_dx;
};

__global__ __launch_bounds__(256) void hl_dx(const Finish p) {
    const int row = blockIdx.x, n = p.pos[row];
    const float s = *p.scale;
    for (int d = 4 * threadIdx.x; d < p.dim; d += 1024) {
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
        if (n >= 0)
            for (int i = 0; i < p.splits; ++i) v += *reinterpret_cast<const f32x4*>(p.acc + i * p.stride + n * p.ld + d);
        *reinterpret_cast<uint2*>(p.dx + row * p.ld_dx + d) = make_uint2(cvt2(v[0] * s, v[1] * s), cvt2(v[2] * s, v[3] * s));
    }
}

__global__ __launch_bounds__(256) void hl_zero_rows(uint16_t* p, long long ld, int dim) {
    for (int d = 4 * threadIdx.x; d < dim; d += 1024)
        *reinterpret_cast<uint2*>(p + blockIdx.x * ld + d) = make_uint2(0u, 0u);
}

// --- the plan ----------------------------------------------------------------------------------------------------------

constexpr long long DZ_BYTES = 1ll << 30;  // dz a piece at most

long long up(long long v, long long to) { return (v + to - 1) / to * to; }

struct Plan {
    int kp, bn, parts, piece, splits;
    bool gather;
    long long ids, q, ent, idx, pos, live, gs, xc, part, dz, acc, bytes;
};

int log2_up(int k) {
    int p = 0;
    while ((1 << p) < k) ++p;
    return p;
}

bool plan_of(const dr_head_loss* a, int what, Plan& p) {
    if (a == nullptr || what < 1 || what > 3 || a->rows < 1 || a->rows > (1 << 20) || a->dim < 8 || a->dim % 8 ||
        a->dim > (1 << 17) || a->vocab < 1 || a->vocab > (1 << 28) || a->valid < 1 || a->valid > a->vocab || a->k < 1 ||
        a->k > DR_LOSS_MAX_K || (a->vals == nullptr && (a->k != 1 || a->temperature != 1.f)) ||
        !(a->temperature > 0.f && a->temperature < INFINITY) || a->ldx < a->dim || a->ldx % 8 || a->ld_head < a->dim ||
        a->ld_head % 8 || a->ldx > (1 << 21) || a->ld_head > (1 << 21) || a->ld_ids < a->k || (a->vals && a->ld_vals < a->k))
        return false;
    const bool back = what & DR_LOSS_BACKWARD;
    const long long n = a->rows, np = up(n, 64);
    p.kp = log2_up(a->k);
    p.bn = n <= 64 ? 64 : n <= 128 ? 128 : 256;
    p.parts = (int)(up(a->valid, 256) / 128);
    p.gather = back || n > 64;
    long long at = 0;
    auto take = [&](long long bytes) {
        const long long here = at;
        at += up(bytes, 256);
        return here;
    };
    p.ids = take(n * 4 << p.kp);
    p.q = take(a->vals ? n * 4 << p.kp : 0);
    p.ent = take(a->vals ? n * 4 : 0);
    p.idx = take(n * 4);
    p.pos = take(n * 4);
    p.live = take(8);
    p.gs = take(back ? n * 4 : 0);
    p.xc = take(p.gather ? n * a->dim * 2 : 0);
    p.part = take(what & DR_LOSS_FORWARD ? p.parts * np * 8 : 0);
    p.piece = 0, p.splits = 1, p.dz = p.acc = 0;
    if (back) {
        // the vocabulary in equal pieces of a multiple of 256
        const long long tiles = up(a->valid, 256) / 256, fit = DZ_BYTES / (n * 512);
        const long long pieces = (tiles + (fit > 1 ? fit : 1) - 1) / (fit > 1 ? fit : 1);
        p.piece = (int)((tiles + pieces - 1) / pieces) * 256;
        p.dz = take(n * p.piece * 2);
        if (a->dx) {
            const long long t = up(n, p.bn) / p.bn * (up(a->dim, 256) / 256), most = p.piece / BK;
            long long s = (512 + t - 1) / t;
            if (s > most / 4) s = most / 4 > 0 ? most / 4 : 1;
            p.splits = (int)s;
            p.acc = take(s * n * a->dim * 4);
        }
    }
    p.bytes = at;
    return true;
}

template <int BM, int BN, int WM, int WN, bool AT, bool BT, int EPI>
void launch(Gemm g, hipStream_t st) {
    g.tm = (g.m + BM - 1) / BM;
    g.tn = (g.n + BN - 1) / BN;
    hipLaunchKernelGGL((hl_gemm<BM, BN, WM, WN, AT, BT, EPI>), dim3(g.tm * g.tn * g.splits), dim3(64 * WM * WN), 0, st, g);
}

template <bool AT, int EPI>
void launch_rows(const Gemm& g, int bn, hipStream_t st) {  // (the columns are rows of x)
    if (bn == 64) launch<256, 64, 2, 2, AT, false, EPI>(g, st);
    else if (bn == 128) launch<256, 128, 2, 2, AT, false, EPI>(g, st);
    else launch<256, 256, 2, 4, AT, false, EPI>(g, st);
}

}  // namespace

extern "C" int64_t dr_head_loss_workspace_bytes(const dr_head_loss* a, int what) {
    Plan p;
    return plan_of(a, what, p) ? p.bytes : -1;
}

extern "C" int dr_head_loss_run(const dr_head_loss* a, int what) {
    Plan P;
    if (!plan_of(a, what, P)) return DR_EINVAL;
    auto aligned = [](const void* p, uintptr_t to) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % to == 0; };
    const bool fwd = what & DR_LOSS_FORWARD, back = what & DR_LOSS_BACKWARD;
    if (!aligned(a->x, 16) || !aligned(a->head, 16) || !aligned(a->ids, a->ids64 ? 8 : 4) || !aligned(a->lse, 4) ||
        !aligned(a->logits, 4) || (fwd && !aligned(a->loss, 4)) || !aligned(a->workspace, 256) || a->workspace_bytes < P.bytes ||
        (back && a->dx && (!aligned(a->dx, 8) || a->ld_dx < a->dim || a->ld_dx % 4)) ||
        (back && a->dhead && (!aligned(a->dhead, 8) || a->ld_dhead < a->dim || a->ld_dhead % 4)))
        return DR_EINVAL;
    if (back && !fwd && !a->dx && !a->dhead) return DR_OK;
    const hipStream_t st = reinterpret_cast<hipStream_t>(a->stream);
    char* ws = reinterpret_cast<char*>(a->workspace);
    const int n = a->rows, kn = a->k;
    Prep p{};
    p.a = *a;
    p.kp = P.kp;
    p.ids = reinterpret_cast<int*>(ws + P.ids);
    p.q = a->vals ? reinterpret_cast<float*>(ws + P.q) : nullptr;
    p.ent = reinterpret_cast<float*>(ws + P.ent);
    p.idx = reinterpret_cast<int*>(ws + P.idx);
    p.pos = reinterpret_cast<int*>(ws + P.pos);
    p.live = reinterpret_cast<int*>(ws + P.live);
    p.scale = reinterpret_cast<float*>(ws + P.live + 4);
    p.gs = reinterpret_cast<float*>(ws + P.gs);
    p.xc = reinterpret_cast<uint16_t*>(ws + P.xc);
    p.fwd = fwd, p.back = back;
    const int eblocks = (int)((((long long)n << P.kp) + 255) / 256);
    hipLaunchKernelGGL(hl_entries, dim3(eblocks), dim3(256), 0, st, p);
    if (P.gather) {
        hipLaunchKernelGGL(hl_count, dim3(1), dim3(256), 0, st, p);
        hipLaunchKernelGGL(hl_gather, dim3(n), dim3(256), 0, st, p);
    }

    Gemm z{};  // z of a range of the vocabulary
    z.A = reinterpret_cast<const uint16_t*>(a->head);
    z.lda = a->ld_head;
    z.B = P.gather ? p.xc : reinterpret_cast<const uint16_t*>(a->x);
    z.ldb = P.gather ? a->dim : a->ldx;
    z.n = n, z.k = z.ka = a->dim;
    z.live = P.gather ? p.live : nullptr;
    z.idx = P.gather ? p.idx : nullptr;
    z.splits = 1, z.steps = (a->dim + BK - 1) / BK;
    z.sc = LOG2E / a->temperature;
    z.ids = p.ids, z.kp = P.kp, z.kn = kn;
    z.lse = a->lse, z.gs = p.gs;
    if (fwd) {
        Gemm s = z;
        s.m = a->valid;
        s.part = reinterpret_cast<f32x2*>(ws + P.part);
        s.ld_part = up(n, 64);
        s.zt = a->logits;
        launch_rows<false, EPI_STATS>(s, P.bn, st);
        Merge m{s.part, s.ld_part, P.parts, n, kn, P.kp, P.gather, p.pos, p.q, p.ent, 1.f / a->temperature, a->loss, a->lse, a->logits};
        if (n <= 256) hipLaunchKernelGGL(hl_merge<1>, dim3(n), dim3(256), 0, st, m);
        else hipLaunchKernelGGL(hl_merge<32>, dim3((n + 31) / 32), dim3(256), 0, st, m);
    }
    if (back && (a->dx || a->dhead)) {
        uint16_t* dz = reinterpret_cast<uint16_t*>(ws + P.dz);
        for (int v0 = 0; v0 < a->valid; v0 += P.piece) {
            const int vn = a->valid - v0 < P.piece ? a->valid - v0 : P.piece, vp = (int)up(vn, 256);
            Gemm s = z;
            s.A += (long long)v0 * a->ld_head;
            s.m = vn;
            s.out = dz;
            s.ld_out = P.piece;
            launch_rows<false, EPI_DZ>(s, P.bn, st);
            Fix f{p.live, p.idx, p.ids, p.q, a->lse, a->logits, p.gs, kn, P.kp, v0, v0 + vn, z.sc, dz, P.piece};
            hipLaunchKernelGGL(hl_fix, dim3(eblocks), dim3(256), 0, st, f);
            if (a->dhead) {
                Gemm w{};
                w.A = p.xc, w.lda = a->dim;
                w.B = dz, w.ldb = P.piece;
                w.m = a->dim, w.n = vn, w.k = n, w.live = p.live;
                w.splits = 1, w.steps = (n + BK - 1) / BK;
                w.out = reinterpret_cast<uint16_t*>(a->dhead) + (long long)v0 * a->ld_dhead;
                w.ld_out = a->ld_dhead;
                w.scale = p.scale;
                launch<256, 256, 2, 4, true, true, EPI_DHEAD>(w, st);
            }
            if (a->dx) {
                Gemm d{};
                d.A = z.A + (long long)v0 * a->ld_head, d.lda = a->ld_head;
                d.B = dz, d.ldb = P.piece;
                d.m = a->dim, d.n = n, d.k = (int)up(vn, 8), d.ka = vn, d.live = p.live;
                d.splits = P.splits;
                d.steps = (int)up((vp / BK + P.splits - 1) / P.splits, 2);  // (steps run in pairs)
                d.acc = reinterpret_cast<float*>(ws + P.acc);
                d.acc_stride = (long long)n * a->dim;
                d.ld_out = a->dim;
                d.add = v0 > 0;
                launch_rows<true, EPI_DX>(d, P.bn, st);
            }
        }
        if (a->dx) {
            Finish f{reinterpret_cast<const float*>(ws + P.acc), (long long)n * a->dim, a->dim, P.splits, n, a->dim, p.pos, p.scale,
                     reinterpret_cast<uint16_t*>(a->dx), a->ld_dx};
            hipLaunchKernelGGL(hl_dx, dim3(n), dim3(256), 0, st, f);
        }
        if (a->dhead && a->vocab > a->valid)
            hipLaunchKernelGGL(hl_zero_rows, dim3(a->vocab - a->valid), dim3(256), 0, st,
                               reinterpret_cast<uint16_t*>(a->dhead) + (long long)a->valid * a->ld_dhead, a->ld_dhead, a->dim);
    }
    return hipGetLastError() == hipSuccess ? DR_OK : DR_EHIP;
}
