// gated.hip: the gated feed-forward block in training and its gradients for MI355X (gfx950), behind include/gated.h.
//
//   g = x . gate^T, u = x . up^T, h = a(g) u              one product of gate's and up's rows together; h is its epilogue
//   du = dh a(g), dg = dh u a'(g)                         value by value, from what the forward call kept; or the same product
//                                                         again with this as its epilogue
//   dgate = dg^T . x, dup = du^T . x                      one product of dg's and du's columns together, summed over rows
//   dx = dg . gate + du . up                              one product, summed over gate's and then up's outputs
//
// All are of one tiled MFMA kernel (gt_gemm) whose operands are read as they lie, along the summed dimension or across it
// (mfma_tile.h). In the first every 32 rows of a tile are 16 of gate and the same 16 of up, so that two neighbouring fragments of 16 x
// 16 sums have g and u of an output in one lane. dg, du and what is kept lie in panels of 256 outputs ([output / 256][row][256]), which
// the products that read them take in contiguous blocks. No atomics but counters: every sum has one order.
//
// What bounds them. 8192 rows x 4096 x 14336, a step in 4.50 to 4.59 ms (one machine and another): 1500 us for h and what is kept (1283
// TFLOP/s; h alone 1395), 216 for dg and du (1.41 GB, 6.5 TB/s), 1390 for both weights' gradients (1384), 1480 for dx (1300): the matrix
// cores, busy 65 to 70 % of the clocks, and the power that random values draw, which holds the clock at 1.6 to 1.8 GHz (a large
// library product of the three layouts, the card as warm: 1220, 1580, 1370 us). 32 rows x 4096 x 14336: the weights' 235 MB in
// 38.4 us, 6.1 TB/s. A few rows by a small layer: each launch's start, its first loads and the way of a few sums (48 x 1024 x
// 4096: 3 launches of 10 to 13 us for a step).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <initializer_list>

#include "dense_reader.h"
#include "gated.h"
#include "mfma_tile.h"

#pragma clang fp contract(off)

namespace {

// --- the activation -----------------------------------------------------------------------------------------------------

// 1 / (1 + exp(-v))
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * v)); }

// a(g) and a'(g). gelu's tanh form is g p with p = sigmoid(c (g + 0.044715 g^3)), c = 2 sqrt(2 / pi). (Where p is 0 or 1 its slope
// is 0, and what that is multiplied by stays finite.)
template <bool GELU>
__device__ __forceinline__ void act_of(float g, float& a, float& slope) {
    constexpr float C = 1.5957691216057308f, C3 = 0.044715f * C;
    if constexpr (GELU) {
        const float p = sigmoid(g * __builtin_fmaf(C3, g * g, C));
        const float t = fminf(fmaxf(g, -16.f), 16.f);
        a = g * p;
        slope = __builtin_fmaf(t * (p * (1.f - p)), __builtin_fmaf(3.f * C3, t * t, C), p);
    } else {
        const float p = sigmoid(g);
        a = g * p;
        slope = __builtin_fmaf(a, 1.f - p, p);
    }
}

// What a forward call keeps of an output: g and u, in 24 bits each (float32's without the last 8 of the mantissa): the upper 16 of
// g's and of u's, then g's lower 8 over u's. (In bf16 alone a step's gradients would be off by 2.9e-3 of their norm instead of
// 2.35e-3, of which the rounding of dg and du and their own make 1.7e-3 each. a(g) and a'(g) u in their place would cost the product's
// epilogue, where nothing else runs, what the pass that reads them has time for.)
__device__ __forceinline__ uint32_t bytes(uint32_t hi, uint32_t lo, uint32_t pick) { return __builtin_amdgcn_perm(hi, lo, pick); }
__device__ __forceinline__ uint2 upper(const uint32_t (&v)[4]) {
    return make_uint2(bytes(v[1], v[0], 0x07060302u), bytes(v[3], v[2], 0x07060302u));
}
__device__ __forceinline__ uint2 lower(const uint32_t (&g)[4], const uint32_t (&u)[4]) {
    return make_uint2(bytes(g[0], u[0], 0x0C0C0501u) | bytes(g[1], u[1], 0x05010C0Cu),
                      bytes(g[2], u[2], 0x0C0C0501u) | bytes(g[3], u[3], 0x05010C0Cu));
}
// value e of 4, from its upper part and the lower ones of both
__device__ __forceinline__ float kept_g(uint2 hi, uint2 lo, int e) {
    return __uint_as_float(bytes(e < 2 ? hi.x : hi.y, e < 2 ? lo.x : lo.y, e & 1 ? 0x0706030Cu : 0x0504010Cu));
}
__device__ __forceinline__ float kept_u(uint2 hi, uint2 lo, int e) {
    return __uint_as_float(bytes(e < 2 ? hi.x : hi.y, e < 2 ? lo.x : lo.y, e & 1 ? 0x0706020Cu : 0x0504000Cu));
}
__device__ __forceinline__ float bf16_of(uint2 v, int e) {
    const uint32_t w = e < 2 ? v.x : v.y;
    return __uint_as_float(e & 1 ? w & 0xFFFF0000u : w << 16);
}

// (the K loop's arrays are seen as what they are only where everything is in one function)
#define INLINE __attribute__((always_inline))

// --- the tiled product --------------------------------------------------------------------------------------------------

// ACT, KEEP, AGAIN: D[2 width][rows], A gate and up, B x; DW: D[dim][outputs], A x, B dg and du; DX: D[dim][rows], A gate and up,
// B dg and du. DWF: DW of one step, which makes its dg and du from what was kept for itself (the first row of tiles leaves them in memory).
// DXJ: DX whose splits' sums the last workgroup of a tile adds up.
enum Epi { EPI_ACT, EPI_KEEP, EPI_AGAIN, EPI_DW, EPI_DWF, EPI_DX, EPI_DXJ };

struct Prod {
    const uint16_t *x, *gate, *up;
    int ldx, ld_gate, ld_up;
    int rows, dim, width;
    int panels;             // of 256 outputs, a side
    long long panel;        // values of one: rows * 256
    int tm, tn;             // tiles
    uint16_t* h;
    long long ld_h;
    uint16_t* kept;         // [3][panels][rows][256]: g's upper parts, u's, the lower ones of both
    const uint16_t* dh;
    long long ld_dh;
    uint16_t* dz;           // dg, then du, each [panels][rows][256]
    int side0;              // DW: the first of the sides that are asked for
    uint16_t *dgate, *dup;
    long long ld_dgate, ld_dup;
    uint16_t* dx;           // or NULL: the sums of each split
    long long ld_dx;
    float* acc;             // [splits][rows][dim]
    int splits;
    int past;               // ACT, KEEP: the outputs pass the caches by
    uint32_t* arrived;      // DXJ: of each tile the splits that are done; AGAIN, DWF: to be cleared for it
    int counters;
};

// The tile of dg or du that a DWF workgroup multiplies by, from dh and what was kept: rows (its k) by BN outputs from c0 on, in the
// places of its operand's loads; to memory too (leave). All loads first: they would wait for each other's values else.
template <typename T, int BN, int NT, bool GELU>
__device__ __forceinline__ void dz_tile(const Prod& a, uint4* to, int tid, int side, int c0, bool leave) {
    constexpr int C = BN / 8;
    const long long one = a.panels * a.panel, panel = (long long)(c0 >> 8) * a.panel + (c0 & 255);
    uint4 dh[T::N], g[T::N], u[T::N], lo[T::N];
    auto place = [&](int i, int& k, int& f) INLINE {  // chunk i's row and first output; false past the last
        const int s = i * NT + tid, c = s % C;
        k = s / C, f = 8 * ((((c >> 1) ^ T::turn(k)) << 1) | (c & 1));
        return k < a.rows && f < a.width - c0;
    };
#pragma unroll
    for (int i = 0; i < T::N; ++i) {
        int k, f;
        if (!place(i, k, f)) k = f = 0;  // (there is one)
        const long long at = panel + (long long)k * 256 + f;
        dh[i] = *reinterpret_cast<const uint4*>(a.dh + k * a.ld_dh + c0 + f);
        g[i] = *reinterpret_cast<const uint4*>(a.kept + at);
        u[i] = *reinterpret_cast<const uint4*>(a.kept + one + at);
        lo[i] = *reinterpret_cast<const uint4*>(a.kept + 2 * one + at);
    }
#pragma unroll
    for (int i = 0; i < T::N; ++i) {
        auto four = [&](uint2 d, uint2 g, uint2 u, uint2 lo) INLINE {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float act, slope;
                act_of<GELU>(kept_g(g, lo, e), act, slope);
                o[e] = bf16_of(d, e) * (side ? act : slope * kept_u(u, lo, e));
            }
            return make_uint2(cvt2(o[0], o[1]), cvt2(o[2], o[3]));
        };
        const uint2 x = four(make_uint2(dh[i].x, dh[i].y), make_uint2(g[i].x, g[i].y), make_uint2(u[i].x, u[i].y), make_uint2(lo[i].x, lo[i].y));
        const uint2 y = four(make_uint2(dh[i].z, dh[i].w), make_uint2(g[i].z, g[i].w), make_uint2(u[i].z, u[i].w), make_uint2(lo[i].z, lo[i].w));
        int k, f;
        const bool in = place(i, k, f);
        const uint4 out = in ? make_uint4(x.x, x.y, y.x, y.y) : make_uint4(0u, 0u, 0u, 0u);
        if (leave && in) *reinterpret_cast<uint4*>(a.dz + side * one + panel + (long long)k * 256 + f) = out;
        to[i * NT + tid] = out;
    }
}

// D[m][n] in tiles of BM x BN, a wavefront BM / WM x BN / WN of 16 x 16 x 32 matrix instructions (from registers alone 2090 TFLOP/s on
// random bf16 values, 32 x 32 x 16 ones 1830; here 1502 us fell to 1410, h alone of 8192 x 4096 x 14336); NS stages of BK k in LDS, filled
// straight from memory.
// - 256 x 256 by 8 wavefronts, along k (h) in two stages of 64, a whole 128-byte line of a row; across (dx, the weights' gradients) in four
//   of 32. 4 wavefronts of 128 x 128 that read their fragments a step ahead, accumulators pinned, took 1474 us for h and 3 % off the
//   others, with matrix instructions that the compiler cannot see the waits of; h in four stages of 32 1490 to 1600; fragments read
//   ahead by 8 wavefronts 1500 to 1640.
// - 192 x 256 where 256 x 256 leaves CUs idle in its last round (2047 x 2880 x 2880: 240 tiles for 184, h 68 to 62 us; 57 since).
// - 128 x 128, 64 x 128 twice a CU, 64 x 64 by two groups of wavefronts that split K: fewer tiles than CUs (choose).
// - few rows: choose_few.
// The epilogues' bf16 leave through LDS in whole runs of a row.
// ONCE: of one column tile each weight's row is read once, past the caches (choose_few).
template <int BM, int BN, int WM, int WN, int WK, int NS, int BK, int EPI, bool GELU, bool ONCE>
__global__ __launch_bounds__(64 * WM * WN * WK) void gt_gemm(const Prod a) {
    constexpr bool PAIR = EPI <= EPI_AGAIN, DW = EPI == EPI_DW || EPI == EPI_DWF, DX = EPI == EPI_DX || EPI == EPI_DXJ;
    constexpr bool AT = !PAIR, BT = DW;
    constexpr int AUX = ONCE ? 2 : 0;
    static_assert(!ONCE || (PAIR && BN <= 64), "one column tile of few rows");
    constexpr int NW = WM * WN, NT = 64 * NW, TM = BM / WM, TN = BN / WN, MI = TM / 16, NI = TN / 16;
    constexpr int CA = BM * BK / 8, CH = CA + BN * BK / 8;  // chunks of A, a stage
    constexpr int NL = CH / NT, NA = CA / NT;               // loads a lane and stage, of A
    constexpr int FM = PAIR ? BM / 2 : BM, FT = PAIR ? TM / 2 : TM;  // outputs of a tile, of a wavefront
    static_assert(NS >= 1 && NS <= 5, "one to five stages");
    constexpr int C1 = NS > 1 ? CH * WK : 1, C2 = NS > 2 ? CH * WK : 1, C3 = NS > 3 ? CH * WK : 1, C4 = NS > 4 ? CH * WK : 1;
    // (an array each, named where it is used: a read waits for the loads to every array that the compiler cannot rule out)
    __shared__ uint4 s0[CH * WK], s1[C1], s2[C2], s3[C3], s4[C4];
    typedef Tile<BM, AT, NT, BK, true> TileA;
    typedef Tile<BN, BT, NT, BK, true> TileB;
    // WK groups of wavefronts, each a share of K in stages of its own, all with the same barriers; tid within the group
    const int group = WK == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / NT), tid = threadIdx.x - group * NT;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), mine = group * CH;
    const int wm = wave / WN, wn = wave % WN;
    if constexpr (EPI == EPI_AGAIN || EPI == EPI_DWF) {
        if (blockIdx.x == 0)
            for (int i = threadIdx.x; i < a.counters; i += 64 * WM * WN * WK) a.arrived[i] = 0;
    }
    int mt, nt, split;
    if (!tile_of(a.tm, a.tn, DX ? a.splits : 1, mt, nt, split)) return;
    const int m0 = mt * FM, n0 = nt * BN;
    // DW: the tile's side, and its first output there
    const int side_n = DW ? a.side0 + (n0 >= a.panels * 256) : 0, c0 = DW ? n0 - (side_n - a.side0) * a.panels * 256 : n0;
    const int n_end = DW ? a.width : a.rows, m_end = PAIR ? a.width : a.dim;
    if (c0 >= n_end) return;  // (what a side's last panel has past its last output)
    // the steps of K: DX sums over gate's outputs, then over up's, each side whole steps
    const int k_end = PAIR ? a.dim : DW ? a.rows : a.width, own = (k_end + BK - 1) / BK;
    const int all = DX ? 2 * own : own;
    // (a split's steps are whole rounds of the stages: the next split's are not its own)
    constexpr int ROUND = NS * WK;
    const int splits = DX ? a.splits : 1;
    const int per = ((all + splits - 1) / splits + ROUND - 1) / ROUND * ROUND, step0 = split * per;
    const int steps = min(per, all - step0);
    const int rounds = steps > 0 ? ((steps + WK - 1) / WK + NS - 1) / NS : 0;  // (of the stages)

    TileA ta;
    TileB tb;
    const int ra = m_end - m0, rb = n_end - c0;  // (rows past the tile's)
    const int ldb = PAIR ? a.ldx : 256;
    if constexpr (PAIR) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int s = i * NT + tid, r = s / ta.CK, c = (s % ta.CK) ^ ta.swz(r);
            ta.off[i] = (uint32_t)((r / 32 * 16 + r % 16) * (r & 16 ? a.ld_up : a.ld_gate) * 2) + 16u * c;
        }
    } else {
        ta.init(tid, DW ? a.ldx : a.ld_gate, ra);
    }
    tb.init(tid, ldb, rb);
    // PAIR: a load of a wavefront has 64 / CK rows, all of gate or all of up: by the wavefront, or where it has fewer than 32
    // rows' loads by the load
    constexpr int ROWS = NT / TileA::CK;  // of a load of all wavefronts
    static_assert(!PAIR || (64 / TileA::CK <= 16 && (ROWS % 32 == 0 || NT == 64 || NT == 128)), "a load is of gate or of up");
    const bool up_wave = wave * (64 / TileA::CK) & 16;
    __amdgpu_buffer_rsrc_t from_a, from_u, from_b;
    int left_a, left_b;
    // where the next step to be loaded lies, and its k (DX: within its side)
    const int st = step0 + group * rounds * NS;
    bool second = DX && st >= own;  // DX: up's steps
    int k = (st - (second ? own : 0)) * BK, la = DW ? a.ldx : second || (PAIR && up_wave) ? a.ld_up : a.ld_gate;
    const uint16_t *pa, *pu = nullptr, *pb;
    if constexpr (PAIR) {
        pa = (ROWS % 32 == 0 && up_wave ? a.up : a.gate) + (long long)m0 * (ROWS % 32 == 0 ? la : a.ld_gate) + k;
        pu = a.up + (long long)m0 * a.ld_up + k;
        pb = a.x + (long long)n0 * a.ldx + k;
    } else if constexpr (DW) {
        pa = a.x + (long long)k * a.ldx + m0;
        pb = a.dz + (side_n * a.panels + (c0 >> 8)) * a.panel + (c0 & 255) + (long long)k * 256;
    } else {
        pa = (second ? a.up : a.gate) + (long long)k * la + m0;
        pb = a.dz + ((second ? a.panels : 0) + (k >> 8)) * a.panel + (k & 255) + n0 * 256ll;
    }
    if (DX && second) ta.init(tid, a.ld_up, ra);
    auto next = [&] INLINE {
        if (DX && k == own * BK && !second) {  // on to up's, whose rows may lie otherwise apart
            second = true, k = 0, la = a.ld_up;
            pa = a.up + m0;
            pb = a.dz + a.panels * a.panel + n0 * 256ll;
            ta.init(tid, la, ra);
        }
        left_a = left_b = k_end - k;
        if constexpr (PAIR) {
            const int r = min(FM, ra);
            from_a = ta.source(pa, ROWS % 32 == 0 ? la : a.ld_gate, r, left_a);
            if constexpr (ROWS % 32) from_u = ta.source(pu, a.ld_up, r, left_a);
            from_b = tb.source(pb, a.ldx, min(BN, rb), left_b);
            pa += BK, pu += BK, pb += BK, k += BK;
        } else if constexpr (DW) {
            from_a = ta.source(pa, a.ldx, ra, left_a);
            from_b = tb.source(pb, 256, rb, left_b);
            pa += (long long)BK * a.ldx, pb += BK * 256, k += BK;
        } else {
            from_a = ta.source(pa, la, ra, left_a);
            from_b = tb.source(pb, 256, min(BN, rb), left_b);
            pa += (long long)BK * la;
            pb += (k & 255) == 256 - BK ? a.panel - 256 + BK : BK;
            k += BK;
        }
    };
    auto load = [&](int i0, int i1, uint4* b) INLINE {  // its loads i0 .. i1 - 1 of NL
#pragma unroll
        for (int i = i0; i < i1; ++i) {
            if (i < NA) {
                if constexpr (PAIR) ta.template load<AUX>(i, ROWS % 32 && (i * ROWS & 16) ? from_u : from_a, left_a, b + mine, tid);
                else ta.load(i, from_a, left_a, b + mine, tid);
            } else {
                tb.load(i - NA, from_b, left_b, b + (mine + CA), tid);
            }
        }
    };
    f32x4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // A step's sums from one stage, the loads of a later step to another; with three stages and more between the sums: a wavefront
    // that issues all of its loads at once stands still until the memory pipeline has taken them, and all do after the barrier.
    // (LATE: the next step's addresses behind the fragments' reads: 2047 x 2880 x 2880 in 192 x 256 73.8 to 72.2 us; 8192 x 4096 x 14336 in
    // 256 x 256 takes 1 % longer with it)
    constexpr bool LATE = NS == 2 && MI * NI < 32;
    auto sum = [&](const uint4* b, uint4* to) INLINE {
        constexpr int U = BK / 32, H = NS >= 3 && MI >= 4 ? 2 : 1;  // (parts of the sums between which the loads lie)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint4 fa[MI], fb[NI];
#pragma unroll
            for (int j = 0; j < NI; ++j) fb[j] = TileB::frag16(b, mine + CA, wn * TN + 16 * j, u, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i) fa[i] = TileA::frag16(b, mine, wm * TM + 16 * i, u, lane);
            if (LATE && u == 0) next();
#pragma unroll
            for (int p = 0; p < H; ++p) {
                if constexpr (NS >= 3) load((u * H + p) * NL / (U * H), (u * H + p + 1) * NL / (U * H), to);
                else if (NS == 2 && u == 0) load(0, NL, to);
#pragma unroll
                for (int i = p * MI / H; i < (p + 1) * MI / H; ++i)
#pragma unroll
                    for (int j = 0; j < NI; ++j) acc[i][j] = mfma16(fa[i], fb[j], acc[i][j]);
                // (one u's fragments at a time: the registers hold no more; a small tile reads them all at once)
                if constexpr (MI * NI > 8) __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // (whole rounds of the stages: steps past the last are zeros, as are the loads past the end into stages that nothing
    // reads. A last step of its own behind a branch would have the compiler copy every accumulator.)
    auto step = [&](uint4* to, const uint4* from) INLINE {
        step_barrier<NS >= 3 ? (NS - 2) * NL : 0>();
        if constexpr (!LATE) next();
        sum(from, to);
    };
    auto first = [&](uint4* to) INLINE {
        next();
        load(0, NL, to);
    };
    if constexpr (EPI == EPI_DWF) {
        static_assert(EPI != EPI_DWF || (NS == 1 && WK == 1), "one stage");
        next();
        load(0, NA, s0);
        dz_tile<TileB, BN, NT, GELU>(a, s0 + CA, tid, side_n, c0, mt == 0);
    } else if (rounds > 0) {
        first(s0);
        if constexpr (NS >= 3) first(s1);
        if constexpr (NS >= 4) first(s2);
        if constexpr (NS >= 5) first(s3);
    }
    for (int s = 0; s < rounds; ++s) {
        if constexpr (NS == 1) {  // (more workgroups instead)
            step_barrier<0>();
            sum(s0, s0);
            if (s + 1 < rounds) {
                step_barrier<0>();
                first(s0);
            }
        } else if constexpr (NS == 2) {
            step(s1, s0);
            step(s0, s1);
        } else if constexpr (NS == 3) {
            step(s2, s0);
            step(s0, s1);
            step(s1, s2);
        } else if constexpr (NS == 4) {
            step(s3, s0);
            step(s0, s1);
            step(s1, s2);
            step(s2, s3);
        } else {
            step(s4, s0);
            step(s0, s1);
            step(s1, s2);
            step(s2, s3);
            step(s3, s4);
        }
    }
    step_barrier<0>();  // (the last loads landed: they write this workgroup's LDS)
    if constexpr (WK > 1) {  // the other groups' sums to the first
        static_assert(WK == 1 || (WK - 1) * NW * MI * NI * 64 <= C1, "their sums fit a stage");
        f32x4* const at = reinterpret_cast<f32x4*>(s1) + wave * MI * NI * 64 + lane;
        if (group) {
            f32x4* to = at + (group - 1) * NW * MI * NI * 64;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) to[64 * (i * NI + j)] = acc[i][j];
        }
        step_barrier<0>();
        if (EPI != EPI_DXJ && group) return;
#pragma unroll
        for (int w = 0; w < WK - 1 && group == 0; ++w)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] += at[w * NW * MI * NI * 64 + 64 * (i * NI + j)];
    }

    if constexpr (EPI == EPI_DXJ) {
        // The L2s of the XCDs are not coherent with each other: device-scope accesses, each lane's own places, in the splits' order.
        __shared__ uint32_t before;
        if (splits > 1) {
            const int tile = mt * a.tn + nt;
            // (two at a time)
            uint64_t* const sums = reinterpret_cast<uint64_t*>(a.acc) + (long long)tile * splits * (BM * BN / 2) + tid;
            // (the fragments with rows: both gradients of 8 x 1024 x 4096 23.2 to 21.8 us, of 48 rows 24.9 to 24.6)
            const int live = (rb - wn * TN + 15) / 16;
            if (!group) {
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    if (j >= live) break;
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            __hip_atomic_store(sums + split * (BM * BN / 2) + ((i * NI + j) * 2 + e) * NT,
                                               __builtin_bit_cast(uint64_t, (f32x2{acc[i][j][2 * e], acc[i][j][2 * e + 1]})), __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_AGENT);
                }
            }
            step_barrier<0>();  // (they have landed)
            if (threadIdx.x == 0) before = __hip_atomic_fetch_add(a.arrived + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            step_barrier<0>();
            if (before != (uint32_t)(splits - 1)) return;
            auto join = [&](int fragments) INLINE {
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < fragments; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                for (int w = 0; w < splits; ++w)
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int j = 0; j < fragments; ++j)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const f32x2 v = __builtin_bit_cast(f32x2, __hip_atomic_load(sums + w * (BM * BN / 2) + ((i * NI + j) * 2 + e) * NT,
                                                                                            __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
                                acc[i][j][2 * e] += v[0], acc[i][j][2 * e + 1] += v[1];
                            }
            };
            static_assert(EPI != EPI_DXJ || NI == 2, "one fragment or both");
            if (!group && live >= 2) join(2);
            else if (!group && live == 1) join(1);
        }
        if (group) return;
    }

    // lane: columns n = c0 + wn TN + 16 j + lane % 16, rows mw + 16 i + 4 (lane / 16) + 0 .. 3; two j's columns at a time
    const int r = lane & 15, q4 = lane >> 4;
    const int mw = m0 + wm * FT;
    // the wavefront's own part of the stages: 32 columns of its FT rows in bf16
    constexpr int C16 = FT / 8, CP = C16 == 6 ? 8 : C16 == 12 ? 16 : C16, SWZ = CP < 16 ? CP - 1 : 15;  // 16-byte chunks a column, their stride and turn
    static_assert((CP & (CP - 1)) == 0, "chunks turn within a power of two");
    constexpr int PART = 32 * CP, FIT = CH * WK / PART, PER = FIT < NW ? FIT : NW, PARTS = (NW + PER - 1) / PER;
    static_assert(PARTS <= NS && PARTS <= 4 && (WK == 1 || PARTS == 1), "the wavefronts' parts fit the stages that are free");
    uint4* region = s0 + (wave % PER) * PART;
    if constexpr (PARTS > 1) {
        const int at = wave / PER;
        region = (at == 0 ? s0 : at == 1 ? s1 : at == 2 ? s2 : s3) + (wave % PER) * PART;
    }
    // 32 columns in bf16, 4 rows of column 16 jj + r at 8-byte unit q: to and from whole runs of a column's rows in memory
    uint2* const half = reinterpret_cast<uint2*>(region);
    auto unit = [&](int jj, int q) -> uint2& { return half[((16 * jj + r) * CP + ((q >> 1) ^ (r & SWZ))) * 2 + (q & 1)]; };
    auto each = [&](auto&& f) INLINE {  // f(column, 8 of its rows, where they lie) over the wavefront's chunks
#pragma unroll
        for (int t = 0; t < C16 / 2; ++t) {
            const int s = t * 64 + lane, c = s / C16, q = s % C16;
            f(c, 8 * q, region[c * CP + (q ^ (c & SWZ))]);
        }
        __builtin_amdgcn_wave_barrier();
    };
    auto store = [&](auto&& at, int cols, int rows) INLINE {  // at(c, row): column c's place for 8 of its rows from `row` on
        __builtin_amdgcn_wave_barrier();
        each([&](int c, int row, const uint4& v) INLINE {
            if (c >= cols || row >= rows) return;
            f32x4* o = reinterpret_cast<f32x4*>(at(c, row));
            const f32x4 w = __builtin_bit_cast(f32x4, v);
            if (PAIR && a.past) {
                asm volatile("" ::: "memory");  // (around it: else the compiler makes one plain store of both)
                __builtin_nontemporal_store(w, o);
                asm volatile("" ::: "memory");
            } else {
                *o = w;
            }
        });
    };
#pragma unroll
    for (int j = 0; j < NI; j += 2) {
        const int nj = c0 + wn * TN + 16 * j;
        if constexpr (PAIR) {
            constexpr int HI = MI / 2;  // (gate's and up's rows in turn)
            // output mw + row of row nj + c in the panels
            auto panel = [&](int c, int row) INLINE { return ((mw + row) >> 8) * a.panel + (long long)(nj + c) * 256 + ((mw + row) & 255); };
            const int left = a.width - mw;
            const long long side = a.panels * a.panel;
            uint2 d[2][HI];
            if constexpr (EPI == EPI_AGAIN) {
                const uint16_t* from = a.dh + nj * a.ld_dh + mw;
                each([&](int c, int row, uint4& v) INLINE {
                    v = nj + c < n_end && row < left ? *reinterpret_cast<const uint4*>(from + c * a.ld_dh + row) : make_uint4(0u, 0u, 0u, 0u);
                });
#pragma unroll
                for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                    for (int i = 0; i < HI; ++i) d[jj][i] = unit(jj, 4 * i + q4);
                __builtin_amdgcn_wave_barrier();
            }
            uint2 more[3][2][HI];  // AGAIN: du; KEEP: what is kept
#pragma unroll
            for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                for (int i = 0; i < HI; ++i) {
                    float o[4], p[4];
                    uint32_t gb[4], ub[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float gate = acc[2 * i][j + jj][e], u = acc[2 * i + 1][j + jj][e];
                        float act, slope;
                        act_of<GELU>(gate, act, slope);
                        if constexpr (EPI == EPI_AGAIN) {
                            const float dh = bf16_of(d[jj][i], e);
                            o[e] = dh * (slope * u);
                            p[e] = dh * act;
                        } else {
                            o[e] = act * u;
                            gb[e] = __float_as_uint(gate);
                            ub[e] = __float_as_uint(u);
                        }
                    }
                    unit(jj, 4 * i + q4) = make_uint2(cvt2(o[0], o[1]), cvt2(o[2], o[3]));
                    if constexpr (EPI == EPI_AGAIN) more[0][jj][i] = make_uint2(cvt2(p[0], p[1]), cvt2(p[2], p[3]));
                    if constexpr (EPI == EPI_KEEP) more[0][jj][i] = upper(gb), more[1][jj][i] = upper(ub), more[2][jj][i] = lower(gb, ub);
                }
            if constexpr (EPI == EPI_AGAIN) store([&](int c, int row) INLINE { return a.dz + panel(c, row); }, n_end - nj, left);
            else store([&](int c, int row) INLINE { return a.h + (nj + c) * a.ld_h + mw + row; }, n_end - nj, left);
            constexpr int MORE = EPI == EPI_KEEP ? 3 : EPI == EPI_AGAIN ? 1 : 0;
            uint16_t* const to = EPI == EPI_KEEP ? a.kept : a.dz + side;
#pragma unroll
            for (int m = 0; m < MORE; ++m) {
#pragma unroll
                for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                    for (int i = 0; i < HI; ++i) unit(jj, 4 * i + q4) = more[m][jj][i];
                store([&](int c, int row) INLINE { return to + m * side + panel(c, row); }, n_end - nj, left);
            }
        } else if (DW || EPI == EPI_DXJ || a.dx != nullptr) {
#pragma unroll
            for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    const f32x4 v = acc[i][j + jj];
                    unit(jj, 4 * i + q4) = make_uint2(cvt2(v[0], v[1]), cvt2(v[2], v[3]));
                }
            const long long ld = DX ? a.ld_dx : side_n ? a.ld_dup : a.ld_dgate;
            uint16_t* o = (DX ? a.dx : side_n ? a.dup : a.dgate) + nj * ld + mw;
            store([&](int c, int row) INLINE { return o + c * ld + row; }, n_end - nj, m_end - mw);
        } else {
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
                const int n = nj + 16 * jj + r;
                if (n >= n_end) continue;
                float* o = a.acc + ((long long)split * a.rows + n) * a.dim + mw + 4 * q4;
#pragma unroll
                for (int i = 0; i < MI; ++i)
                    if (mw + 16 * i + 4 * q4 < m_end) *reinterpret_cast<f32x4*>(o + 16 * i) = acc[i][j + jj];
            }
        }
    }
}

// --- between and after the products -------------------------------------------------------------------------------------

struct Slope {
    const uint16_t *kept, *dh;
    uint16_t* dz;
    long long ld_dh, panel, side;  // (values of one panel, of one side)
    int rows, width;
    uint32_t* arrived;  // cleared
    int counters;
};

__device__ __forceinline__ uint2 passing(const uint16_t* at) {  // read once
    typedef __attribute__((__vector_size__(8))) uint32_t u32x2;
    const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(at));
    return make_uint2(v[0], v[1]);
}

// dg and du from dh and what the forward call kept: a wavefront's rows of one panel. PAST: the caches hold none of it (8192 x 14336: 1.41
// GB in 216 us, 6.5 TB/s; 224 to 268 without).
constexpr int SLOPE_ROWS = 8;  // a wavefront, asked for at once
template <bool GELU, bool PAST>
__global__ __launch_bounds__(256) void gt_slope(const Slope p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = (blockIdx.y * 4 + wave) * SLOPE_ROWS, f = blockIdx.x * 256 + 4 * lane;
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = threadIdx.x; i < p.counters; i += 256) p.arrived[i] = 0;
    if (n0 >= p.rows || f >= p.width) return;
    const long long at = blockIdx.x * p.panel + (long long)n0 * 256 + 4 * lane;
    uint2 dh[SLOPE_ROWS], g[SLOPE_ROWS], u[SLOPE_ROWS], lo[SLOPE_ROWS];
#pragma unroll
    for (int i = 0; i < SLOPE_ROWS; ++i) {
        const int n = min(i, p.rows - 1 - n0);
        const uint16_t *d = p.dh + (n0 + n) * p.ld_dh + f, *k = p.kept + at + n * 256;
        auto get = [](const uint16_t* at) { return PAST ? passing(at) : *reinterpret_cast<const uint2*>(at); };
        dh[i] = get(d), g[i] = get(k), u[i] = get(k + p.side), lo[i] = get(k + 2 * p.side);
    }
#pragma unroll
    for (int i = 0; i < SLOPE_ROWS; ++i) {
        if (n0 + i >= p.rows) break;
        float dg[4], du[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float act, slope;
            act_of<GELU>(kept_g(g[i], lo[i], e), act, slope);
            const float d = bf16_of(dh[i], e);
            dg[e] = d * (slope * kept_u(u[i], lo[i], e));
            du[e] = d * act;
        }
        *reinterpret_cast<uint2*>(p.dz + at + i * 256) = make_uint2(cvt2(dg[0], dg[1]), cvt2(dg[2], dg[3]));
        *reinterpret_cast<uint2*>(p.dz + p.side + at + i * 256) = make_uint2(cvt2(du[0], du[1]), cvt2(du[2], du[3]));
    }
}

struct Join {
    const float* acc;
    uint16_t* dx;
    long long ld_dx;
    int splits, rows, dim;
};

// dx from the splits' sums, in their order: 4 values a lane
__global__ __launch_bounds__(256) void gt_join(const Join p) {
    const int cols = p.dim / 4;
    const long long stride = (long long)p.rows * p.dim;
    for (long long w = blockIdx.x * 256ll + threadIdx.x; w < (long long)p.rows * cols; w += gridDim.x * 256ll) {
        const int n = (int)(w / cols), d = 4 * (int)(w - (long long)n * cols);
        const float* at = p.acc + (long long)n * p.dim + d;
        f32x4 v = *reinterpret_cast<const f32x4*>(at);
#pragma unroll 4
        for (int i = 1; i < p.splits; ++i) v += *reinterpret_cast<const f32x4*>(at + i * stride);
        *reinterpret_cast<uint2*>(p.dx + n * p.ld_dx + d) = make_uint2(cvt2(v[0], v[1]), cvt2(v[2], v[3]));
    }
}

// --- the plan -----------------------------------------------------------------------------------------------------------

constexpr int MOST_TILES = (1 << 23) - 8;  // of 512 lanes: a launch holds fewer than 2^32

long long up(long long v, long long to) { return (v + to - 1) / to * to; }

// (K: groups of wavefronts that split the sum)
enum Tiles { T256, T192x256, T128, T64x128, T64K2, T256x64, T128x64, T32x64K4, T64x32, T64x32K4, T32K4 };
struct Size {
    int bm, bn, wk;
};
constexpr Size SIZE[] = {{256, 256, 1}, {192, 256, 1}, {128, 128, 1}, {64, 128, 1}, {64, 64, 2}, {256, 64, 1},
                         {128, 64, 1},  {32, 64, 4},   {64, 32, 1},   {64, 32, 4},  {32, 32, 4}};

// The times of a workgroup, fitted to the kernels' at 35 to 60 shapes of 72 to 4096 rows, 512 to 4096 values and 1408 to 14336 outputs,
// most within 6 % (dx 12 %); what they choose is the fastest of these tiles or within 2 % of it at all of them (dx: within 8 %).
Pace pace_of(int epi, int t) {
    const bool dx = epi == EPI_DX, dw = epi == EPI_DW;
    switch (t) {
        case T256: return dx ? Pace{CUS, 1.45f, 0.05f, 1.5f} : dw ? Pace{CUS, 0.66f, 0.77f, 7.9f} : Pace{CUS, 1.07f, 0.435f, 3.f};
        case T192x256: return dw ? Pace{CUS, 0.73f, 0.33f, 6.2f} : Pace{CUS, 0.875f, 0.313f, 3.1f};
        case T128: return dx ? Pace{2 * CUS, 0.63f, 0.55f, 0.5f} : dw ? Pace{2 * CUS, 0.23f, 0.62f, 4.2f} : Pace{2 * CUS, 0.557f, 0.351f, 2.f};
        case T64x128: return Pace{2 * CUS, 0.244f, 0.327f, 1.9f};
        case T256x64: return Pace{CUS, 1.05f, 0.3f, 8.f};
        default: return dx ? Pace{CUS, 0.19f, 0.05f, 2.f} : Pace{CUS, 0.25f, 0.03f, 2.1f};
    }
}

long long tiles_of(int t, long long m, long long n) { return up(m, SIZE[t].bm) / SIZE[t].bm * (up(n, SIZE[t].bn) / SIZE[t].bn); }

// dx's splits of its long sum, for half a round of workgroups to two: their sums' way back through memory costs a launch and about 3.5
// TB/s, or (T64K2) the last workgroup of a tile half a us for each.
int splits_of(int t, int tiles, int steps, float* us) {
    const Pace p = pace_of(EPI_DX, t);
    int best = 1;
    *us = tiled_us(p, tiles, steps);
    for (int h = 1; h <= 4; ++h) {
        int s = h * p.at_once / (2 * tiles);
        if (s > steps / 4) s = steps / 4;
        if (s < 2) continue;
        const float join = t == T64K2 ? 0.55f * s : 4.f + (float)tiles * s * SIZE[t].bm * SIZE[t].bn * 4 * 0.28e-6f;
        const float here = tiled_us(p, tiles * s, ((steps + s - 1) / s + 1) & ~1) + join;
        if (here < *us) *us = here, best = s;
    }
    return best;
}

// the tile of `tiles` that takes the least time for a product of m rows by n columns, summed over k; -1: more of each than a launch holds
int choose(int epi, long long m, long long n, long long k, std::initializer_list<int> tiles, int* splits = nullptr) {
    int best = -1;
    float least = 1e30f;
    const int steps = (int)(up(k, KSTEP) / KSTEP);
    for (int t : tiles) {
        if (tiles_of(t, m, n) >= MOST_TILES) continue;
        float us;
        int s = 1;
        if (epi == EPI_DX) s = splits_of(t, (int)tiles_of(t, m, n), steps, &us);
        else us = tiled_us(pace_of(epi, t), (int)tiles_of(t, m, n), steps);
        if (us < least) {
            least = us, best = t;
            if (splits) *splits = s;
        }
    }
    return best;
}

// dx of few rows waits for the weights: past what the caches hold by tall tiles (64 x 4096 x 14336 57 us, by T64K2 63; 8 rows 48 and 54; 64
// x 4096 x 4096 28 and 27)
constexpr long long HELD = 96ll << 20;

// g and u of few rows wait for the weights alone: tiles as narrow as the rows, as many of them and as many groups of wavefronts each as
// keep the most of them on the way. us, weights from memory, n x dim x width: 8 x 4096 x 4096 13.8 by T32K4 and 17.9 by T64x32K4, 16 x
// 2048 x 8192 17.6 and 15.1, 32 x 512 x 14336 19.5, 13.5 and 8.5 by T64x32; 33 x 2880 x 2880 13.4 by T32x64K4 and 15.7 by T64K2, 64 x
// 2048 x 8192 22.4 and 15.5, 64 x 4096 x 14336 67, 51 and 43.8 by T128x64.
// One tile has all rows (FEW), so a product reads each weight once, past the caches: 8 x 4096 x 4096 13.8 and 15.2 through them, 64 x 2048
// x 8192 15.8 and 17.7, 16 x 1024 x 4096 6.9 and 7.1, 32 x 4096 x 14336 42 and 47. (What reads them after it then finds none there: both
// gradients computed again, 48 x 1024 x 4096 31.5 and 29.1, 8 x 4096 x 4096 55 and 55, 32 x 4096 x 14336 154 and 164.) T64K2 of more rows
// has several tiles read each weight and leaves them in the caches: 128 x 2880 x 2880 18.4 and 19.4 past them, a step 55 and 62; 256 x
// 512 x 1408 5.8 and 6.9; 100 x 1024 x 4096 8.9 and 8.7, a step 35.2 and 38.6.
constexpr int FEW = 64;
int choose_few(int n, int width) {
    const int units = (width + 15) / 16;
    if (n <= 32) return units <= CUS ? T32K4 : units <= 2 * CUS ? T64x32K4 : T64x32;
    return units <= CUS ? T32x64K4 : units <= 2 * CUS ? T64K2 : T128x64;
}

struct Plan {
    int panels, z, w, d, splits;
    bool once;       // z's loads of the weights pass the caches
    bool one_stage;  // DW
    bool fused;      // DWF
    int counters;    // DXJ
    long long kept, acc, arrived, bytes;  // (the workspace: dg and du, then the sums of dx's splits, then the counters)
};

bool ld_ok(long long ld, long long least) { return ld >= least && ld % 8 == 0; }

bool plan_of(const dr_gated* a, int what, Plan& p) {
    if (a == nullptr || (what != DR_GATED_FORWARD && what != DR_GATED_BACKWARD) || a->rows < 1 || a->rows > (1 << 20) ||
        a->dim < 8 || a->dim > (1 << 17) || a->dim % 8 || a->width < 8 || a->width > (1 << 20) || a->width % 8 || a->act < 0 ||
        a->act > 1 || !ld_ok(a->ldx, a->dim) || !ld_ok(a->ld_gate, a->dim) || !ld_ok(a->ld_up, a->dim) ||
        a->ldx > DR_GATED_MAX_LD || a->ld_gate > DR_GATED_MAX_LD || a->ld_up > DR_GATED_MAX_LD)
        return false;
    const long long n = a->rows, f = a->width, d = a->dim;
    p = Plan{};
    p.panels = (int)(up(f, 256) / 256);
    p.kept = 3ll * p.panels * n * 512;
    const bool back = what == DR_GATED_BACKWARD;
    // (a backward call's sizes are those of a forward call)
    p.z = n <= FEW ? choose_few((int)n, a->width) : choose(EPI_ACT, 2 * f, n, d, {T256, T192x256, T128, T64x128, T64K2});
    p.once = n <= FEW;
    if (p.z < 0) return false;
    if (!back) return true;
    long long at = 2ll * p.panels * n * 512;
    if (a->dgate || a->dup) {
        p.w = choose(EPI_DW, d, up(f, 256) * ((a->dgate != nullptr) + (a->dup != nullptr)), n, {T256, T192x256, T128});
        p.one_stage = n <= KSTEP || (p.w == T128 && n <= 1024);
        if (p.w < 0 || (p.one_stage && tiles_of(T128, d, 2 * up(f, 256)) >= MOST_TILES)) return false;
    }
    p.acc = at;
    if (a->dx) {
        if (n > 64) p.d = choose(EPI_DX, d, n, 2 * f, {T256, T128, T64K2}, &p.splits);
        else if (4 * f * d > HELD) p.d = choose(EPI_DX, d, n, 2 * f, {T256x64}, &p.splits);
        else p.d = choose(EPI_DX, d, n, 2 * f, {T64K2}, &p.splits);
        if (p.d < 0) return false;
        if (p.splits > 1 && p.d == T64K2) {
            p.counters = (int)tiles_of(T64K2, d, n);
            at += (long long)p.splits * p.counters * (64 * 64 * 4);
            p.arrived = at;
            at += up(p.counters * 4, 256);
        } else if (p.splits > 1) at += up(p.splits * n * d * 4, 256);
    }
    // of both sides, so that dx finds them; and few tiles, each row of which makes them again (16 x 4096 x 1408, 768 tiles, 22 us and 24 by a
    // pass of its own; 33 x 2880 x 2880, 1104 tiles, 29.6 and 28.8; 64 x 4096 x 14336 154 and 126)
    p.fused = p.one_stage && a->kept && a->dgate && a->dup && n <= KSTEP && tiles_of(T128, d, 2 * up(f, 256)) <= 4 * CUS;
    p.bytes = a->dx || a->dgate || a->dup ? at : 0;
    return true;
}

template <int BM, int BN, int WM, int WN, int WK, int NS, int BK, int EPI, bool GELU, bool ONCE = false>
void launch(Prod g, int m, int n, hipStream_t st) {
    g.tm = (m + BM - 1) / BM;
    g.tn = (n + BN - 1) / BN;
    const int grid = (g.tm * g.tn * (EPI == EPI_DX || EPI == EPI_DXJ ? g.splits : 1) + 7) & ~7;  // (as many for each XCD)
    hipLaunchKernelGGL((gt_gemm<BM, BN, WM, WN, WK, NS, BK, EPI, GELU, ONCE>), dim3(grid), dim3(64 * WM * WN * WK), 0, st, g);
}

template <int EPI, bool GELU>
void launch_act(const Prod& g, int t, bool once, hipStream_t st) {
    const int m = 2 * g.width, n = g.rows;
    switch (t) {
        case T256: return launch<256, 256, 2, 4, 1, 2, 64, EPI, GELU>(g, m, n, st);
        case T192x256: return launch<192, 256, 2, 4, 1, 2, 64, EPI, GELU>(g, m, n, st);
        case T64x128: return launch<64, 128, 1, 4, 1, 3, 64, EPI, GELU>(g, m, n, st);
        case T32K4: return launch<32, 32, 1, 1, 4, 4, 64, EPI, GELU, true>(g, m, n, st);
        case T64x32K4: return launch<64, 32, 1, 1, 4, 3, 64, EPI, GELU, true>(g, m, n, st);
        case T64x32: return launch<64, 32, 1, 1, 1, 5, 64, EPI, GELU, true>(g, m, n, st);
        case T32x64K4: return launch<32, 64, 1, 1, 4, 3, 64, EPI, GELU, true>(g, m, n, st);
        case T128: return launch<128, 128, 2, 2, 1, 2, 64, EPI, GELU>(g, m, n, st);
        case T128x64: return launch<128, 64, 2, 2, 1, 3, 64, EPI, GELU, true>(g, m, n, st);
        default: return once ? launch<64, 64, 1, 2, 2, 4, 64, EPI, GELU, true>(g, m, n, st) : launch<64, 64, 1, 2, 2, 4, 64, EPI, GELU>(g, m, n, st);
    }
}

template <int EPI>
void launch_act(const Prod& g, int act, const Plan& p, hipStream_t st) {
    if (act) launch_act<EPI, true>(g, p.z, p.once, st);
    else launch_act<EPI, false>(g, p.z, p.once, st);
}

// What a forward call leaves passes the caches by where they (256 MB) could not hold it until it is read: 8192 x 4096 x 14336 1604 to
// 1464 us with what is kept, the pass that reads that 10 us less; but 1003 x 2048 x 5632 40 and 44.
bool past_caches(const dr_gated* a) { return (a->kept ? 8ll : 2ll) * a->rows * a->width > 256ll << 20; }

bool aligned(const void* p, uintptr_t to) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace

extern "C" int64_t dr_gated_kept_bytes(const dr_gated* a) {
    Plan p;
    return plan_of(a, DR_GATED_FORWARD, p) ? p.kept : -1;
}

extern "C" int64_t dr_gated_workspace_bytes(const dr_gated* a, int what) {
    Plan p;
    return plan_of(a, what, p) ? p.bytes : -1;
}

extern "C" int dr_gated_plan(const dr_gated* a, int what, dr_gated_info* info) {
    Plan p;
    if (info == nullptr || !plan_of(a, what, p)) return DR_EINVAL;
    *info = dr_gated_info{};
    auto tile = [](int32_t (&to)[3], int t) { to[0] = SIZE[t].bm, to[1] = SIZE[t].bn, to[2] = SIZE[t].wk; };
    const bool back = what == DR_GATED_BACKWARD;
    if (!back || (a->kept == nullptr && (a->dx || a->dgate || a->dup))) tile(info->act, p.z), info->act_once = p.once;
    if (!back) return DR_OK;
    if (a->dgate || a->dup) tile(info->dweight, p.one_stage ? T128 : p.w), info->dweight_stages = p.one_stage ? 1 : p.w == T192x256 ? 2 : 4;
    if (a->dx) tile(info->dx, p.d), info->dx_splits = p.splits;
    return DR_OK;
}

extern "C" int dr_gated_run(const dr_gated* a, int what) {
    Plan P;
    if (!plan_of(a, what, P)) return DR_EINVAL;
    const bool back = what == DR_GATED_BACKWARD;
    if (!aligned(a->x, 16) || !aligned(a->gate, 16) || !aligned(a->up, 16) || (a->kept && !aligned(a->kept, 16)) ||
        (!back && (!aligned(a->h, 16) || !ld_ok(a->ld_h, a->width))) ||
        (back && (!aligned(a->dh, 16) || !ld_ok(a->ld_dh, a->width) || (P.bytes && (!aligned(a->workspace, 256) || a->workspace_bytes < P.bytes)) ||
                  (a->dx && (!aligned(a->dx, 16) || !ld_ok(a->ld_dx, a->dim))) ||
                  (a->dgate && (!aligned(a->dgate, 16) || !ld_ok(a->ld_dgate, a->dim))) ||
                  (a->dup && (!aligned(a->dup, 16) || !ld_ok(a->ld_dup, a->dim))))))
        return DR_EINVAL;
    const hipStream_t st = reinterpret_cast<hipStream_t>(a->stream);
    Prod g{};
    g.x = reinterpret_cast<const uint16_t*>(a->x), g.ldx = (int)a->ldx;
    g.gate = reinterpret_cast<const uint16_t*>(a->gate), g.ld_gate = (int)a->ld_gate;
    g.up = reinterpret_cast<const uint16_t*>(a->up), g.ld_up = (int)a->ld_up;
    g.rows = a->rows, g.dim = a->dim, g.width = a->width;
    g.panels = P.panels, g.panel = a->rows * 256ll;
    const bool past = past_caches(a);
    if (!back) {
        g.h = reinterpret_cast<uint16_t*>(a->h), g.ld_h = a->ld_h;
        g.kept = reinterpret_cast<uint16_t*>(a->kept);
        g.past = past;
        if (a->kept) launch_act<EPI_KEEP>(g, a->act, P, st);
        else launch_act<EPI_ACT>(g, a->act, P, st);
        return hipGetLastError() == hipSuccess ? DR_OK : DR_EHIP;
    }
    if (!a->dx && !a->dgate && !a->dup) return DR_OK;
    char* ws = reinterpret_cast<char*>(a->workspace);
    g.dz = reinterpret_cast<uint16_t*>(ws);
    g.dh = reinterpret_cast<const uint16_t*>(a->dh), g.ld_dh = a->ld_dh;
    g.kept = reinterpret_cast<uint16_t*>(a->kept);
    g.arrived = reinterpret_cast<uint32_t*>(ws + P.arrived), g.counters = P.counters;
    if (a->kept && !P.fused) {
        Slope s{reinterpret_cast<const uint16_t*>(a->kept), g.dh, g.dz, a->ld_dh, g.panel, P.panels * g.panel, a->rows, a->width,
                g.arrived, g.counters};
        const int rows = 4 * SLOPE_ROWS;
        const dim3 grid(P.panels, (a->rows + rows - 1) / rows);
        auto slope = a->act ? past ? gt_slope<true, true> : gt_slope<true, false> : past ? gt_slope<false, true> : gt_slope<false, false>;
        hipLaunchKernelGGL(slope, grid, dim3(256), 0, st, s);
    } else if (!a->kept) {
        launch_act<EPI_AGAIN>(g, a->act, P, st);
    }
    if (a->dgate || a->dup) {
        g.dgate = reinterpret_cast<uint16_t*>(a->dgate), g.ld_dgate = a->ld_dgate;
        g.dup = reinterpret_cast<uint16_t*>(a->dup), g.ld_dup = a->ld_dup;
        g.side0 = a->dgate ? 0 : 1;
        const int outputs = 256 * P.panels * (a->dgate && a->dup ? 2 : 1);
        if (P.fused && a->act) launch<128, 128, 2, 2, 1, 1, 64, EPI_DWF, true>(g, a->dim, outputs, st);
        else if (P.fused) launch<128, 128, 2, 2, 1, 1, 64, EPI_DWF, false>(g, a->dim, outputs, st);
        else if (P.one_stage) launch<128, 128, 2, 2, 1, 1, 64, EPI_DW, false>(g, a->dim, outputs, st);
        else if (P.w == T256) launch<256, 256, 2, 4, 1, 4, 32, EPI_DW, false>(g, a->dim, outputs, st);
        else if (P.w == T192x256) launch<192, 256, 2, 4, 1, 2, 64, EPI_DW, false>(g, a->dim, outputs, st);
        else launch<128, 128, 2, 2, 1, 4, 32, EPI_DW, false>(g, a->dim, outputs, st);
    }
    if (a->dx) {
        g.splits = P.splits;
        g.acc = reinterpret_cast<float*>(ws + P.acc);
        g.dx = P.splits > 1 ? nullptr : reinterpret_cast<uint16_t*>(a->dx), g.ld_dx = a->ld_dx;
        if (P.d == T64K2) {
            g.dx = reinterpret_cast<uint16_t*>(a->dx);
            launch<64, 64, 2, 2, 2, 4, 64, EPI_DXJ, false>(g, a->dim, a->rows, st);
        }
        else if (P.d == T256x64) launch<256, 64, 2, 2, 1, 4, 32, EPI_DX, false>(g, a->dim, a->rows, st);
        else if (P.d == T128) launch<128, 128, 2, 2, 1, 4, 32, EPI_DX, false>(g, a->dim, a->rows, st);
        else launch<256, 256, 2, 4, 1, 4, 32, EPI_DX, false>(g, a->dim, a->rows, st);
        if (P.splits > 1 && P.d != T64K2) {
            Join j{g.acc, reinterpret_cast<uint16_t*>(a->dx), a->ld_dx, P.splits, a->rows, a->dim};
            const long long items = ((long long)a->rows * (a->dim / 4) + 255) / 256;
            hipLaunchKernelGGL(gt_join, dim3((unsigned)(items < 4096 ? items : 4096)), dim3(256), 0, st, j);
        }
    }
    return hipGetLastError() == hipSuccess ? DR_OK : DR_EHIP;
}
