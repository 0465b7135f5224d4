// head_loss.hip: the LM head's losses and their gradients for MI355X (gfx950), behind include/lm_head.h.
//
// Three products carry the work, all of one tiled MFMA kernel (hl_gemm), whose operands lie in memory either along the
// summed dimension or across it (read through the LDS transpose read), so that nothing is transposed in memory:
//   z  [v][n]  = head . x^T      summed over dim;    the softmax's statistics, or dz, are its epilogue
//   dhead [v][d] = dz^T . x      summed over rows;   x and dz across
//   dx [n][d]  = dz . head       summed over v;      head across
// A call is a few launches: the entries (ids checked, the teacher's softmax), the rows that count found (and gathered, where
// some do not: rows left out cost nothing and whatever they hold enters no sum), z with each tile's maximum and sum of a row,
// their merge into lse and loss; backward, piece by piece of the vocabulary, dz from z computed again, a teacher's entries' own
// dz, dhead's rows, dx's sum so far. Large calls do not keep the logits: that is one product more than a program that keeps
// them. One of both directions whose dz is one piece (1 GB) keeps them from the loss to dz where that is faster (KEEP_DIM), and
// of few rows takes all between the products in one launch (hl_few).
//
// What bounds them (8192 rows x 4096 against 128256 tokens, 27.68 ms in one trace; a large library product of the same layouts
// runs at 1200, 985 and 1110 TFLOP/s): z 6.85 ms (1256 TFLOP/s), dz 7.21 (1195), dhead 6.72 (1281), dx 6.88 (1252), all else
// 0.03. With zeros for inputs the same kernels run at 1530 to 1790 TFLOP/s and 2.4 GHz: the power that random values draw, at
// 1.8 GHz, holds them there. 32 rows: 171 us for the 1.05 GB of the head, 6.1 TB/s. A few rows against a small
// vocabulary: each launch's start, its first loads and a chain of LDS reads and matrix instructions (48 x 1024 against 8192:
// 5 launches of 4 to 9 us).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <initializer_list>

#include "dense_reader.h"
#include "lm_head.h"
#include "mfma_tile.h"

#pragma clang fp contract(off)

namespace {

constexpr float LN2 = 0.6931471805599453f;

// two maxima, in the exponent of 2, and sums of what exceeds them
__device__ __forceinline__ void join(float& m, float& s, float v, float w) {
    if (v == -INFINITY) return;  // (nothing there)
    const float top = fmaxf(m, v);
    s = s * __builtin_amdgcn_exp2f(m - top) + w * __builtin_amdgcn_exp2f(v - top);
    m = top;
}

// --- the tiled product ------------------------------------------------------------------------------------------------

struct Gemm {
    const uint16_t *A, *B;  // D[m][n] = sum over k of A[m][k] B[n][k]; an operand lies [rows][k] or (across) [k][rows]
    long long lda, ldb;
    int m, n, k;            // (k: of a [rows][k] operand a multiple of 8)
    int ka;                 // the k rows that an A across has (past them zeros)
    int nb;                 // dhead: the columns that B has (past them zeros)
    long long panel;        // dz lies in panels of 256 v: v at (v / 256) panel + row 256 + v % 256
    const int* live;        // the rows that count: n of z and dx, k of dhead
    const uint16_t* whole;  // x where it lies ([rows][ldx]), for B of z and A of dhead where every row counts; or NULL
    long long ldx;
    int rows;
    int tm, tn;             // tiles
    // z's epilogues
    float sc;               // z to the exponent of 2: log2(e) / T
    int v0;                 // z's row 0 is the vocabulary's v0
    const int* idx;         // row that counts -> row, or NULL: itself
    const float* lse;       // [rows]
    const float* g;         // [rows], or NULL: ones
    const float* top;       // the factor taken out of dz
    f32x2* part;            // [m / BM][n] maximum and sum
    long long ld_part;
    const int* ids;         // [rows that count][1 << kp] entries, -1 none
    const void* raw;        // or tokens as they came ([rows] int32, or int64: raw64; one after another), those past m none
    int raw64;
    int kp, kn;
    float* zt;              // [rows][kn]
    float* kept;            // KEEP: z itself, in panels as dz
    // outputs
    uint16_t* out;          // dz (panels), dhead [n = v][ld_out], dx [row][ld_out] or NULL: the sums are not complete
    long long ld_out;
    float* acc;             // dx sums [splits][rows that count][ld_acc]
    long long ld_acc;
    int plan_steps;         // dx: the steps of a whole piece, which its splits go by
    int add;                // dx: onto the sums so far
    const float* scale;     // dhead, dx: the factor taken out of dz
};

// About the time (us) that a workgroup of each product and tile takes for a step of 64 k (more with more of the CUs at work:
// the memory and the power are shared) and for its beginning and end, as many workgroups at once as fit the CUs. Fitted to the
// kernels' times at eight shapes of 73 to 8192 rows, 584 to 4096 values and 2898 to 94639 tokens, most within 15 %; what
// decides between two tiles is mostly how many rounds they take.
// (KEEP: the statistics, z kept instead of the entries' taken; DZ1: tokens, their own logit's 1 taken off there)
enum Epi { EPI_STATS, EPI_KEEP, EPI_DZ, EPI_DZ1, EPI_DHEAD, EPI_DX };
__host__ __device__ constexpr Pace pace(int epi, int bm, int bn, int wk) {
    const bool dx = epi == EPI_DX, dhead = epi == EPI_DHEAD;
    if (wk == 2) return Pace{CUS, dx ? 0.23f : 0.28f, 0.f, dx ? 4.5f : 2.8f};  // 64 x 64, two groups of wavefronts
    if (bm == 64) return Pace{2 * CUS, 0.32f, 0.16f, 3.5f};
    if (bn == 64) return Pace{2 * CUS, 0.6f, 0.9f, 8.f};
    if (bm == 256) return Pace{CUS, dx ? 1.05f : dhead ? 1.15f : 1.2f, 0.45f, dx ? 13.f : dhead ? 8.f : 12.f};
    return Pace{2 * CUS, dx ? 0.75f : dhead ? 0.6f : 0.62f, dhead ? 0.3f : 0.35f, dx ? 7.f : dhead ? 4.f : 8.f};
}

// dx's splits of its long sum, for one or two rounds of workgroups: their sums' way back through memory costs a launch and
// about 3.5 TB/s. The rows that count are known on the device alone, so every workgroup finds the splits for itself.
constexpr int ROUNDS = 2;
__host__ __device__ inline int dx_splits(const Pace& p, int tiles, int steps, int tile_bytes, float* us = nullptr) {
    int best = 1;
    float least = tiled_us(p, tiles, steps);
    for (int r = 1; r <= ROUNDS; ++r) {
        int s = r * p.at_once / (tiles > 0 ? tiles : 1);
        if (s > steps / 4) s = steps / 4;
        if (s < 2) continue;
        const float t = tiled_us(p, tiles * s, ((steps + s - 1) / s + 1) & ~1) + 4.f + (float)tiles * (float)s * (float)tile_bytes * 0.28e-6f;
        if (t < least) least = t, best = s;
    }
    if (us) *us = least;
    return best;
}

// D[m][n] in tiles of BM x BN, a wavefront BM / WM x BN / WN of 32x32x16 matrix instructions; NS stages of BK k in LDS, filled
// straight from memory.
// - 256 x 256 by 8 wavefronts: the largest that the registers hold, so the fewest bytes into a CU for each operation. Its
//   operands along k (z) come in steps of 64, a whole 128-byte line of a row, two stages; those across (dhead, dx) in four
//   stages of 32 k, which leaves the loads three steps: dhead 1270 -> 1305 TFLOP/s, z the other way round (1210 to 1284 in two
//   stages of 64, 1194 to 1241 in four of 32). 4 wavefronts of 128 x 128 read a third less LDS, but nothing runs beside them
//   (1190 to 1270); 256 x 128 twice a CU 950 to 1060; fragments read a step ahead or wave priorities change nothing.
//   (8192 x 4096 x 16384.)
// - 128 x 128 and 64 x 64, twice a CU, where larger tiles would leave CUs idle (choose); 64 x 64 also by two groups of
//   wavefronts that split K, where there is at most one tile a CU.
// - 128 x 64 for up to 64 rows of x: the head is read once, at the memory's rate.
// The epilogues' bf16 leave through LDS in whole runs of a row (with that and dz in panels dhead of 64128 tokens went from 4840
// to 4593 us).
template <int BM, int BN, int WM, int WN, int WK, int NS, int BK, bool AT, bool BT, int EPI>
__global__ __launch_bounds__(64 * WM * WN * WK) void hl_gemm(const Gemm a) {
    constexpr int NW = WM * WN, NT = 64 * NW, TM = BM / WM, TN = BN / WN, MI = TM / 32, NI = TN / 32;
    constexpr int CA = BM * BK / 8, CH = CA + BN * BK / 8;  // chunks of A, a stage
    constexpr int NL = CH / NT;        // loads a lane and stage
    static_assert(NS >= 1 && NS <= 4, "one to four stages");
    constexpr int C1 = NS > 1 ? CH * WK : 1, C2 = NS > 2 ? CH * WK : 1, C3 = NS > 3 ? CH * WK : 1;
    // (an array each, named where it is used: a read waits for the loads to every array that the compiler cannot rule out)
    __shared__ uint4 s0[CH * WK], s1[C1], s2[C2], s3[C3];
    constexpr bool STATS = EPI == EPI_STATS || EPI == EPI_KEEP;
    __shared__ f32x2 stat[STATS ? WM : 1][STATS ? BN : 1];
    // WK groups of wavefronts, each a share of K in stages of its own, all with the same barriers; tid within the group
    const int group = WK == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / NT), tid = threadIdx.x - group * NT;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), mine = group * CH;
    const int wm = wave / WN, wn = wave % WN;
    const int live = a.live ? *a.live : (EPI == EPI_DHEAD ? a.k : a.n);
    // (dx: the tiles of the rows that count, split as many ways as fill the CUs)
    const int tn = EPI == EPI_DX ? (live + BN - 1) / BN : a.tn;
    const int splits = EPI == EPI_DX ? dx_splits(pace(EPI, BM, BN, WK), a.tm * tn, a.plan_steps, BM * BN * 4) : 1;
    int mt, nt, split;
    if (!tile_of(a.tm, tn, splits, mt, nt, split)) return;
    const int m0 = mt * BM, n0 = nt * BN;
    const int n_end = EPI == EPI_DHEAD ? a.n : live, k_end = EPI == EPI_DHEAD ? live : a.k;
    const int nb = EPI == EPI_DHEAD ? a.nb : n_end, ka = EPI == EPI_DHEAD ? live : a.ka;
    if (n0 >= n_end) return;
    // (a split's steps are whole rounds of the stages: the next split's are not its own)
    constexpr int ROUND = NS * WK;
    const int all = (k_end + BK - 1) / BK, per = ((all + splits - 1) / splits + ROUND - 1) / ROUND * ROUND, step0 = split * per;
    const int steps = EPI == EPI_DHEAD && n0 >= nb ? 0 : min(per, all - step0);
    const int rounds = ((steps + WK - 1) / WK + NS - 1) / NS;  // (of the stages)

    Tile<BM, AT, NT, BK> ta;
    Tile<BN, BT, NT, BK> tb;
    constexpr bool X_A = EPI == EPI_DHEAD, X_B = STATS || EPI == EPI_DZ || EPI == EPI_DZ1;
    const bool whole = (X_A || X_B) && a.whole && live == a.rows;
    const uint16_t *A = X_A && whole ? a.whole : a.A, *B = X_B && whole ? a.whole : a.B;
    const long long la = X_A && whole ? a.ldx : a.lda, lb = X_B && whole ? a.ldx : a.ldb;
    const int lda = (int)la, ldb = (int)lb, ra = a.m - m0, rb = nb - n0;  // (rows past the tile's)
    ta.init(tid, lda, ra);
    tb.init(tid, ldb, rb);
    // where the next step to be loaded lies, and the k left from it on
    int k = (step0 + group * rounds * NS) * BK;
    const uint16_t* pa = A + (AT ? k * la + m0 : m0 * la + k);
    const uint16_t* pb = EPI == EPI_DHEAD ? B + (n0 >> 8) * a.panel + (n0 & 255) + k * lb
                         : EPI == EPI_DX  ? B + (k >> 8) * a.panel + (k & 255) + n0 * lb
                                          : B + n0 * lb + k;
    const long long next_panel = a.panel - 256 + BK;
    __amdgpu_buffer_rsrc_t from_a, from_b;
    int left_a, left_b;
    auto next = [&] {  // the next step to be loaded
        left_a = (AT ? ka : k_end) - k, left_b = k_end - k;
        from_a = Tile<BM, AT, NT, BK>::source(pa, lda, AT ? ra : min(BM, ra), left_a);
        from_b = Tile<BN, BT, NT, BK>::source(pb, ldb, BT ? rb : min(BN, rb), left_b);
        pa += AT ? BK * la : BK;
        pb += BT ? BK * lb : EPI == EPI_DX && (k & 255) == 256 - BK ? next_panel : BK;
        k += BK;
    };
    constexpr int NA = CA / NT;
    auto load = [&](int i0, int i1, uint4* b) {  // its loads i0 .. i1 - 1 of NL
#pragma unroll
        for (int i = i0; i < i1; ++i) {
            if (i < NA) ta.load(i, from_a, left_a, b + mine, tid);
            else tb.load(i - NA, from_b, left_b, b + (mine + CA), tid);
        }
    };
    constexpr int CN = MI * NI > 1 ? 1 : 2;  // sums of one tile: two in turn, which need not wait for each other
    f32x16 acc[MI][NI], odd;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        odd[e] = 0.f;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j][e] = 0.f;
    }
    // A step's sums from one stage, the loads of a later step to another, with three stages and more between the sums: a wavefront that
    // issues all of its loads at once stands still until the memory pipeline has taken them, and all do after the barrier.
    // (With two they would land too late for the next step.)
    auto sum = [&](const uint4* b, uint4* to) {
        constexpr int U = BK / 16;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint4 fa[MI], fb[NI];
#pragma unroll
            for (int j = 0; j < NI; ++j) fb[j] = Tile<BN, BT, NT, BK>::frag(b, mine + CA, wn * TN + 32 * j, u, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i) fa[i] = Tile<BM, AT, NT, BK>::frag(b, mine, wm * TM + 32 * i, u, lane);
            if constexpr (NS >= 3) load(u * NL / U, (u + 1) * NL / U, to);
            else if (NS == 2 && u == 0) load(0, NL, to);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    f32x16& to = CN == 2 && (u & 1) ? odd : acc[i][j];
                    to = mfma32(fa[i], fb[j], to);
                }
            // (one u's fragments at a time: the registers hold no more; a small tile reads them all at once)
            if constexpr (MI * NI > 1) __builtin_amdgcn_sched_barrier(0);
        }
    };
    // (whole rounds of the stages: steps past the last are zeros, as are the loads past the end into stages that nothing
    // reads. A last step of its own behind a branch would have the compiler copy every accumulator.)
    auto step = [&](uint4* to, const uint4* from) {
        step_barrier<NS >= 3 ? (NS - 2) * NL : 0>();
        next();
        sum(from, to);
    };
    auto first = [&](uint4* to) {
        next();
        load(0, NL, to);
    };
    if (steps > 0) {
        first(s0);
        if constexpr (NS >= 3) first(s1);
        if constexpr (NS >= 4) first(s2);
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
        } else {
            step(s3, s0);
            step(s0, s1);
            step(s1, s2);
            step(s2, s3);
        }
    }
    step_barrier<0>();  // (the last loads landed: they write this workgroup's LDS)
    if constexpr (CN == 2) acc[0][0] += odd;
    if constexpr (WK == 2) {  // the second group's sums to the first
        static_assert(WK == 1 || (MI * NI == 1 && NW * 256 <= C1), "their sums fit a stage");
        f32x4* at = reinterpret_cast<f32x4*>(s1) + wave * 256 + lane;
        if (group) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
                at[64 * g] = f32x4{acc[0][0][4 * g], acc[0][0][4 * g + 1], acc[0][0][4 * g + 2], acc[0][0][4 * g + 3]};
        }
        step_barrier<0>();
        if (!group) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 v = at[64 * g];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[0][0][4 * g + e] += v[e];
            }
        }
    }
    const bool second = WK == 2 && group;  // (it has nothing left to do but the statistics' barrier)

    // lane: columns n = n0 + wn TN + 32 j + lane % 32, rows m0 + wm TM + 32 i + 8 g + 4 (lane / 32) + 0 .. 3 in words 4 g ..
    const int r = lane & 31, h = lane >> 5;
    const int mw = m0 + wm * TM;
    // the wavefront's own part of the stages: 32 columns of its TM rows in float32
    constexpr int PER = NS == 1 || WK > 1 ? NW : NS == 4 ? (NW + 3) / 4 : (NW + 1) / 2;
    static_assert(PER * 8 * TM <= CH * WK, "a wavefront's sums of 32 columns fit its part of a stage");
    uint4* region = s0 + (wave % PER) * 8 * TM;
    if constexpr (PER < NW) {
        const int at = wave / PER;
        if constexpr (NS == 4) region = (at == 0 ? s0 : at == 1 ? s1 : at == 2 ? s2 : s3) + (wave % PER) * 8 * TM;
        else region = (at ? s1 : s0) + (wave % PER) * 8 * TM;
    }
    // 32 columns in bf16, 4 rows of column r at 8-byte unit q: to whole runs of a column's rows in memory
    uint2* const half = reinterpret_cast<uint2*>(region);
    constexpr int C16 = TM / 8, SWZ = C16 < 16 ? C16 - 1 : 15;  // 16-byte chunks a column; their turn by column
    auto put = [&](int q, uint2 v) { half[(r * C16 + ((q >> 1) ^ (r & SWZ))) * 2 + (q & 1)] = v; };
    auto store = [&](auto&& at, int cols, int rows) {  // at(c, row): column c's place for 8 of its rows from `row` on
        __builtin_amdgcn_wave_barrier();
        constexpr int PC = 64 / C16;  // columns a turn
#pragma unroll
        for (int t = 0; t < 32 / PC; ++t) {
            const int c = t * PC + lane / C16, q = lane % C16;
            if (c < cols && 8 * q < rows) *reinterpret_cast<uint4*>(at(c, 8 * q)) = region[c * C16 + (q ^ (c & SWZ))];
        }
        __builtin_amdgcn_wave_barrier();
    };
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        if (second) continue;
        const int nj = n0 + wn * TN + 32 * j, n = nj + r;
        if constexpr (STATS) {
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
            // (no sum: nothing there; a NaN with nothing else beside it is something)
            if (h == 0) stat[wm][wn * TN + 32 * j + r] = f32x2{total == 0.f ? -INFINITY : base, total};
            // the entries that lie here: the wavefront's sums of these 32 rows through its own LDS
            f32x4* mine = reinterpret_cast<f32x4*>(region);
            const int here = min(TM, left), w = 1 << a.kp;
            auto lay = [&] {
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        mine[r * (TM / 4) + ((8 * i + 2 * g + h) ^ (r & 7))] =
                            f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                __builtin_amdgcn_wave_barrier();
            };
            auto take = [&](int t, int kk, int d) {  // column t's entry kk at this wavefront's row d
                const long long row = a.idx ? a.idx[nj + t] : nj + t;
                a.zt[row * a.kn + kk] = mine[t * (TM / 4) + ((d >> 2) ^ (t & 7))][d & 3];
            };
            if constexpr (EPI == EPI_KEEP) {  // (the entries are read from it)
                lay();
                constexpr int C4 = TM / 4, PC = 64 / C4;  // 16-byte chunks a column, columns a turn
                float* o = a.kept + (mw >> 8) * a.panel + (long long)nj * 256 + (mw & 255);
#pragma unroll 2
                for (int t = 0; t < 32 / PC; ++t) {
                    const int c = t * PC + lane / C4, q = lane % C4;
                    if (nj + c < n_end)  // (read once, much later)
                        __builtin_nontemporal_store(mine[c * C4 + (q ^ (c & 7))], reinterpret_cast<f32x4*>(o + c * 256 + 4 * q));
                }
            } else if (a.kp < 2) {
                const int t = lane >> a.kp;
                int d = -1;
                if (t < 32 && nj + t < n_end) {
                    if (a.raw) {
                        const long long id = a.raw64 ? reinterpret_cast<const long long*>(a.raw)[nj + t]
                                                     : reinterpret_cast<const int*>(a.raw)[nj + t];
                        d = id >= mw && id < mw + here ? (int)(id - mw) : -1;
                    } else {
                        d = a.ids[((long long)nj << a.kp) + lane] - mw;
                    }
                }
                const bool hit = (unsigned)d < (unsigned)here && here > 0;
                if (__ballot(hit)) {
                    lay();
                    if (hit) take(t, lane & (w - 1), d);
                }
            } else {  // four a load, eight loads at once
                const int count = 8 << a.kp;
                const int4* at = reinterpret_cast<const int4*>(a.ids + ((long long)nj << a.kp));
                int4 v[8];
                bool hit = false;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const int e = lane + 64 * q;
                    v[q] = e < count && nj + (4 * e >> a.kp) < n_end ? at[e] : make_int4(-1, -1, -1, -1);
                }
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    v[q].x -= mw, v[q].y -= mw, v[q].z -= mw, v[q].w -= mw;
                    hit |= (unsigned)v[q].x < (unsigned)here || (unsigned)v[q].y < (unsigned)here ||
                           (unsigned)v[q].z < (unsigned)here || (unsigned)v[q].w < (unsigned)here;
                }
                if (here > 0 && __ballot(hit)) {
                    lay();
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const int e = 4 * (lane + 64 * q), t = e >> a.kp, kk = e & (w - 1);
                        if ((unsigned)v[q].x < (unsigned)here) take(t, kk, v[q].x);
                        if ((unsigned)v[q].y < (unsigned)here) take(t, kk + 1, v[q].y);
                        if ((unsigned)v[q].z < (unsigned)here) take(t, kk + 2, v[q].z);
                        if ((unsigned)v[q].w < (unsigned)here) take(t, kk + 3, v[q].w);
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        } else if constexpr (EPI == EPI_DZ || EPI == EPI_DZ1) {
            const long long row = n < n_end ? a.idx[n] : 0;
            const float top = *a.top, l2 = n < n_end ? a.lse[row] * LOG2E : 0.f, gr = a.g && n < n_end ? a.g[row] : 1.f;
            const float gs = gr / top;
            const int left = a.m - mw;
            const int own = EPI == EPI_DZ1 && n < n_end ? a.ids[n] - a.v0 - mw - 4 * h : -1;  // (the token's own logit)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][4 * g + e], a.sc, -l2));
                        if (EPI == EPI_DZ1 && own == 32 * i + 8 * g + e) p[e] -= 1.f;
                        p[e] *= gs;
                    }
                    if (left < TM) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (32 * i + 8 * g + 4 * h + e >= left) p[e] = 0.f;
                    }
                    put(8 * i + 2 * g + h, make_uint2(cvt2(p[0], p[1]), cvt2(p[2], p[3])));
                }
            uint16_t* o = a.out + (mw >> 8) * a.panel + (long long)nj * 256 + (mw & 255);
            store([&](int c, int row) { return o + c * 256 + row; }, n_end - nj, TM);
        } else if constexpr (EPI == EPI_DHEAD) {
            const float s = *a.scale;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    put(8 * i + 2 * g + h, make_uint2(cvt2(acc[i][j][4 * g] * s, acc[i][j][4 * g + 1] * s),
                                                      cvt2(acc[i][j][4 * g + 2] * s, acc[i][j][4 * g + 3] * s)));
            uint16_t* o = a.out + nj * a.ld_out + mw;
            store([&](int c, int row) { return o + c * a.ld_out + row; }, n_end - nj, a.m - mw);
        } else if (a.out != nullptr && splits == 1) {  // the last sums: dx itself
            const float s = *a.scale;
            const long long at = n * a.ld_acc + mw;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * i + 8 * g + 4 * h;
                    f32x4 v = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                    if (a.add && n < n_end && mw + d < a.m) v += *reinterpret_cast<const f32x4*>(a.acc + at + d);
                    put(8 * i + 2 * g + h, make_uint2(cvt2(v[0] * s, v[1] * s), cvt2(v[2] * s, v[3] * s)));
                }
            store([&](int c, int row) { return a.out + a.idx[nj + c] * a.ld_out + mw + row; }, n_end - nj, a.m - mw);
        } else {
            if (n >= n_end) continue;
            float* o = a.acc + ((long long)split * live + n) * a.ld_acc + mw;
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
    if constexpr (STATS) {  // the wavefronts' rows of a column together
        __syncthreads();
        if (wm == 0 && h == 0 && !second) {
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const int c = wn * TN + 32 * j + r;
                float m = stat[0][c][0], s = stat[0][c][1];
#pragma unroll
                for (int i = 1; i < WM; ++i) join(m, s, stat[i][c][0], stat[i][c][1]);
                if (n0 + c < n_end) a.part[mt * a.ld_part + n0 + c] = f32x2{m, s};
            }
        }
    }
}

// --- entries, rows that count, merges -----------------------------------------------------------------------------------

struct Prep {
    dr_head_loss a;
    int kp;         // log2 of the entries' stride
    int* ids;       // [rows][1 << kp], -1: not held
    int* idc;       // [rows that count][1 << kp]
    float* q;       // [rows][1 << kp] (a teacher's)
    float* ent;     // [rows] sum q log q (a teacher's)
    uint8_t* held;  // [rows] whether the row counts
    int* idx;       // [rows] row that counts -> row
    int* pos;       // [rows] row -> row that counts, -1: left out
    int* live;      // rows that count
    float* top;     // the factor taken out of dz, the largest |g| of them, and that over T
    uint16_t* xc;   // [rows that count][dim]
    uint16_t* dx;   // whose rows left out get zeros, or NULL
};

__device__ __forceinline__ int entry_id(const dr_head_loss& a, int row, int j) {
    const long long at = (long long)row * a.ld_ids + j;
    const long long id = a.ids64 ? reinterpret_cast<const long long*>(a.ids)[at] : reinterpret_cast<const int*>(a.ids)[at];
    return id >= 0 && id < a.valid ? (int)id : -1;
}

// A row's softmax over w lanes, of entries v (-inf and id -1: none), and its sum of q log q. (The temperature after the
// difference: the type's lowest value, at a temperature below 1, is still no empty slot.)
__device__ __forceinline__ void teacher(float v, int id, int w, float temperature, float& q, float& ent) {
    float top = v;
    for (int o = w >> 1; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float d = id < 0 ? 0.f : (v - top) / temperature;
    const float x = id < 0 ? 0.f : __expf(d);
    float total = x;
    for (int o = w >> 1; o; o >>= 1) total += __shfl_xor(total, o);
    q = id < 0 ? 0.f : x / total;
    ent = q == 0.f ? 0.f : q * (d - __logf(total));
    for (int o = w >> 1; o; o >>= 1) ent += __shfl_xor(ent, o);
}

// entry e of all rows' (row e >> kp; the lanes of a row are neighbours): id, q, the row's sum; whether the row counts
__device__ __forceinline__ bool entries_of(const Prep& p, int e, int rows) {
    const int row = e >> p.kp, w = 1 << p.kp, j = e & (w - 1);
    const bool in = row < rows && j < p.a.k;
    int id = in ? entry_id(p.a, row, j) : -1;
    if (p.a.vals) {
        float v = in ? p.a.vals[(long long)row * p.a.ld_vals + j] : -INFINITY;
        if (v == -INFINITY) id = -1;
        if (id < 0) v = -INFINITY;
        float q, ent;
        teacher(v, id, w, p.a.temperature, q, ent);
        if (row < rows) {
            p.q[e] = q;
            if (j == 0) p.ent[row] = ent;
        }
    }
    const unsigned long long held = __ballot(id >= 0);
    const int lane = threadIdx.x & 63;
    const unsigned long long mine = w == 64 ? held : (held >> (lane & ~(w - 1))) & ((1ull << w) - 1);
    if (row < rows) {
        p.ids[e] = id;
        if (j == 0) p.held[row] = mine != 0;
    }
    return mine != 0;
}

__global__ __launch_bounds__(256) void hl_entries(const Prep p) { entries_of(p, blockIdx.x * 256 + threadIdx.x, p.a.rows); }

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

constexpr int GROWS = 4;     // rows a workgroup of hl_gather, one a wavefront
constexpr int MANY = 32768;  // rows past which it takes 64, and looks through the flags a sixteenth as often (2^18 rows x 64
                             // against 300 tokens, the whole call: 1.97 ms, 2.50 by 4; 2^20 8.97 and 17.0; 2^15 the same)
constexpr int FEW = 2048;    // entries that every workgroup looks through itself

// the factor taken out of dz, of the rows' weights that count (positive, finite) the largest; weights so far apart that the
// smallest over the largest would near the smallest float32, or none (all 0, or infinite: 0 times those is a NaN): as they are
__device__ __forceinline__ float factor(float top, float low) { return top > 0.f && low > top * 0x1p-40f ? top : 1.f; }


// The rows that count, one after another: each workgroup finds the place of its own from the flags of all rows before
// (16 a load), so that nothing waits for anything; one more finds how many there are and the largest |g|. Where every row
// counts none is copied. OWN: the entries too, of few rows, every workgroup looking through all of the ids for the flags (a
// launch less).
template <bool OWN, int GR>
__global__ __launch_bounds__(256) void hl_gather(const Prep p) {
    __shared__ int sums[4];
    __shared__ float tops[4], lows[4];
    __shared__ int rows[GR];
    __shared__ uint4 flag4[OWN ? FEW / 16 : 1];
    uint8_t* const flags = reinterpret_cast<uint8_t*>(flag4);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = p.a.rows;
    const bool last = blockIdx.x == gridDim.x - 1;
    const int r0 = last ? n : blockIdx.x * GR;
    const uint8_t* held = p.held;
    if constexpr (OWN) {
        for (int i = tid; i < FEW / 16; i += 256) flag4[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        const int upto = n << p.kp, w = 1 << p.kp;
        for (int e = tid; e < upto; e += 256) {
            const int row = e >> p.kp, j = e & (w - 1);
            if (j < p.a.k && entry_id(p.a, row, j) >= 0 && (!p.a.vals || p.a.vals[(long long)row * p.a.ld_vals + j] != -INFINITY))
                flags[row] = 1;
        }
        __syncthreads();
        held = flags;
        if (!last)
            for (int e = tid; e < GR << p.kp; e += 256) entries_of(p, (r0 << p.kp) + e, min(n, r0 + GR));
    }
    int c = 0, out = 0;  // rows that count before this workgroup's; rows left out, all of them
    for (int i = tid; i < n / 16; i += 256) {
        const uint4 f = reinterpret_cast<const uint4*>(held)[i];
        const int here = __popc(f.x) + __popc(f.y) + __popc(f.z) + __popc(f.w);
        c += i < r0 / 16 ? here : 0;
        out += 16 - here;
    }
    if (tid < r0 % 16) c += held[r0 / 16 * 16 + tid];
    if (tid < n % 16) out += 1 - held[n / 16 * 16 + tid];
    c = wave_sum(c);
    const bool some = __syncthreads_or(out != 0);
    float top = 0.f, low = INFINITY;
    if (last && p.a.g) {
#pragma unroll 8
        for (int r = tid; r < n; r += 256) {
            const float g = fabsf(p.a.g[r]);
            const bool in = held[r] && g > 0.f && g < INFINITY;  // (an infinite weight stays in its row)
            top = fmaxf(top, in ? g : 0.f);
            low = fminf(low, in ? g : INFINITY);
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o)), low = fminf(low, __shfl_xor(low, o));
    if (lane == 0) sums[wave] = c, tops[wave] = top, lows[wave] = low;
    __syncthreads();
    const int before = sums[0] + sums[1] + sums[2] + sums[3];
    if (last) {
        if (tid == 0) {
            top = p.a.g ? fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) : 1.f;
            low = fminf(fminf(lows[0], lows[1]), fminf(lows[2], lows[3]));
            if (p.a.g) top = factor(top, low);
            *p.live = before;
            p.top[0] = top;
            p.top[1] = top / p.a.temperature;
        }
        return;
    }
    if (wave == 0) {
        const int r = r0 + lane;
        const bool on = lane < GR && r < n && held[r] != 0;
        const unsigned long long b = __ballot(on);
        const int at = before + __popcll(b & ((1ull << lane) - 1));
        if (lane < GR) rows[lane] = on ? at : -1;
        if (lane < GR && r < n) p.pos[r] = on ? at : -1;
        if (on) p.idx[at] = r;
    }
    __syncthreads();  // (OWN: this workgroup's entries are written too)
    for (int i = wave; i < GR; i += 4) {
        const int at = rows[i];
        if (at < 0) {
            if (p.dx && r0 + i < n)  // (a row left out)
                for (int q = lane; q < p.a.dim / 4; q += 64)
                    *reinterpret_cast<uint2*>(p.dx + (r0 + i) * p.a.ld_dx + 4 * q) = make_uint2(0u, 0u);
            continue;
        }
        if (lane < 1 << p.kp) p.idc[((long long)at << p.kp) + lane] = p.ids[((long long)(r0 + i) << p.kp) + lane];
        if (!some) continue;  // (every row counts: x is read where it lies)
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.a.x) + (r0 + i) * p.a.ldx);
        uint4* dst = reinterpret_cast<uint4*>(p.xc + (long long)at * p.a.dim);
#pragma unroll 8
        for (int q = lane; q < p.a.dim / 8; q += 64) dst[q] = src[q];
    }
}

struct Merge {
    const f32x2* part;
    long long ld;
    int parts, rows, k, kp;
    const int* pos;       // NULL: a row's own place
    const uint8_t* held;  // NULL: tokens as they came
    const void* raw;
    int raw64, valid;
    const int* ids;
    const float *q, *ent;
    float inv_t;
    float *loss, *lse, *zt;
    const float* kept;    // z itself, the entries' not taken yet; or NULL
    long long panel;
};

// a row's tiles' maxima and sums, one slice of SL: from `sl` on
template <int SL>
__device__ __forceinline__ void slice_of(const f32x2* at, long long ld, int parts, int sl, float& m, float& s) {
    int i = sl;
    for (; i + 3 * SL < parts; i += 4 * SL) {
        f32x2 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = at[(i + u * SL) * ld];
#pragma unroll
        for (int u = 0; u < 4; ++u) join(m, s, v[u][0], v[u][1]);
    }
    for (; i < parts; i += SL) {
        const f32x2 v = at[i * ld];
        join(m, s, v[0], v[1]);
    }
}
__device__ __forceinline__ void wave_join(float& m, float& s) {
#pragma unroll
    for (int o = 32; o; o >>= 1) join(m, s, __shfl_xor(m, o), __shfl_xor(s, o));
}

// a row's tiles' maxima and sums joined, then lse and loss: TB rows a workgroup, SL slices of each (16 and 64: 4096 rows of 125
// tiles and 64 kept entries 15.1 us, by 32 and 32 22.1; 8192 of 501 11.9 and 11.0)
template <int TB, int SL>
__global__ __launch_bounds__(TB* SL) void hl_merge(const Merge p) {
    __shared__ float ms[TB * SL], ss[TB * SL];
    const int tid = threadIdx.x, t = tid % TB, sl = tid / TB, row = blockIdx.x * TB + t;
    bool in = false;
    if (row < p.rows) {
        if (p.held) {
            in = p.held[row];
        } else {
            const long long id = p.raw64 ? reinterpret_cast<const long long*>(p.raw)[row] : reinterpret_cast<const int*>(p.raw)[row];
            in = id >= 0 && id < p.valid;
        }
    }
    const int n = !in ? -1 : p.pos ? p.pos[row] : row;
    float m = -INFINITY, s = 0.f;
    if (n >= 0) slice_of<SL>(p.part + n, p.ld, p.parts, sl, m, s);
    if constexpr (TB == 1) wave_join(m, s);  // (a row's slices are whole wavefronts)
    constexpr int LEFT = TB == 1 ? SL / 64 : SL;  // slices that are left
    if (TB > 1 || (tid & 63) == 0) ms[TB == 1 ? tid >> 6 : tid] = m, ss[TB == 1 ? tid >> 6 : tid] = s;
    __syncthreads();
    if constexpr (TB == 1) m = ms[tid % LEFT], s = ss[tid % LEFT];
#pragma unroll
    for (int o = LEFT / 2; o; o >>= 1) {
        if (sl < o) {
            join(m, s, ms[tid + o * TB], ss[tid + o * TB]);
            ms[tid] = m;
            ss[tid] = s;
        }
        __syncthreads();
    }
    const float lse = in ? (ms[t] + __builtin_amdgcn_logf(ss[t])) * LN2 : 0.f;
    __syncthreads();
    float c = 0.f;
    float* z = p.zt + (long long)row * p.k;
    if (p.kept && in) {  // (each read by the lane that took it)
        for (int j = sl; j < p.k; j += SL) {
            const int id = p.ids[((long long)row << p.kp) + j];
            z[j] = id < 0 ? 0.f : p.kept[(id >> 8) * p.panel + (long long)n * 256 + (id & 255)];
        }
    }
    if (p.q) {
        for (int j = sl; j < p.k && row < p.rows; j += SL) {
            const long long e = ((long long)row << p.kp) + j;
            if (p.ids[e] < 0) z[j] = 0.f;
            else if (const float q = p.q[e]; q != 0.f) c += q * (lse - z[j] * p.inv_t);
        }
    } else if (sl == 0 && row < p.rows) {
        if (in) c = lse - z[0];
        else z[0] = 0.f;
    }
    if (p.q) {
        ms[tid] = c;
        __syncthreads();
        for (int i = 1; sl == 0 && i < SL && i < p.k; ++i) c += ms[i * TB + t];
    }
    if (sl || row >= p.rows) return;
    p.lse[row] = lse;
    p.loss[row] = in ? (p.q ? p.ent[row] + c : c) : 0.f;
}

struct Dz {
    const int *live, *idx, *ids;  // (ids: tokens' own, of the rows that count, or NULL)
    const float *z, *lse, *g, *top;
    uint16_t* dz;
    long long panel;
    int valid;
    float sc;
};

// dz from z as the loss left it: a wavefront's rows of one panel, 1 KB read and 512 bytes written each (1842 rows against 128256
// tokens: 239 us, 5.9 TB/s)
constexpr int DZ_ROWS = 8;  // a wavefront, asked for at once
__global__ __launch_bounds__(256) void hl_dz(const Dz p) {
    const int live = *p.live, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = (blockIdx.y * 4 + wave) * DZ_ROWS, v0 = blockIdx.x * 256 + 4 * lane;
    if (n0 >= live) return;
    const float top = *p.top;
    const long long at = blockIdx.x * p.panel + (long long)n0 * 256 + 4 * lane;
    f32x4 z[DZ_ROWS];
#pragma unroll
    for (int i = 0; i < DZ_ROWS; ++i) z[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p.z + at + min(i, live - 1 - n0) * 256));
#pragma unroll
    for (int i = 0; i < DZ_ROWS; ++i) {
        const int n = n0 + i;
        if (n >= live) break;
        const int row = p.idx[n], own = p.ids ? p.ids[n] - v0 : -1;
        const float l2 = p.lse[row] * LOG2E, gr = p.g ? p.g[row] : 1.f, gs = gr / top;
        float d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            d[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i][e], p.sc, -l2));
            if (own == e) d[e] -= 1.f;
            d[e] = v0 + e < p.valid ? d[e] * gs : 0.f;
        }
        *reinterpret_cast<uint2*>(p.dz + at + i * 256) = make_uint2(cvt2(d[0], d[1]), cvt2(d[2], d[3]));
    }
}

struct Few {
    dr_head_loss a;
    int kp, parts;
    const f32x2* part;
    long long ld;
    const float* kept;
    uint16_t* dz;
    long long panel, dz_panel;
    float sc, inv_t;
    int *idx, *live;
    float* top;
    uint16_t *xc, *dx;
    int fine;  // what dz's rounding leaves, rounded too, as so many rows more (of x as well)
};

// a row's tiles' maxima and sums joined, in hl_merge<1, 256>'s order: one part a row for hl_few
__global__ __launch_bounds__(256) void hl_join(const f32x2* part, long long ld, int parts, f32x2* out) {
    __shared__ float ms[4], ss[4];
    const int tid = threadIdx.x;
    float m = -INFINITY, s = 0.f;
    slice_of<256>(part + blockIdx.x, ld, parts, tid, m, s);
    wave_join(m, s);
    if ((tid & 63) == 0) ms[tid >> 6] = m, ss[tid >> 6] = s;
    __syncthreads();
    if (tid) return;
    join(ms[0], ss[0], ms[2], ss[2]);
    join(ms[1], ss[1], ms[3], ss[3]);
    join(ms[0], ss[0], ms[1], ss[1]);
    out[blockIdx.x] = f32x2{ms[0], ss[0]};
}

// Few rows (one a wavefront and panel), from z as the loss left it: what hl_gather, hl_merge, hl_dz and hl_fix do, in one launch.
// Every wavefront joins its row's tiles for itself and counts the rows that count from all of the ids; the first panel's write
// what there is one of.
constexpr int FEW_ROWS = 256, FEW_PARTS = 512, FEW_IDS = 4096;
// (every panel's wavefronts join the parts again: 64 rows x 1024 against 16384 tokens, 256 parts, 42.2 us, 49.0 in launches of
// their own; against 32768 65.4 and 64.7; 128 rows against 8192 37.7 and 45.7, 16384 57.4 and 56.4)
constexpr int FEW_JOINS = 16384;
__host__ __device__ inline bool few_parts(int rows, int parts) {
    return rows <= FEW_ROWS && parts <= FEW_PARTS && rows * parts <= FEW_JOINS;
}
__global__ __launch_bounds__(256) void hl_few(const Few p) {
    __shared__ uint32_t flags[FEW_ROWS];
    static_assert(FEW_ROWS == 256, "a flag a lane");
    __shared__ f32x4 taken[4][64];  // the entries' q in the wavefront's panel
    const dr_head_loss& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), w = 1 << p.kp;
    const int r = blockIdx.y * 4 + wave, row = min(r, a.rows - 1), v0 = blockIdx.x * 256;
    const bool first = blockIdx.x == 0;
    const f32x4 z = *reinterpret_cast<const f32x4*>(p.kept + blockIdx.x * p.panel + row * 256 + 4 * lane);
    float m = -INFINITY, s = 0.f;
    slice_of<64>(p.part + row, p.ld, p.parts, lane, m, s);
    flags[tid] = 0;
    taken[wave][lane] = f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    for (int e = tid; e < a.rows << p.kp; e += 256) {
        const int er = e >> p.kp, j = e & (w - 1);
        if (j < a.k && entry_id(a, er, j) >= 0 && (!a.vals || a.vals[(long long)er * a.ld_vals + j] != -INFINITY)) flags[er] = 1;
    }
    __syncthreads();
    int live = 0, at = 0;  // the rows that count; those before this one
    bool in = false;
    float top = 0.f, low = INFINITY;
#pragma unroll
    for (int i = 0; i < FEW_ROWS / 64; ++i) {
        const bool mine = flags[64 * i + lane] != 0;
        const unsigned long long on = __ballot(mine);
        const int here = row - 64 * i;
        live += __popcll(on);
        at += here >= 64 ? __popcll(on) : here > 0 ? __popcll(on & ((1ull << here) - 1)) : 0;
        in |= here >= 0 && here < 64 && (on >> (here & 63) & 1);
        const float g = a.g && mine ? fabsf(a.g[64 * i + lane]) : 0.f;
        if (g > 0.f && g < INFINITY) top = fmaxf(top, g), low = fminf(low, g);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o)), low = fminf(low, __shfl_xor(low, o));
    top = a.g ? factor(top, low) : 1.f;
    if (first && r == 0 && lane == 0) {
        *p.live = p.fine ? 2 * live : live;
        p.top[0] = top;
        p.top[1] = top / a.temperature;
    }
    if (r >= a.rows) return;
    float* const zt = a.logits + (long long)row * a.k;
    if (!in) {  // (a row left out)
        if (!first) return;
        if (a.loss && lane < a.k) zt[lane] = 0.f;
        if (a.loss && lane == 0) a.loss[row] = a.lse[row] = 0.f;
        if (p.dx)
            for (int q = lane; q < a.dim / 4; q += 64) *reinterpret_cast<uint2*>(p.dx + row * a.ld_dx + 4 * q) = make_uint2(0u, 0u);
        return;
    }
    wave_join(m, s);
    const float lse = (m + __builtin_amdgcn_logf(s)) * LN2;
    int id = lane < a.k ? entry_id(a, row, lane) : -1;
    float q = id < 0 ? 0.f : 1.f, ent = 0.f;
    if (a.vals) {
        float v = lane < a.k ? a.vals[(long long)row * a.ld_vals + lane] : -INFINITY;
        if (v == -INFINITY) id = -1;
        if (id < 0) v = -INFINITY;
        teacher(v, id, w, a.temperature, q, ent);
    }
    float all = 0.f;  // (an id that comes twice)
    for (int i = 0; i < a.k; ++i) {
        const float other = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(q), i));
        if (__builtin_amdgcn_readlane(id, i) == id) all += other;
    }
    if (id >= v0 && id < v0 + 256) reinterpret_cast<float*>(taken[wave])[id - v0] = all;
    __builtin_amdgcn_wave_barrier();
    const f32x4 less = taken[wave][lane];
    const float l2 = lse * LOG2E, gr = a.g ? a.g[row] : 1.f, gs = gr / top;
    float d[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        d[e] = v0 + 4 * lane + e < a.valid ? (__builtin_amdgcn_exp2f(__builtin_fmaf(z[e], p.sc, -l2)) - less[e]) * gs : 0.f;
    const uint2 hi = make_uint2(cvt2(d[0], d[1]), cvt2(d[2], d[3]));
    uint16_t* const dz = p.dz + blockIdx.x * p.dz_panel + 4 * lane;
    *reinterpret_cast<uint2*>(dz + at * 256) = hi;
    if (p.fine) {
        const uint32_t bits[4] = {hi.x << 16, hi.x & 0xFFFF0000u, hi.y << 16, hi.y & 0xFFFF0000u};
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // (of an infinite value nothing is left)
            const float h = __uint_as_float(bits[e]);
            d[e] = __builtin_fabsf(h) == INFINITY ? 0.f : d[e] - h;
        }
        *reinterpret_cast<uint2*>(dz + (live + at) * 256) = make_uint2(cvt2(d[0], d[1]), cvt2(d[2], d[3]));
    }
    if (!first) return;
    if (lane == 0) p.idx[at] = row;
    if (a.loss) {
        const float zj = id < 0 ? 0.f : p.kept[(id >> 8) * p.panel + row * 256 + (id & 255)];
        if (lane < a.k) zt[lane] = zj;
        const float c = id < 0 || q == 0.f ? 0.f : q * (lse - zj * p.inv_t);
        float loss = 0.f;
        for (int i = 0; i < a.k; ++i) loss += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(c), i));
        if (lane == 0) {
            a.lse[row] = lse;
            a.loss[row] = a.vals ? ent + loss : loss;
        }
    }
    if (live == a.rows && !p.fine) return;  // (x is read where it lies)
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.x) + (long long)row * a.ldx);
    uint4 *dst = reinterpret_cast<uint4*>(p.xc + (long long)at * a.dim), *more = dst + (long long)live * (a.dim / 8);
#pragma unroll 4
    for (int i = lane; i < a.dim / 8; i += 64) {
        const uint4 v = src[i];
        dst[i] = v;
        if (p.fine) more[i] = v;
    }
}

struct Fix {
    const int *live, *idx, *ids;
    const float *q, *lse, *zt, *g, *top;
    int k, kp, v0, v1;
    float sc;
    uint16_t* dz;
    long long panel;
};

// a teacher's entries' own dz: p less the entries' q of that id
__global__ __launch_bounds__(256) void hl_fix(const Fix p) {
    const int e = blockIdx.x * 256 + threadIdx.x, n = e >> p.kp, w = 1 << p.kp, j = e & (w - 1);
    const bool in = n < *p.live;
    const long long row = in ? p.idx[n] : 0;
    const int id = in ? p.ids[(row << p.kp) + j] : -1;
    const float q = id < 0 ? 0.f : p.q[(row << p.kp) + j];
    float all = 0.f;
    if (w == 64) {
        for (int i = 0; i < 64; ++i) {
            const float oq = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(q), i));
            if (__builtin_amdgcn_readlane(id, i) == id) all += oq;
        }
    } else {
        for (int i = 0; i < w; ++i) {
            const int oid = __shfl(id, i, w);
            const float oq = __shfl(q, i, w);
            if (oid == id) all += oq;
        }
    }
    if (id < p.v0 || id >= p.v1) return;
    const float top = *p.top, gr = p.g ? p.g[row] : 1.f, gs = gr / top;
    const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(p.zt[row * p.k + j], p.sc, -p.lse[row] * LOG2E));
    const int v = id - p.v0;
    p.dz[(v >> 8) * p.panel + (long long)n * 256 + (v & 255)] = (uint16_t)cvt2(gs * (pr - all), 0.f);
}

struct Finish {
    const float* acc;
    int tm, bm, bn, wk, steps, dim;
    const int *live, *idx;
    const float* scale;
    uint16_t* dx;
    long long ld_dx;
    int fine;  // two rows of sums each
};

// dx from the splits' sums (none: it is there): 256 columns of a row at a time, a quarter of the splits a wavefront
__global__ __launch_bounds__(256) void hl_dx(const Finish p) {
    __shared__ f32x4 part[4][64];
    const int live = *p.live, splits = dx_splits(pace(EPI_DX, p.bm, p.bn, p.wk), p.tm * ((live + p.bn - 1) / p.bn), p.steps, p.bm * p.bn * 4);
    if (splits == 1 && !p.fine) return;
    const int sums = splits << p.fine, rows = live >> p.fine;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cols = (p.dim + 255) / 256;
    const float s = *p.scale;
    const long long stride = (long long)live * p.dim;
    for (int w = blockIdx.x; w < rows * cols; w += gridDim.x) {
        const int n = w / cols, d = 256 * (w - n * cols) + 4 * lane;
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
        if (d < p.dim) {
            const float* at = p.acc + (long long)n * p.dim + d;
#pragma unroll 8
            for (int i = wave; i < sums; i += 4)
                v += *reinterpret_cast<const f32x4*>(at + (i >> p.fine) * stride + (i & p.fine) * (long long)rows * p.dim);
        }
        part[wave][lane] = v;
        __syncthreads();
        if (wave == 0 && d < p.dim) {
            v = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
            *reinterpret_cast<uint2*>(p.dx + p.idx[n] * p.ld_dx + d) = make_uint2(cvt2(v[0] * s, v[1] * s), cvt2(v[2] * s, v[3] * s));
        }
        __syncthreads();
    }
}

// --- the plan ----------------------------------------------------------------------------------------------------------

constexpr long long DZ_BYTES = 1ll << 30;  // dz a piece at most
// z of a call that is one piece (float32, 2 GB at most) is kept from the loss to dz where computing it again takes longer than
// writing and reading it: 2048 rows x 1024 against 128256 tokens 1.88 ms kept, 2.03 again, x 768 1.59 and 1.62, x 512 1.26 and
// 1.20, x 64 0.83 and 0.59; 4096 x 2048 6.20 and 7.29.
constexpr int KEEP_DIM = 768;

// dz is rounded to bf16 because the matrix instructions take bf16: it is off by half a step, and so is what one value of it
// dominates, at any number of rows (a token's row of dhead that one row's p - 1 makes, a row's dx that a teacher's best entry
// does). Over all of dhead or dx that adds 1.6e-3 of the norm at most to the 1.65e-3 of their own rounding (root of the squares:
// 2.3e-3 with a teacher's 16 entries, 1.7e-3 for 401 rows' tokens). Of one piece and few rows it is the worst (one row x 552,
// 5 entries: dhead off by 2.8e-3 of its norm, by its own rounding alone 1.7e-3). Up to 32 rows what the rounding
// leaves goes through the products as rows of its own, which a tile of 64 has room for (8 rows x 1024 against 8192 tokens 34 us
// with it and without, 32 x 4096 against 128256 677 and 659).
constexpr int FINE_ROWS = 32;
constexpr int MOST_TILES = (1 << 23) - 8;  // of 512 lanes: a launch holds fewer than 2^32

long long up(long long v, long long to) { return (v + to - 1) / to * to; }

struct Plan {
    int kp, piece;
    int z, y, w, d;  // the tiles of z for the statistics and for dz, of dhead and of dx
    int parts;
    bool gather, raw, own, keep, few, fine;
    bool one_stage;  // dhead
    int dz_rows;  // the rows of dz and of what is made of it
    long long joined, kept, ids, idc, q, ent, held, idx, pos, live, xc, part, dz, acc, bytes;
};

int log2_up(int k) {
    int p = 0;
    while ((1 << p) < k) ++p;
    return p;
}

enum Tiles { T256, T128, T64, T64K, T256x64, T128x64 };  // (T64K: two groups of wavefronts split K)
struct Size {
    int bm, bn, wk;
};
constexpr Size SIZE[] = {{256, 256, 1}, {128, 128, 1}, {64, 64, 1}, {64, 64, 2}, {256, 64, 1}, {128, 64, 1}};

constexpr Pace pace_of(int epi, int t) { return pace(epi, SIZE[t].bm, SIZE[t].bn, SIZE[t].wk); }

int tiles_of(int t, long long m, long long n) {
    return (int)(up(m, SIZE[t].bm) / SIZE[t].bm * (up(n, SIZE[t].bn) / SIZE[t].bn));
}

// the tile of `tiles` that takes the least time for a product of m rows by n columns, summed over k
int choose(int epi, long long m, long long n, long long k, std::initializer_list<int> tiles) {
    int best = 0;
    float least = 1e30f;
    const int steps = (int)(up(k, KSTEP) / KSTEP);
    for (int t : tiles) {
        float us;
        if (epi == EPI_DX) dx_splits(pace_of(epi, t), tiles_of(t, m, n), steps, SIZE[t].bm * SIZE[t].bn * 4, &us);
        else us = tiled_us(pace_of(epi, t), tiles_of(t, m, n), steps);
        if (us < least) least = us, best = t;
    }
    return best;
}

// z's: up to 64 columns take tiles as narrow, of 128 rows where there are two a CU and more, which then only wait for the head
// (32 rows x 4096: 131072 tokens 171 us, 6.2 TB/s, 65536 tokens 110; in tiles of 256 rows 174 and 136)
int choose_z(long long m, long long n, long long k) {
    if (n <= 64 && tiles_of(T128x64, m, n) >= 2 * CUS) return T128x64;
    return n <= 64 ? choose(EPI_DZ, m, n, k, {T64, T64K}) : choose(EPI_DZ, m, n, k, {T256, T128, T64, T64K});
}

bool plan_of(const dr_head_loss* a, int what, Plan& p) {
    if (a == nullptr || what < 1 || what > 3 || a->rows < 1 || a->rows > (1 << 20) || a->dim < 8 || a->dim % 8 ||
        a->dim > (1 << 17) || a->vocab < 1 || a->vocab > (1 << 28) || a->valid < 1 || a->valid > a->vocab || a->k < 1 ||
        a->k > DR_LOSS_MAX_K || (a->vals == nullptr && (a->k != 1 || a->temperature != 1.f)) ||
        !(a->temperature >= 0x1p-20f && a->temperature < INFINITY) || a->ldx < a->dim || a->ldx % 8 || a->ld_head < a->dim ||
        a->ld_head % 8 || a->ldx > DR_LOSS_MAX_LD || a->ld_head > DR_LOSS_MAX_LD || a->ld_ids < a->k || (a->vals && a->ld_vals < a->k))
        return false;
    const bool back = what & DR_LOSS_BACKWARD && (a->dx || a->dhead);  // (asked for neither: the forward alone)
    const long long n = a->rows, np = up(n, 64);
    if (up(a->valid, 64) / 64 * (np / 64) > 1 << 30) return false;  // (tiles counted in 32 bits)
    p.kp = log2_up(a->k);
    p.z = choose_z(a->valid, n, a->dim);
    if (tiles_of(p.z, a->valid, n) >= MOST_TILES) return false;
    p.parts = (int)(up(a->valid, SIZE[p.z].bm) / SIZE[p.z].bm);
    // the vocabulary in equal pieces of a multiple of 256; what is made of one
    const long long tiles = up(a->valid, 256) / 256, fit = DZ_BYTES / (n * 512);
    const long long pieces = (tiles + (fit > 1 ? fit : 1) - 1) / (fit > 1 ? fit : 1);
    p.piece = back ? (int)((tiles + pieces - 1) / pieces) * 256 : 0;
    const bool one = back && pieces == 1;
    p.few = one && (n <= FINE_ROWS || few_parts((int)n, p.parts)) && n << p.kp <= FEW_IDS;
    p.fine = p.few && n <= FINE_ROWS;
    p.keep = p.few || (one && what & DR_LOSS_FORWARD && a->dim >= KEEP_DIM);
    // (forward alone, the rows that count are gathered where leaving out the others may save more than that takes, about 10 us)
    p.gather = back || (double)n * a->valid * a->dim > 3e10;
    p.raw = !p.gather && a->vals == nullptr && a->ld_ids == 1;  // (tokens read where they are: no launch before z's)
    p.own = p.gather && n << p.kp <= FEW;
    long long at = 0;
    auto take = [&](long long bytes) {
        const long long here = at;
        at += up(bytes, 256);
        return here;
    };
    p.ids = take(n * 4 << p.kp);
    p.idc = take(p.gather ? n * 4 << p.kp : 0);
    p.q = take(a->vals ? n * 4 << p.kp : 0);
    p.ent = take(a->vals ? n * 4 : 0);
    p.held = take(n);
    p.idx = take(n * 4);
    p.pos = take(n * 4);
    p.live = take(12);
    p.xc = take(p.gather ? (p.fine ? 2 : 1) * n * a->dim * 2 : 0);
    p.part = take(what & DR_LOSS_FORWARD || p.few ? p.parts * np * 8 : 0);
    p.dz = p.acc = p.kept = p.joined = p.dz_rows = 0;
    if (back) {
        const long long nr = p.dz_rows = (int)(p.fine ? 2 * n : n);
        p.dz = take(nr * p.piece * 2);
        p.joined = take(p.few ? n * 8 : 0);
        p.kept = take(p.keep ? n * p.piece * 4 : 0);
        p.y = choose_z(p.piece, n, a->dim);
        p.w = choose(EPI_DHEAD, a->dim, p.piece, nr, {T256, T128});
        // (few steps: one stage and five workgroups a CU instead of four and two; 400 rows x 2880 against 50257 tokens, dx
        // aside, 365 us and 382, 1003 rows 709 and 711, 1500 x 1024 against 8192 98.7 and 94.0)
        p.one_stage = nr <= KSTEP || (p.w == T128 && n <= 1024);
        if (a->dx) {
            p.d = nr <= 64 ? choose(EPI_DX, a->dim, nr, p.piece, {T256x64, T64K})
                           : choose(EPI_DX, a->dim, nr, p.piece, {T256, T128, T64K});
            // the sums of all rows where there are several pieces, or two rows of sums for one; of splits no more than ROUNDS
            // rounds of tiles
            const long long whole = p.piece < a->valid || p.fine ? nr * a->dim : 0;
            const long long split = (long long)ROUNDS * pace_of(EPI_DX, p.d).at_once * SIZE[p.d].bm * SIZE[p.d].bn;
            p.acc = take((whole > split ? whole : split) * 4);
        }
    }
    p.bytes = at;
    return true;
}

template <int BM, int BN, int WM, int WN, int WK, int NS, int BK, bool AT, bool BT, int EPI>
void launch(Gemm g, hipStream_t st) {
    g.tm = (g.m + BM - 1) / BM;
    g.tn = (g.n + BN - 1) / BN;
    int grid = g.tm * g.tn;
    constexpr int most = ROUNDS * pace(EPI, BM, BN, WK).at_once;
    if (EPI == EPI_DX && grid < most) grid = most;
    grid = (grid + 7) & ~7;  // (as many for each XCD)
    hipLaunchKernelGGL((hl_gemm<BM, BN, WM, WN, WK, NS, BK, AT, BT, EPI>), dim3(grid), dim3(64 * WM * WN * WK), 0, st, g);
}

template <int EPI>
void launch_z(const Gemm& g, int t, hipStream_t st) {
    switch (t) {
        case T256: return launch<256, 256, 2, 4, 1, 2, 64, false, false, EPI>(g, st);
        case T128: return launch<128, 128, 2, 2, 1, 2, 64, false, false, EPI>(g, st);
        case T128x64: return launch<128, 64, 2, 2, 1, 3, 64, false, false, EPI>(g, st);
        case T64: return launch<64, 64, 2, 2, 1, 4, 64, false, false, EPI>(g, st);
        default: return launch<64, 64, 2, 2, 2, 4, 64, false, false, EPI>(g, st);
    }
}

}  // namespace

extern "C" int64_t dr_head_loss_workspace_bytes(const dr_head_loss* a, int what) {
    Plan p;
    return plan_of(a, what, p) ? p.bytes : -1;
}

extern "C" int dr_head_loss_plan(const dr_head_loss* a, int what, dr_head_loss_info* info) {
    Plan p;
    if (info == nullptr || !plan_of(a, what, p)) return DR_EINVAL;
    *info = dr_head_loss_info{};
    const bool fwd = what & DR_LOSS_FORWARD, back = p.piece > 0;
    auto tile = [](int32_t (&to)[3], int t) { to[0] = SIZE[t].bm, to[1] = SIZE[t].bn, to[2] = SIZE[t].wk; };
    if (fwd || p.few) tile(info->z, p.z);
    info->kept = p.keep;
    info->few = p.few + p.fine;
    if (!back) return DR_OK;
    info->piece = p.piece;
    info->pieces = (a->valid + p.piece - 1) / p.piece;
    if (!p.keep) tile(info->dz, p.y);
    if (a->dhead) tile(info->dhead, p.one_stage ? T128 : p.w), info->dhead_stages = p.one_stage ? 1 : 4;
    if (a->dx) {
        tile(info->dx, p.d);
        const Size s = SIZE[p.d];
        info->dx_splits = dx_splits(pace_of(EPI_DX, p.d), tiles_of(p.d, a->dim, p.dz_rows), p.piece / KSTEP, s.bm * s.bn * 4);
    }
    return DR_OK;
}

extern "C" int dr_head_loss_run(const dr_head_loss* a, int what) {
    Plan P;
    if (!plan_of(a, what, P)) return DR_EINVAL;
    auto aligned = [](const void* p, uintptr_t to) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % to == 0; };
    const bool fwd = what & DR_LOSS_FORWARD, back = what & DR_LOSS_BACKWARD && (a->dx || a->dhead);
    if (!aligned(a->x, 16) || !aligned(a->head, 16) || !aligned(a->ids, a->ids64 ? 8 : 4) || !aligned(a->lse, 4) ||
        !aligned(a->logits, 4) || (fwd && !aligned(a->loss, 4)) || !aligned(a->workspace, 256) || a->workspace_bytes < P.bytes ||
        (back && a->dx && (!aligned(a->dx, 16) || a->ld_dx < a->dim || a->ld_dx % 8)) ||
        (back && a->dhead && (!aligned(a->dhead, 16) || a->ld_dhead < a->dim || a->ld_dhead % 8)))
        return DR_EINVAL;
    if (!fwd && !back) return DR_OK;
    const hipStream_t st = reinterpret_cast<hipStream_t>(a->stream);
    char* ws = reinterpret_cast<char*>(a->workspace);
    const int n = a->rows, kn = a->k;
    Prep p{};
    p.a = *a;
    p.kp = P.kp;
    p.ids = reinterpret_cast<int*>(ws + P.ids);
    p.q = a->vals ? reinterpret_cast<float*>(ws + P.q) : nullptr;
    p.ent = reinterpret_cast<float*>(ws + P.ent);
    p.held = reinterpret_cast<uint8_t*>(ws + P.held);
    p.idx = reinterpret_cast<int*>(ws + P.idx);
    p.pos = reinterpret_cast<int*>(ws + P.pos);
    p.live = reinterpret_cast<int*>(ws + P.live);
    p.top = reinterpret_cast<float*>(ws + P.live + 4);
    p.xc = reinterpret_cast<uint16_t*>(ws + P.xc);
    p.dx = back ? reinterpret_cast<uint16_t*>(a->dx) : nullptr;
    p.idc = reinterpret_cast<int*>(ws + P.idc);
    const int eblocks = (int)((((long long)n << P.kp) + 255) / 256);
    const dim3 gblocks((n + GROWS - 1) / GROWS + 1);
    const bool gather = P.gather && !P.few;  // (before the products)
    if (!P.raw && !P.own && !P.few) hipLaunchKernelGGL(hl_entries, dim3(eblocks), dim3(256), 0, st, p);
    if (gather && P.own) hipLaunchKernelGGL((hl_gather<true, GROWS>), gblocks, dim3(256), 0, st, p);
    else if (gather && n <= MANY) hipLaunchKernelGGL((hl_gather<false, GROWS>), gblocks, dim3(256), 0, st, p);
    else if (gather) hipLaunchKernelGGL((hl_gather<false, 64>), dim3((n + 63) / 64 + 1), dim3(256), 0, st, p);

    Gemm z{};  // z of a range of the vocabulary
    z.A = reinterpret_cast<const uint16_t*>(a->head);
    z.lda = a->ld_head;
    z.B = gather ? p.xc : reinterpret_cast<const uint16_t*>(a->x);
    z.ldb = gather ? a->dim : a->ldx;
    z.n = n, z.k = z.ka = a->dim;
    z.whole = P.gather ? reinterpret_cast<const uint16_t*>(a->x) : nullptr, z.ldx = a->ldx, z.rows = n;
    z.live = gather ? p.live : nullptr;
    z.idx = gather ? p.idx : nullptr;
    z.sc = LOG2E / a->temperature;
    z.ids = P.gather ? p.idc : p.ids, z.kp = P.kp, z.kn = kn;
    z.raw = P.raw ? a->ids : nullptr, z.raw64 = a->ids64;
    z.lse = a->lse, z.g = a->g, z.top = p.top;
    if (fwd || P.few) {  // (few rows' gradients are the same with and without their loss)
        Gemm s = z;
        s.m = a->valid;
        s.part = reinterpret_cast<f32x2*>(ws + P.part);
        s.ld_part = up(n, 64);
        s.zt = a->logits;
        s.kept = P.keep ? reinterpret_cast<float*>(ws + P.kept) : nullptr;
        s.panel = (long long)n * 256;
        if (P.keep) launch_z<EPI_KEEP>(s, P.z, st);
        else launch_z<EPI_STATS>(s, P.z, st);
        Merge m{s.part, s.ld_part, P.parts, n, kn, P.kp, P.gather ? p.pos : nullptr, P.raw ? nullptr : p.held, a->ids,
                a->ids64, a->valid, p.ids, p.q, p.ent, 1.f / a->temperature, a->loss, a->lse, a->logits, s.kept, s.panel};
        if (P.few) {
            const bool few = few_parts(n, P.parts);  // (more are joined once, by a launch of its own)
            f32x2* joined = reinterpret_cast<f32x2*>(ws + P.joined);
            if (!few) hipLaunchKernelGGL(hl_join, dim3(n), dim3(256), 0, st, s.part, s.ld_part, P.parts, joined);
            Few f{*a, P.kp, few ? P.parts : 1, few ? s.part : joined, s.ld_part, s.kept, reinterpret_cast<uint16_t*>(ws + P.dz),
                  s.panel, 256ll * P.dz_rows, z.sc, 1.f / a->temperature, p.idx, p.live, p.top, p.xc, p.dx, P.fine};
            if (!fwd) f.a.loss = nullptr;
            hipLaunchKernelGGL(hl_few, dim3((a->valid + 255) / 256, (n + 3) / 4), dim3(256), 0, st, f);
        } else if (few_parts(n, P.parts)) {  // (in hl_few's order: the loss alone is the same)
            hipLaunchKernelGGL((hl_merge<1, 64>), dim3(n), dim3(64), 0, st, m);
        } else if (n <= 64) hipLaunchKernelGGL((hl_merge<1, 256>), dim3(n), dim3(256), 0, st, m);
        else hipLaunchKernelGGL((hl_merge<16, 64>), dim3((n + 15) / 16), dim3(1024), 0, st, m);
    }
    if (back) {
        uint16_t* dz = reinterpret_cast<uint16_t*>(ws + P.dz);
        const long long panel = 256ll * P.dz_rows;
        for (int v0 = 0; v0 < a->valid; v0 += P.piece) {
            const int vn = a->valid - v0 < P.piece ? a->valid - v0 : P.piece;
            Gemm s = z;
            s.A += (long long)v0 * a->ld_head;
            s.m = vn;
            s.v0 = v0;
            s.out = dz;
            s.panel = panel;
            if (P.keep && !P.few) {
                Dz d{p.live, p.idx, a->vals ? nullptr : p.idc, reinterpret_cast<const float*>(ws + P.kept), a->lse, a->g, p.top,
                     dz, panel, vn, z.sc};
                hipLaunchKernelGGL(hl_dz, dim3((vn + 255) / 256, (n + 4 * DZ_ROWS - 1) / (4 * DZ_ROWS)), dim3(256), 0, st, d);
            } else if (!P.few && a->vals) {
                launch_z<EPI_DZ>(s, P.y, st);
            } else if (!P.few) {
                launch_z<EPI_DZ1>(s, P.y, st);
            }
            if (a->vals && !P.few) {
                Fix f{p.live, p.idx, p.ids, p.q, a->lse, a->logits, a->g, p.top, kn, P.kp, v0, v0 + vn, z.sc, dz, panel};
                hipLaunchKernelGGL(hl_fix, dim3(eblocks), dim3(256), 0, st, f);
            }
            if (a->dhead) {
                Gemm w{};
                w.A = p.xc, w.lda = a->dim;
                w.whole = P.fine ? nullptr : z.whole, w.ldx = z.ldx, w.rows = n;
                w.B = dz, w.ldb = 256, w.panel = panel;
                // (the rows past valid: zeros, with the last piece)
                w.m = a->dim, w.nb = vn, w.n = v0 + vn == a->valid ? a->vocab - v0 : vn, w.k = P.dz_rows, w.live = p.live;
                w.out = reinterpret_cast<uint16_t*>(a->dhead) + (long long)v0 * a->ld_dhead;
                w.ld_out = a->ld_dhead;
                w.scale = p.top + 1;
                if (P.one_stage) launch<128, 128, 2, 2, 1, 1, 64, true, true, EPI_DHEAD>(w, st);
                else if (P.w == T256) launch<256, 256, 2, 4, 1, 4, 32, true, true, EPI_DHEAD>(w, st);
                else launch<128, 128, 2, 2, 1, 4, 32, true, true, EPI_DHEAD>(w, st);
            }
            if (a->dx) {
                Gemm d{};
                d.A = z.A + (long long)v0 * a->ld_head, d.lda = a->ld_head;
                d.B = dz, d.ldb = 256, d.panel = panel;
                d.m = a->dim, d.n = P.dz_rows, d.k = (int)up(vn, 8), d.ka = vn, d.live = p.live;
                d.plan_steps = P.piece / KSTEP;
                d.acc = reinterpret_cast<float*>(ws + P.acc);
                d.ld_acc = a->dim;
                d.add = v0 > 0;
                d.idx = p.idx;
                d.scale = p.top + 1;
                if (v0 + vn == a->valid && !P.fine) d.out = reinterpret_cast<uint16_t*>(a->dx), d.ld_out = a->ld_dx;
                if (P.d == T64K) launch<64, 64, 2, 2, 2, 4, 64, true, false, EPI_DX>(d, st);
                else if (P.d == T256x64) launch<256, 64, 2, 2, 1, 4, 32, true, false, EPI_DX>(d, st);
                else if (P.d == T128) launch<128, 128, 2, 2, 1, 4, 32, true, false, EPI_DX>(d, st);
                else launch<256, 256, 2, 4, 1, 4, 32, true, false, EPI_DX>(d, st);
            }
        }
        if (a->dx) {
            const Size t = SIZE[P.d];
            Finish f{reinterpret_cast<const float*>(ws + P.acc), (int)(up(a->dim, t.bm) / t.bm), t.bm, t.bn, t.wk, P.piece / KSTEP, a->dim, p.live,
                     p.idx, p.top + 1, reinterpret_cast<uint16_t*>(a->dx), a->ld_dx, P.fine};
            const long long items = (long long)n * ((a->dim + 255) / 256);
            hipLaunchKernelGGL(hl_dx, dim3((unsigned)(items < 4096 ? items : 4096)), dim3(256), 0, st, f);
        }
    }
    return hipGetLastError() == hipSuccess ? DR_OK : DR_EHIP;
}
