// mfma_tile.h: what the tiled MFMA products for MI355X (gfx950) that read both operands as they lie in memory are made of:
// an operand's tile in LDS, filled straight from memory and read along the summed dimension or across it; the order of the
// tiles; the time that a plan expects of them.
#ifndef MFMA_TILE_H
#define MFMA_TILE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

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

constexpr int KSTEP = 64;                  // k that plans count in
constexpr uint32_t PAST = 0x80000000u;     // a buffer offset past every record: the load gives zeros
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ uint32_t cvt2(float lo, float hi) {  // to bf16, to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}

__device__ __forceinline__ f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The wavefront's LDS reads done and all but its newest VM loads landed, then the workgroup's barrier.
template <int VM>
__device__ __forceinline__ void step_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((VM & 15) | (7 << 4) | ((VM >> 4) << 14));  // vmcnt(VM) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// One operand's tile of ROWS x BK values in LDS: 16-byte chunks, laid out so that neither the loads straight from memory
// (64 chunks in a row a wavefront) nor the fragments' reads meet in a bank.
// QUARTERS: for fragments of 16 rows by 32 k (frag16), else of 32 by 16 (frag).
template <int ROWS, bool T, int NT, int BK, bool QUARTERS = false>
struct Tile {
    static constexpr int N = ROWS * BK / 8 / NT;  // chunks a lane loads
    static constexpr int CK = BK / 8;             // chunks of a row's k
    uint32_t off[N];

    // row r's chunk c (8 k) turned by row, so that 16 rows' fill all banks; across: k's chunk c (8 rows), in pairs (32 bytes)
    // turned by k
    // (QUARTERS, 64 bytes a row: lanes 0-3, 12-15 and 20-27 read together, 8 rows of one chunk and 8 of the next)
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (BK == 64) return (r >> 1) & 7;
        const int v = (r >> 2) & 3;
        return QUARTERS ? ((v << 1) & 3) ^ (3 * (v >> 1)) : v;
    }
    static __device__ __forceinline__ int turn(int k) {
        const int t = ROWS % 128 == 0 ? 2 * (k & 3) : ROWS % 64 == 0 ? 2 * ((k >> 1) & 1) : 0;  // (a row of k is 0 or 128 bytes mod 256)
        return QUARTERS ? t | ((k >> 3) & 1) : t;  // (32 lanes at a time: 32 rows of the same k, or 16 of k and 8 further)
    }

    __device__ __forceinline__ void init(int tid, int ld, int rows) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int s = i * NT + tid;
            if constexpr (T) {
                constexpr int C = ROWS / 8;
                const int k = s / C, c = s % C, src = ((((c >> 1) ^ turn(k))) << 1) | (c & 1);
                off[i] = 8 * src < rows ? (uint32_t)(k * ld * 2) + 16u * src : PAST;
            } else {
                const int r = s / CK, c = (s % CK) ^ swz(r);
                off[i] = (uint32_t)(r * ld * 2) + 16u * c;
            }
        }
    }
    // The step's loads: at: its first value; ld; rows: the operand's rows in the tile (at least 1); left: its k from this step
    // on (none left: zeros). Never further than the tile's own run of its last row: what comes after may be rows that are not
    // to be read.
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t source(const uint16_t* at, int ld, int rows, int left) {
        const int r = T ? min(left, BK) : rows, run = min(T ? (rows + 7) & ~7 : (left + 7) & ~7, T ? ROWS : BK);
        if constexpr (QUARTERS) {  // (no branch in the K loop: 2 % of a large product's time)
            return __builtin_amdgcn_make_buffer_rsrc((void*)at, (short)0, (((r - 1) * ld + run) * 2) & (-left >> 31), 0x00020000);
        }
        return __builtin_amdgcn_make_buffer_rsrc((void*)at, (short)0, left > 0 ? ((r - 1) * ld + run) * 2 : 0, 0x00020000);
    }
    // the lane's chunk i of it to LDS (AUX 2: not to be kept in the caches)
    template <int AUX = 0>
    __device__ __forceinline__ void load(int i, __amdgpu_buffer_rsrc_t from, int left, uint4* lds, int tid) const {
        uint32_t o = off[i];
        if constexpr (!T) {
            if (left < BK) {  // (the last step of a ragged k)
                const int s = i * NT + tid, c = (s % CK) ^ swz(s / CK);
                if (8 * c >= left) o = PAST;
            }
        }
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_ptr)(lds + i * NT + 64 * __builtin_amdgcn_readfirstlane(tid >> 6)), 16, o,
                                                 0, 0, AUX);
    }
    // lane's 8 values of row r0 + lane % 32, k = 16 u + 8 (lane / 32) .., the tile from chunk `from` of the stage on. (One
    // index from the stage's array: through longer chains the compiler no longer sees which stage a read is of, and has it
    // wait for the loads to the other.)
    static __device__ __forceinline__ uint4 frag(const uint4* lds, int from, int r0, int u, int lane) {
        if constexpr (T) {
            constexpr int C = ROWS / 8;
            const int h = lane >> 5, half = (lane >> 4) & 1, i = lane & 15;
            const int k = 8 * h + (i >> 2), pair = ((r0 >> 4) + half) ^ turn(k);  // (turn: the same 4 and 16 k further)
            const int at = (from + k * C + 2 * pair) * 8 + 4 * (i & 3) + 16 * u * ROWS;
            const uint16_t* v = reinterpret_cast<const uint16_t*>(lds);
            const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(v + at)));
            const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(v + (at + 4 * ROWS))));
            return make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
            const int r = lane & 31, h = lane >> 5;
            return lds[from + (r0 + r) * CK + ((2 * u + h) ^ swz(r))];
        }
    }
    // lane's 8 values of row r0 + lane % 16, k = 32 u + 8 (lane / 16) ..
    static __device__ __forceinline__ uint4 frag16(const uint4* lds, int from, int r0, int u, int lane) {
        static_assert(QUARTERS && ROWS % 32 == 0, "a tile laid out for them");
        const int i = lane & 15, q = lane >> 4;
        if constexpr (T) {
            constexpr int C = ROWS / 8;
            const int k = 8 * q + (i >> 2), pair = (r0 >> 4) ^ turn(k);  // (turn: the same 4 and 32 k further)
            const int at = (from + k * C + 2 * pair) * 8 + 4 * (i & 3) + 32 * u * ROWS;
            const uint16_t* v = reinterpret_cast<const uint16_t*>(lds);
            const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(v + at)));
            const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(v + (at + 4 * ROWS))));
            return make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
            return lds[from + (r0 + i) * CK + ((4 * u + q) ^ swz(r0 + i))];
        }
    }
};

// What a plan takes a workgroup's time to be: so many at once on the card, us for a step of KSTEP k, more of them with more of
// the CUs at work, and for its beginning and end.
struct Pace {
    int at_once;
    float step, shared, ends;
};
constexpr int CUS = 256;

__host__ __device__ inline float tiled_us(const Pace& p, int tiles, int steps) {
    const int rounds = (tiles + p.at_once - 1) / p.at_once;
    const float full = rounds ? (float)tiles / (float)(rounds * p.at_once) : 0.f;
    return (float)rounds * ((p.step + p.shared * full) * (float)steps + p.ends);
}

// workgroups go to the XCDs in turn; each XCD takes a run of tiles, in groups of GM row tiles by all column tiles, so that
// what runs at once on an XCD shares rows and columns in its L2. False past the last.
__device__ __forceinline__ bool tile_of(int tm, int tn, int splits, int& mt, int& nt, int& split) {
    const int total = tm * tn * splits, xcd = blockIdx.x & 7, own = (total >> 3) + (xcd < (total & 7));
    if ((int)(blockIdx.x >> 3) >= own) return false;
    int w = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
    split = w / (tm * tn);
    w -= split * tm * tn;
    constexpr int GM = 4;
    const int g = w / (GM * tn), first = g * GM, gm = min(GM, tm - first);
    w -= g * GM * tn;
    nt = w / gm;
    mt = first + w - nt * gm;
    return true;
}

}  // namespace

#endif
