// What the float head's matrix products share (linear.hip, gated.hip, linear_loss.hip): activations, an operand's tiles in LDS, the sums of a
// tile of the product, the kernel core for few rows, and the plan that cuts a product into tiles and splits its sum.
//
// A product is c[i][j] = sum over s of I(i, s) J(j, s), where an operand lies in memory either along the sum (rows of s) or across it (a
// row for every s).
#pragma once

#include <cmath>

#include "head.h"

namespace tcbnn {
namespace head {

// Rows: sums over them, and what is requested ahead of them, are counted in 32 bits.
constexpr int kMaxIn = 1 << 20, kMaxOut = 1 << 28, kMaxRows = 0x7fffffff - (1 << 22) + 1;

// ---- activations.  fp32 uses the library's erf and exp.  In 16-bit types, whose rounding is 2^-9 or 2^-12 of a result, they
// cost as much as a quarter of a large product; there exp is 2^x of the hardware, a quotient its reciprocal (each good to
// one unit in the last place of fp32), and the normal distribution's tail
//   h(z) = erfc(|z| / sqrt 2) / 2 = exp(-z^2 / 2) Q(1 / (1 + 0.3 |z|)),
// Q a polynomial of degree 8 without a constant term, fitted here for the least relative error of h over 0 <= |z| <= 13 (a Lawson
// iteration: least squares, weights multiplied by the errors): 1.2e-7.  Evaluated in fp32 it is good to 5e-7 up to |z| = 2, 2e-6
// up to 6 and 8e-6 at 13, where the rounding of the exponential's argument counts.
constexpr float kLog2e = 1.44269504088896341f;
template <typename T>
__device__ __forceinline__ float exp_of(float x) {
    if constexpr (sizeof(T) == 4) return expf(x);
    return __builtin_amdgcn_exp2f(x * kLog2e);
}
template <typename T>
__device__ __forceinline__ float over(float a, float b) {
    if constexpr (sizeof(T) == 4) return a / b;
    return a * __builtin_amdgcn_rcpf(b);
}
// the normal distribution function of z, and exp(-z^2 / 2)
template <typename T>
__device__ __forceinline__ float normal(float z, float& e) {
    e = exp_of<T>(-0.5f * z * z);
    if constexpr (sizeof(T) == 4) return 0.5f * (1.0f + erff(z * 0.70710678118654752f));
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(z), 0.3f, 1.0f));
    float q = 0.036194976f;
    q = __builtin_fmaf(q, t, -0.15937878f);
    q = __builtin_fmaf(q, t, 0.21011917f);
    q = __builtin_fmaf(q, t, -0.05716805f);
    q = __builtin_fmaf(q, t, 0.13041681f);
    q = __builtin_fmaf(q, t, 0.09934702f);
    q = __builtin_fmaf(q, t, 0.12084555f);
    q = __builtin_fmaf(q, t, 0.11962326f);
    const float h = q * t * e;
    return z < 0.0f ? h : 1.0f - h;
}
template <typename T, int ACT>
__device__ __forceinline__ float activate(float z) {
    float e;
    if constexpr (ACT == TCBNN_ACT_RELU) return z > 0.0f || z != z ? z : 0.0f;
    if constexpr (ACT == TCBNN_ACT_GELU) return z * normal<T>(z, e);
    if constexpr (ACT == TCBNN_ACT_SILU) return over<T>(z, 1.0f + exp_of<T>(-z));
    return z;
}
template <typename T, int ACT>
__device__ __forceinline__ float slope(float z) {
    float e;
    if constexpr (ACT == TCBNN_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if constexpr (ACT == TCBNN_ACT_GELU) {
        const float phi = normal<T>(z, e);
        return __builtin_fmaf(z * 0.39894228040143268f, e, phi);
    }
    if constexpr (ACT == TCBNN_ACT_SILU) {
        const float p = over<T>(1.0f, 1.0f + exp_of<T>(-z));
        return p * __builtin_fmaf(z, 1.0f - p, 1.0f);
    }
    return 1.0f;
}
template <typename F>
__host__ __device__ __forceinline__ void by_activation(int act, F&& f) {
    if (act == TCBNN_ACT_RELU) return f(std::integral_constant<int, TCBNN_ACT_RELU>());
    if (act == TCBNN_ACT_GELU) return f(std::integral_constant<int, TCBNN_ACT_GELU>());
    if (act == TCBNN_ACT_SILU) return f(std::integral_constant<int, TCBNN_ACT_SILU>());
    return f(std::integral_constant<int, TCBNN_ACT_NONE>());
}

// ---- matrix instructions.  16 bytes of a row or column of each operand are one instruction's share of a lane in the 16-bit types
// (32 x 32, 16 of the sum) and four instructions' in fp32 (32 x 32, 2 of the sum each).  Lane l holds row l % 32 of its operand,
// half l / 32 of the sum.  Accumulator register v of lane l is row 8 (v / 4) + 4 (l / 32) + v % 4 of the first operand and row
// l % 32 of the second: with J first a lane holds runs of four neighbouring j.
typedef int Words __attribute__((ext_vector_type(4)));
typedef float Acc __attribute__((ext_vector_type(16)));
template <typename T>
__device__ __forceinline__ Acc mma(Words j, Words i, Acc c) {
    if constexpr (std::is_same_v<T, __bf16>) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Vec<__bf16>, j), __builtin_bit_cast(Vec<__bf16>, i), c, 0, 0, 0);
    } else if constexpr (std::is_same_v<T, _Float16>) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(Vec<_Float16>, j), __builtin_bit_cast(Vec<_Float16>, i), c, 0, 0, 0);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__int_as_float(j[e]), __int_as_float(i[e]), c, 0, 0, 0);
        return c;
    }
}

// ---- an operand's tiles.  A step of the sum is 128 bytes of a row (64 elements of 16 bits, 32 of fp32); a tile is `ROWS` rows
// (i or j) of a step, in LDS in pieces of 16 bytes as it lies in memory:
//   along the sum:  [ROWS][8 pieces], piece c of row r at place c ^ (r / 2 % 8): 16 lanes read a piece of 16 rows at a time, and
//                   two rows cover all banks;
//   across the sum: [64 or 32 steps][ROWS elements], pieces exchanged so that the rows which one instruction reads lie in
//                   different banks.  A fragment then is two transposing reads of four elements (16 bits), or four of one.
typedef __attribute__((address_space(3))) void LdsVoid;
constexpr int kStepBytes = 128, kMaxSplits = 8;
constexpr int kOutOfRange = (int)0x80000000u;  // (a request there touches no memory and returns 0)

struct Operand {
    const void* p;
    long long ld;  // elements between rows in memory
};

// How an operand's rows lie in memory: at whole pieces (requested into LDS), anywhere (through registers: the last piece of a row is
// requested as the row's last 16 bytes and moved into place), or anywhere in rows shorter than a piece or further apart than 32
// bits hold for a tile (element by element).
enum Access : int { WHOLE_PIECES, ANYWHERE, ELEMENTS };

// HIDDEN: the compiler is not to know of requests into LDS (below).
// PAIRED: the operand is two matrices of the same size, one behind the other, and the tile alternates between 16 rows of the first and the
// same 16 rows of the second: then both products of a column end in registers of one lane, 8 apart.
constexpr int kPairedRows = 16;
template <typename T, int ROWS, bool ACROSS, Access ACCESS, int THREADS, int SLOTS, bool HIDDEN, bool PAIRED>
struct Tile {
    static_assert(!(PAIRED && ACROSS), "");
    static constexpr int V = Elem<T>::kVec, kSteps = kStepBytes / (int)sizeof(T);
    static constexpr int kBytes = ROWS * kStepBytes, kPieces = kBytes / 16, kEach = kPieces / THREADS;
    static constexpr int kReads = !ACROSS ? 1 : (sizeof(T) == 2 ? 2 : 4);  // LDS requests of a fragment
    static constexpr int kRowPieces = ACROSS ? ROWS / V : 8;  // pieces of a row as LDS holds them
    static_assert(kEach * THREADS == kPieces, "whole pieces a thread");

    const T* base;
    long long apart;  // PAIRED: elements between a place of the first matrix and the same place of the second
    int offset[kEach];  // bytes from the tile's first element in memory, at the first step
    Words held[SLOTS][ACCESS == WHOLE_PIECES ? 1 : kEach];
    long long ld;
    int valid;  // rows of the tile that exist

    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (!ACROSS) return (row >> 1) & 7;
        if constexpr (sizeof(T) == 4) return kRowPieces >= 16 ? ((row >> 2) & 1) << 3 : 0;
        return kRowPieces >= 16 ? (row & 3) << 2 : (kRowPieces == 8 ? ((row >> 1) & 1) << 2 : 0);
    }
    // thread's e-th piece: its row and piece in memory
    static __device__ __forceinline__ void where(int e, int& row, int& piece) {
        const int at = e * THREADS + (int)threadIdx.x;
        row = at / kRowPieces;
        piece = (at % kRowPieces) ^ swizzle(row);
    }
    // a row of the tile in memory, from the tile's first one; whether thread's e-th piece lies in the second matrix (8 rows a wavefront, all in one)
    static __device__ __forceinline__ int source(int row) { return PAIRED ? row / (2 * kPairedRows) * kPairedRows + row % kPairedRows : row; }
    __device__ __forceinline__ const T* matrix(int e) const {
        if constexpr (!PAIRED) return base;
        return base + ((e * THREADS + wave_first()) / (8 * kPairedRows) % 2 ? apart : 0);  // (a choice of pointers would put the tile into memory)
    }
    // rows first .. of `total` rows (i or j; of each matrix).  What lies past the last row is some other row's: nothing of it is kept.
    __device__ __forceinline__ void init(const Operand& o, long long first, long long total) {
        ld = o.ld;
        valid = (int)min((long long)(PAIRED ? ROWS / 2 : ROWS), total - first);
        // Across the sum, a tile's last piece is read as the row's last 16 bytes, which begin before the tile where it has fewer
        // columns than that: offsets count from there and are never negative.
        const int lead = ACROSS && ACCESS == ANYWHERE ? max(0, V - valid) : 0;
        base = (const T*)o.p + (ACROSS ? first - lead : first * ld);
        if constexpr (PAIRED) apart = total * ld;
        if constexpr (ACCESS != ELEMENTS) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                int row, piece;
                where(e, row, piece);
                if constexpr (ACROSS)  // (pieces past the last column: the last one)
                    offset[e] = (int)(row * ld + min(piece * V, valid - V) + lead) * (int)sizeof(T);
                else
                    offset[e] = (int)(min(source(row), valid - 1) * ld + piece * V) * (int)sizeof(T);
            }
        }
    }
    // requests a piece of the step that begins at `s` of `sum` into LDS (`plane`: elements to the plane of the sum that the step lies in)
    __device__ __forceinline__ void request_piece(char* lds, int s, int sum, long long plane, int e) {
        int row, piece;
        where(e, row, piece);
        const int at = s + (ACROSS ? row : piece * V) < sum ? offset[e] : kOutOfRange;
        char* to = lds + (e * THREADS + wave_first()) * 16;
        const T* from = ACROSS ? base + plane + s * ld : matrix(e) + plane;
        if constexpr (HIDDEN) {
            // The builtin makes the compiler wait for it before every transposing read of LDS, whichever tile that reads; what is in
            // LDS is for meet() to wait for.  (m0, which the compiler sets itself right before each use of its own: where in LDS.  Nothing comes back into registers.)
            const unsigned long long address = (unsigned long long)(uintptr_t)from;
            const Words r = {__builtin_amdgcn_readfirstlane((int)address), __builtin_amdgcn_readfirstlane((int)(address >> 32) & 0xffff), 0x7fffffff,
                             0x00020000};
            // Five wait states: a vector instruction may have written the descriptor's registers just before.  Never remove them.
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(
                             __builtin_amdgcn_readfirstlane((int)(uintptr_t)(LdsVoid*)to)),
                         "v"(at), "s"(r), "s"(ACROSS ? 0 : s * (int)sizeof(T))
                         : "memory");
        } else {
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(from), 0, 0x7fffffff, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsVoid*)to, 16, at, ACROSS ? 0 : s * (int)sizeof(T), 0, 0);
        }
    }
    // requests the tile of a step: into LDS at once, or into the registers of a slot
    template <int SLOT>
    __device__ __forceinline__ void request(char* lds, int s, int sum, long long plane) {
        if constexpr (ACCESS == WHOLE_PIECES) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) request_piece(lds, s, sum, plane, e);
        } else if constexpr (ACCESS == ANYWHERE) {
            // (no branches: then the requests of several steps can be told apart by their number)
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                int row, piece;
                where(e, row, piece);
                const char* from = reinterpret_cast<const char*>(ACROSS ? base + plane + s * ld : matrix(e) + plane);
                int at = offset[e];
                if constexpr (ACROSS) {
                    at -= max(0, s + row - (sum - 1)) * (int)(ld * (int)sizeof(T));  // rows past the sum: the last one
                } else {
                    const int start = s + piece * V;
                    at += (start >= sum ? -piece * V : min(s, sum - V - piece * V)) * (int)sizeof(T);
                }
                held[SLOT][e] = __builtin_bit_cast(Words, load_vec(reinterpret_cast<const T*>(from + (uint32_t)at)));
            }
        } else {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                int row, piece;
                where(e, row, piece);
                const T* p = plane + (ACROSS ? base + (s + row) * ld + piece * V : matrix(e) + min(source(row), valid - 1) * ld + s + piece * V);
                const int n = ACROSS ? (s + row < sum ? valid - piece * V : 0) : sum - (s + piece * V);
                Vec<T> v;
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = k < n ? p[k] : (T)0.0f;
                held[SLOT][e] = __builtin_bit_cast(Words, v);
            }
        }
    }
    static __device__ __forceinline__ int wave_first() { return __builtin_amdgcn_readfirstlane(threadIdx.x & ~63); }
    // the last `n` elements of a piece in the place of its first, 0 behind them
    static __device__ __forceinline__ Words last_first(Words w, int n) {
        const int bits = (V - n) * 8 * (int)sizeof(T);
        unsigned long long lo = ((unsigned long long)(uint32_t)w[1] << 32) | (uint32_t)w[0];
        unsigned long long hi = ((unsigned long long)(uint32_t)w[3] << 32) | (uint32_t)w[2];
        if (bits >= 64) {
            lo = hi >> (bits - 64);
            hi = 0;
        } else {
            lo = (lo >> bits) | (hi << 1 << (63 - bits));
            hi >>= bits;
        }
        return Words{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
    }
    // a slot, whose step began at `s`, into LDS
    template <int SLOT>
    __device__ __forceinline__ void store(char* lds, int s, int sum) {
        if constexpr (ACCESS == ANYWHERE) {
            if (ACROSS && valid < ROWS && valid % V != 0) {
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    int row, piece;
                    where(e, row, piece);
                    if (piece == valid / V) held[SLOT][e] = last_first(held[SLOT][e], valid % V);
                }
            }
            if (s + kSteps > sum) {
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    int row, piece;
                    where(e, row, piece);
                    const int left = sum - s - (ACROSS ? row : piece * V);
                    if (!ACROSS && left > 0 && left < V) held[SLOT][e] = last_first(held[SLOT][e], sum % V);
                    if (left <= 0) held[SLOT][e] = Words{0, 0, 0, 0};
                }
            }
        }
        if constexpr (ACCESS != WHOLE_PIECES) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) *reinterpret_cast<Words*>(lds + (e * THREADS + (int)threadIdx.x) * 16) = held[SLOT][e];
        }
    }
    // the fragment of rows `first` .. `first` + 31, the k-th quarter of the step
    static __device__ __forceinline__ Words fragment(const char* lds, int first, int k) {
        const int lane = threadIdx.x & 63, h = lane >> 5;
        if constexpr (!ACROSS) {
            const int row = first + (lane & 31);
            return *reinterpret_cast<const Words*>(lds + row * 128 + (((2 * k + h) ^ swizzle(lane)) << 4));
        } else if constexpr (sizeof(T) == 2) {
            typedef short S4 __attribute__((ext_vector_type(4)));
            typedef int I2 __attribute__((ext_vector_type(2)));
            I2 half[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int row = 16 * k + 8 * h + 4 * q + ((lane >> 2) & 3), col = first + (lane & 16) + 4 * (lane & 3);
                const char* at = lds + row * (ROWS * 2) + (((col >> 3) ^ swizzle(row)) << 4) + (col & 7) * 2;
                half[q] = __builtin_bit_cast(I2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) S4*)at));
            }
            return Words{half[0][0], half[0][1], half[1][0], half[1][1]};
        } else {
            Words w;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = 8 * k + 4 * h + q, col = first + (lane & 31);
                w[q] = *reinterpret_cast<const int*>(lds + row * (ROWS * 4) + (((col >> 2) ^ swizzle(row)) << 4) + (col & 3) * 4);
            }
            return w;
        }
    }
};

// (A kernel's parameters come in lines of 64 bytes, whose first reading a small call waits for: what a kernel begins with is in the first, what it ends
// with in the second, and partial sums and planes behind them.)
struct ProductParams {
    Operand i, j;
    int rows, cols, sum;  // c is rows x cols
    int tiles_i, tiles_j, splits, split_sum;
    int first;             // the first column of a launch for few rows
    int activation;
    int carry;             // the sum goes on in `partial`: CARRY_FIRST writes it, CARRY_ON adds to what is there
    const float* bias;     // [cols], or NULL
    const void* residual;  // or NULL
    void* out;
    void* preact;          // or NULL
    long long residual_ld, out_ld, preact_ld;
    float* partial;        // splits > 1 or a carry: [splits][rows][cols]
    long long partial_stride;  // from one split's to the next one's
    const float* factor;   // of the sums, or NULL (a power of two: nothing is rounded by it)
    // I in two planes whose products are added, the second i_low elements behind the first: the sum goes over a step of the first and the same step of the
    // second in turn, so that J's steps are in the cache when they are read again.  `plane`: the sum in whole steps (0: one plane).
    int plane;
    long long i_low;
    bool padded_i, padded_j;  // the operand's rows, 16 bytes or more, go on with zeros to whole 16 bytes
};
enum Carry : int { NO_CARRY, CARRY_FIRST, CARRY_ON };

// C neighbouring columns of a row, of which `n` exist; 0 in the place of the others
template <typename T, int C>
using Columns = T __attribute__((ext_vector_type(C)));
template <typename T, int C>
using ColumnsAnywhere = T __attribute__((ext_vector_type(C), aligned(sizeof(T))));
template <typename T, int C>
__device__ __forceinline__ Columns<T, C> get_columns(const void* base, long long ld, long long i, int j, int n) {
    const T* from = (const T*)base + i * ld + j;
    if (n >= C) return *reinterpret_cast<const ColumnsAnywhere<T, C>*>(from);
    Columns<T, C> v;
#pragma unroll
    for (int e = 0; e < C; ++e) v[e] = e < n ? from[e] : (T)0.0f;
    return v;
}
template <typename T, int C>
__device__ __forceinline__ void put_columns(void* base, long long ld, long long i, int j, int n, const float* z) {
    T* to = (T*)base + i * ld + j;
    Columns<T, C> v;
#pragma unroll
    for (int e = 0; e < C; ++e) v[e] = (T)z[e];
    if (n >= C) {
        *reinterpret_cast<ColumnsAnywhere<T, C>*>(to) = v;
    } else {
#pragma unroll
        for (int e = 0; e < C; ++e)
            if (e < n) to[e] = v[e];
    }
}

// all of the workgroup's wavefronts are here, with all but `N` of their requests done and nothing of LDS under way
template <int N>
__device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A workgroup's tile of c is BI x BJ, WI x WJ wavefronts with 32 x 32 pieces of it each, WS times over: those share the quarters of a
// step, and their sums are added at the end.  STAGES steps of both operands lie in LDS or are on their way there;
// what goes through registers does so HOLD steps ahead, LONG: without a branch in sums of more than kLongSteps steps.
constexpr int kLongSteps = 8;
template <int BI, int BJ, int WI, int WJ, int WS, int STAGES>
constexpr int product_lds() {
    constexpr int kStages = STAGES * (BI + BJ) * kStepBytes, kOut = 32 * (32 * (BJ / WJ / 32) * 4 + 16) * WI * WJ * WS;
    return kStages > kOut ? kStages : kOut;
}
// Where a workgroup's tile lies, and what of it a wavefront has: rows i0 + wi .. and columns j0 + wj .. (PAIRED: of the columns of both matrices, in
// turn), with `share` of the sum.
struct Spot {
    int split, tile_i, tile_j, share, wi, wj, wave, lane;
    long long i0, j0;
};
// The sums of workgroup `block`'s tile, in registers as the matrix instructions leave them; LDS is free afterwards.
template <typename T, int BI, int BJ, int WI, int WJ, int WS, int STAGES, Access ACCESS, int HOLD, bool LONG, bool ACROSS_I, bool ACROSS_J,
          bool PAIRED = false, bool PLANES = false>
__device__ __forceinline__ void product_sums(const ProductParams& p, int block, char* lds, Acc (&acc)[BI / WI / 32][BJ / WJ / 32], Spot& spot) {
    constexpr int kThreads = 64 * WI * WJ * WS, NI = BI / WI / 32, NJ = BJ / WJ / 32, kQuarters = 4 / WS;
    constexpr bool ALIGNED = ACCESS == WHOLE_PIECES;
    constexpr bool kHidden = ALIGNED && sizeof(T) == 2 && (ACROSS_I || ACROSS_J);  // transposing reads
    using TileI = Tile<T, BI, ACROSS_I, ACCESS, kThreads, HOLD, kHidden, false>;
    using TileJ = Tile<T, BJ, ACROSS_J, ACCESS, kThreads, HOLD, kHidden, PAIRED>;
    constexpr int kStage = TileI::kBytes + TileJ::kBytes;
    static_assert(ALIGNED || STAGES == 2, "what registers hold needs two tiles");
    static_assert(STAGES > 1 || WS == 1, "");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Workgroups go to the 8 XCDs in turn: each XCD gets a run of tiles, and a run covers 8 tiles of i after 8 tiles of i, so that what
    // runs at one time on an XCD shares its operands' tiles in that XCD's L2.
    const int tiles = p.tiles_i * p.tiles_j, units = tiles * p.splits;
    const int xcd = block % 8, nth = block / 8;
    const int unit = xcd * (units / 8) + min(xcd, units % 8) + nth;
    const int split = unit / tiles, tile = unit % tiles;
    const int band = tile / (8 * p.tiles_j), in_band = tile % (8 * p.tiles_j), high = min(8, p.tiles_i - 8 * band);
    const int tile_i = 8 * band + in_band % high, tile_j = in_band / high;
    const long long i0 = (long long)tile_i * BI, j0 = (long long)tile_j * (PAIRED ? BJ / 2 : BJ);

    TileI ti;
    TileJ tj;
    constexpr int V = Elem<T>::kVec;
    ti.init(p.i, i0, ACROSS_I && p.padded_i ? ((long long)p.rows + V - 1) / V * V : (long long)p.rows);
    tj.init(p.j, j0, ACROSS_J && p.padded_j ? ((long long)p.cols + V - 1) / V * V : (long long)p.cols);
    const int s0 = split * p.split_sum, s1 = min(PLANES ? 2 * p.plane : p.sum, s0 + p.split_sum);
    const int share = wave / (WI * WJ), wi = wave / WJ % WI * (32 * NI), wj = wave % WJ * (32 * NJ);
    spot = {split, tile_i, tile_j, share, wi, wj, wave, lane, i0, j0};

#pragma unroll
    for (int a = 0; a < NI; ++a)
#pragma unroll
        for (int b = 0; b < NJ; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[a][b][v] = 0.0f;

    using std::integral_constant;
    constexpr integral_constant<int, 0> slot0;
    const int steps = (s1 - s0 + TileI::kSteps - 1) / TileI::kSteps;
    // (a step past the last one: requests that touch no memory)
    // where a step begins: in the sum of its plane, the sum's end (or the split's), the plane
    struct Step {
        int s, end;
        long long i_plane;
    };
    auto where = [&](int step) -> Step {
        const int s = s0 + step * TileI::kSteps;
        if constexpr (!PLANES) return {s, s1, 0};
        const int nth = s / TileI::kSteps;
        return {nth / 2 * TileI::kSteps, s < s1 ? p.sum : 0, nth % 2 ? p.i_low : 0};
    };
    auto request_i = [&](int stage, int step, auto slot) {
        const Step at = where(step);
        ti.template request<slot.value>(lds + stage * kStage, at.s, at.end, at.i_plane);
    };
    auto request_j = [&](int stage, int step, auto slot) {
        const Step at = where(step);
        tj.template request<slot.value>(lds + stage * kStage + TileI::kBytes, at.s, at.end, 0);
    };
    // (registers only) a slot's step goes to LDS, for all to read
    auto hand_over = [&](int stage, int step, auto slot) {
        const Step at = where(step);
        ti.template store<slot.value>(lds + stage * kStage, at.s, at.end);
        tj.template store<slot.value>(lds + stage * kStage + TileI::kBytes, at.s, at.end);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (requests into registers stay under way)
    };
    // A step's fragments come a quarter ahead of their instructions, the first quarter's from the next step's tiles: so the barrier
    // that hands these over, and the request for the step after it into the tiles that are done with, lie before the last quarter's
    // instructions.
    Words fi[2][NI], fj[2][NJ];
    auto fragments = [&](int set, int stage, int k) {
        const char* li = lds + stage * kStage;
        k += share * kQuarters;
#pragma unroll
        for (int b = 0; b < NJ; ++b) fj[set][b] = TileJ::fragment(li + TileI::kBytes, wj + 32 * b, k);
#pragma unroll
        for (int a = 0; a < NI; ++a) fi[set][a] = TileI::fragment(li, wi + 32 * a, k);
    };
    auto multiply = [&](int set) {
#pragma unroll
        for (int a = 0; a < NI; ++a)
#pragma unroll
            for (int b = 0; b < NJ; ++b) acc[a][b] = mma<T>(fj[set][b], fi[set][a], acc[a][b]);
    };
    // (hidden requests are where they are written: after every other matrix instruction)
    auto multiply_and = [&](int set, auto requests, auto request_piece) {
        constexpr int kEvery = std::max(1, NI * NJ / requests.value), kAtOnce = (requests.value + NI * NJ - 1) / (NI * NJ);
        int e = 0;
#pragma unroll
        for (int a = 0; a < NI; ++a)
#pragma unroll
            for (int b = 0; b < NJ; ++b) {
                acc[a][b] = mma<T>(fj[set][b], fi[set][a], acc[a][b]);
                if ((a * NJ + b) % kEvery == 0) {
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u)
                        if (e < requests.value) request_piece(e++);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
        for (; e < requests.value; ++e) request_piece(e);
    };
    // One request of LDS after a matrix instruction, and one of memory after every other: a burst of either holds all wavefronts
    // while the matrix cores wait.  `reads` and `requests` are those of the code up to here.
    constexpr int kInstr = NI * NJ * (sizeof(T) == 4 ? 4 : 1);
    auto interleave = [](auto reads, auto requests) {
        constexpr int kPer = (reads.value + kInstr - 1) / kInstr, kEvery = requests.value > 0 ? std::max(1, kInstr / std::max(1, requests.value)) : kInstr + 1;
        constexpr int kPerRequest = (requests.value + kInstr - 1) / kInstr;
#pragma unroll
        for (int q = 0; q < kInstr; ++q) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (q * kPer < reads.value) __builtin_amdgcn_sched_group_barrier(0x100, kPer, 0);
            if (requests.value > 0 && q % kEvery == 0) __builtin_amdgcn_sched_group_barrier(0x010, std::max(1, kPerRequest), 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr integral_constant<int, NI * TileI::kReads + NJ * TileJ::kReads> reads;
    constexpr integral_constant<int, TileI::kEach> requests_i;
    constexpr integral_constant<int, TileJ::kEach> requests_j;
    constexpr int kRequests = TileI::kEach + TileJ::kEach;
    int stage = 0;
    if (steps > 0) {
        if constexpr (STAGES == 1) {  // (a workgroup waits for its step, others beside it work)
            for (int step = 0; step < steps; ++step) {
                if (step > 0) meet<0>();
                request_j(0, step, slot0);
                request_i(0, step, slot0);
                meet<0>();
                fragments(0, 0, 0);
#pragma unroll
                for (int k = 0; k < kQuarters; ++k) {
                    if (k + 1 < kQuarters) fragments((k + 1) & 1, 0, k + 1);
                    multiply(k & 1);
                }
            }
            meet<0>();
        } else if constexpr (ALIGNED) {
            // Step t + STAGES is requested into the tiles of step t as soon as these are done with: J's with the last quarter of step
            // t, I's with the first of step t + 1 (where a wavefront has a quarter alone, both at once).
            constexpr bool kApart = kQuarters > 1;
#pragma unroll
            for (int k = 0; k < STAGES; ++k) {
                request_j(k, k, slot0);
                if (!kApart || k + 1 < STAGES) request_i(k, k, slot0);
            }
            meet<(STAGES - 1) * kRequests - (kApart ? TileI::kEach : 0)>();
            fragments(0, 0, 0);
            for (int step = 0; step < steps; ++step) {
                const int next = stage + 1 == STAGES ? 0 : stage + 1;
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 0; k + 1 < kQuarters; ++k) {
                    const int last = stage == 0 ? STAGES - 1 : stage - 1;
                    const Step at = where(step + STAGES - 1);
                    if (kApart && k == 0 && !kHidden) request_i(last, step + STAGES - 1, slot0);
                    fragments((k + 1) & 1, stage, k + 1);
                    if (kApart && k == 0 && kHidden) {
                        multiply_and(0, requests_i, [&](int e) { ti.request_piece(lds + last * kStage, at.s, at.end, at.i_plane, e); });
                    } else {
                        multiply(k & 1);
                        if (kApart && k == 0)
                            interleave(reads, requests_i);
                        else
                            interleave(reads, slot0);
                    }
                }
                meet<(STAGES - 2) * kRequests>();
                if (!kHidden || !kApart) request_j(stage, step + STAGES, slot0);
                if (!kApart) request_i(stage, step + STAGES, slot0);
                fragments(kQuarters & 1, next, 0);
                if constexpr (kHidden && kApart) {
                    const Step at = where(step + STAGES);
                    multiply_and((kQuarters - 1) & 1, requests_j, [&](int e) {
                        tj.request_piece(lds + stage * kStage + TileI::kBytes, at.s, at.end, 0, e);
                    });
                } else {
                    multiply((kQuarters - 1) & 1);
                    if constexpr (kApart) interleave(reads, requests_j);
                }
                if constexpr (kQuarters == 1) {  // (registers have no index: the next step's fragments take the place of this one's)
#pragma unroll
                    for (int a = 0; a < NI; ++a) fi[0][a] = fi[1][a];
#pragma unroll
                    for (int b = 0; b < NJ; ++b) fj[0][b] = fj[1][b];
                }
                stage = next;
            }
            meet<0>();
        } else {
            auto each = [&](auto f) {
                f(integral_constant<int, 0>());
                if constexpr (HOLD == 4) f(integral_constant<int, 1>()), f(integral_constant<int, 2>()), f(integral_constant<int, 3>());
            };
            static_assert(HOLD == 1 || HOLD == 4, "");
            auto request_both = [&](int step, auto slot) { request_i(0, step, slot), request_j(0, step, slot); };
            // `slot`: step % HOLD
            enum { NOTHING, IF_ANY, ALWAYS };
            constexpr integral_constant<int, NOTHING> nothing;
            constexpr integral_constant<int, IF_ANY> if_any;
            constexpr integral_constant<int, ALWAYS> always;
            auto advance = [&](int step, auto slot, auto more) {
                const int next = stage ^ 1;
                constexpr integral_constant<int, (slot.value + 1) % HOLD> next_slot;
#pragma unroll
                for (int k = 0; k + 1 < kQuarters; ++k) {
                    fragments((k + 1) & 1, stage, k + 1);
                    multiply(k & 1);
                    interleave(reads, slot0);
                }
                if (more.value == ALWAYS || step + 1 < steps) {
                    hand_over(next, step + 1, next_slot);
                    if (more.value == ALWAYS || (more.value == IF_ANY && step + 1 + HOLD < steps)) request_both(min(step + 1 + HOLD, steps - 1), next_slot);
                    fragments(kQuarters & 1, next, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                multiply((kQuarters - 1) & 1);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (kQuarters == 1) {
#pragma unroll
                    for (int a = 0; a < NI; ++a) fi[0][a] = fi[1][a];
#pragma unroll
                    for (int b = 0; b < NJ; ++b) fj[0][b] = fj[1][b];
                }
                stage = next;
            };
            // LONG: in long sums every step requests another without a branch, the last ones the last step again.  Where a request may or
            // may not have been made the compiler does not know how many came after the one that it waits for, and waits for
            // them all.
            int step = 0;
            if (LONG && steps > kLongSteps) {
                each([&](auto k) { request_both(k.value, k); });
                hand_over(0, 0, slot0);
                request_both(HOLD, slot0);
                fragments(0, 0, 0);
                for (; step + HOLD < steps; step += HOLD) each([&](auto k) { advance(step + k.value, k, always); });
                each([&](auto k) {
                    if (step + k.value < steps) advance(step + k.value, k, nothing);
                });
            } else {
                each([&](auto k) {
                    if (k.value < steps) request_both(k.value, k);
                });
                hand_over(0, 0, slot0);
                if (HOLD < steps) request_both(HOLD, slot0);
                fragments(0, 0, 0);
                for (; step < steps; step += HOLD)
                    each([&](auto k) {
                        if (step + k.value < steps) advance(step + k.value, k, if_any);
                    });
            }
        }
    }
    __syncthreads();
}

// ---- few rows (16 at most): bound by the weights' bytes.  A wavefront has 16 outputs and a share of the sum; 64 bytes of 16 weight
// rows are one request of it and one matrix instruction (four in fp32), and eight requests of each operand are under way at a
// time.  A workgroup's 8 wavefronts are SHARES of the sum by 8 / SHARES groups of outputs: 8, or 2 where a sum is so short that eight
// requests are half of it (1 x 512 x 32768 in 16 bits 7.4 us instead of 10.7, 1 x 128 x 65536 6.4 instead of 12.2).  Nothing goes
// through LDS but the wavefronts' sums, and rows may lie anywhere.  1 x 4096 x 4096 bf16 8.1 us (33.6 MB, half of it the launch and the
// first requests' latency), 1 x 8192 x 28672 77 us (6.1 TB/s).
constexpr int kFewRows = 16, kFewWaves = 8, kFewOutputs = 16, kFewAtOnce = 8;
typedef float Acc4 __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ Acc4 mma16(Vec<T> j, Vec<T> i, Acc4 c) {
    if constexpr (std::is_same_v<T, __bf16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(j, i, c, 0, 0, 0);
    } else if constexpr (std::is_same_v<T, _Float16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(j, i, c, 0, 0, 0);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(j[e], i[e], c, 0, 0, 0);
        return c;
    }
}

// The sums of a wavefront's 16 rows of weights (`w`: the lane's, `x`: its row of the input) over its share, all shares' in share 0
template <typename T, int SHARES>
__device__ __forceinline__ Acc4 few_rows_sums(const ProductParams& p, const T* w, const T* x) {
    constexpr int V = Elem<T>::kVec, kChunk = 4 * V;
    __shared__ Acc4 lds[kFewWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, share = wave % SHARES, start = (lane >> 4) * V;
    const int chunks = (p.sum + kChunk - 1) / kChunk, each = (chunks + SHARES - 1) / SHARES;
    const int c0 = share * each, c1 = min(chunks, c0 + each), whole = min(c1, p.sum / kChunk);
    Acc4 acc = Acc4{0.0f, 0.0f, 0.0f, 0.0f};
    int c = c0;
    auto batch = [&](auto count) {
        constexpr int N = count.value;
        Vec<T> fw[N], fx[N];
#pragma unroll
        for (int u = 0; u < N; ++u) fw[u] = load_vec(w + (c + u) * kChunk + start);
#pragma unroll
        for (int u = 0; u < N; ++u) fx[u] = load_vec(x + (c + u) * kChunk + start);
        __builtin_amdgcn_sched_barrier(0);  // (all requests first: the compiler would rather save registers)
#pragma unroll
        for (int u = 0; u < N; ++u) acc = mma16<T>(fw[u], fx[u], acc);
        c += N;
    };
    while (c + kFewAtOnce <= whole) batch(std::integral_constant<int, kFewAtOnce>());
    if (c + 4 <= whole) batch(std::integral_constant<int, 4>());
    if (c + 2 <= whole) batch(std::integral_constant<int, 2>());
    if (c + 1 <= whole) batch(std::integral_constant<int, 1>());
    if (c < c1) {  // the end of the sum, no whole chunk
        const int k0 = c * kChunk + start;
        auto get = [&](const T* q) {
            if (k0 + V <= p.sum) return load_vec(q + k0);
            Vec<T> v;
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = k0 + e < p.sum ? q[k0 + e] : (T)0.0f;
            return v;
        };
        acc = mma16<T>(get(w), get(x), acc);
    }
    lds[wave][lane] = acc;
    __syncthreads();
    if (share == 0) {
#pragma unroll
        for (int k = 1; k < SHARES; ++k) acc += lds[wave + k][lane];
    }
    return acc;
}

// The tile that a product is cut into, how often its sum is split, and its launch.
//
// The plan is the one with the shortest estimate, from what the tiles measured (us): a step of the sum takes `step` when a
// compute unit has one tile to work on (latency, then), `more` for each when it has several, `tile` besides for every tile after
// the first, and a launch `start`.  A split sum is joined by a kernel of its own: 2.3 (3, where splits of rows that lie anywhere start)
// and the partial sums' bytes, out and back in, at 4 TB/s.
enum Cut : int { CUT_256, CUT_128, CUT_128_DEEP, CUT_64, CUT_32, CUTS };
struct CutCost {
    int size;
    float start, tile, step, more;
};
// Measured in tiles of 256 / 128 / 128 deep / 64 / 32, rows x inputs x outputs, 16-bit types: 8192 x 4096 x 4096 221 / 279 / 315 / 455 / 786,
// 8192 x 4096 x 1024 100 / 74 / 82 / 123 / 210, 4096 x 8192 x 1024 187 / 110 / 76 / 120 / 203, 2048^3 43 / 27 / 23 / 32 / 59, 1024^3 26 / 15 / 12 / 7.9 /
// 11.7, 64 x 4096 x 4096 67 / 42 / 27 / 19 / 11, 512^3 17 / 8.9 / 9.0 / 5.5 / 4.4.  fp32: 4000 x 2000 x 2000 471 / 253 / 261 / 278 / 372, 1000^3 243 / 72 /
// 69 / 24 / 29, 64 x 1024 x 1024 238 / 71 / 68 / 22 / 11.  Rows that lie anywhere: 8192 x 4096 x 4096 - / 346 / - / 584 / 943, 4001 x
// 1999 x 1001 - / 38 / - / 55 / 86, 1000 x 1001 x 999 - / 21 / - / 9.9 / 16, 77 x 1023 x 1537 - / 19 / - / 9.1 / 6.2.  (The estimates take no
// account of what the tiles write: the gradients of fp32 59 x 7192 -> 4060, 117 MB of them the weight's, take 124 us.)
constexpr CutCost kCuts16[CUTS] = {{256, 9.0f, 4.0f, 1.4f, 1.6f}, {128, 6.0f, 1.5f, 0.8f, 0.52f}, {128, 6.0f, 3.0f, 0.4f, 0.55f}, {64, 3.5f, 1.0f, 0.27f, 0.21f}, {32, 3.2f, 0.5f, 0.135f, 0.11f}};
constexpr CutCost kCuts32[CUTS] = {{256, 12.0f, 4.0f, 7.4f, 7.4f}, {128, 6.0f, 1.5f, 2.2f, 1.95f}, {128, 6.0f, 3.0f, 2.0f, 2.05f}, {64, 3.5f, 1.0f, 0.67f, 0.55f}, {32, 3.2f, 0.5f, 0.25f, 0.22f}};
constexpr CutCost kCutsAnywhere[CUTS] = {{}, {128, 6.0f, 0.0f, 1.0f, 0.7f}, {}, {64, 3.2f, 1.2f, 0.42f, 0.33f}, {32, 3.2f, 0.5f, 0.18f, 0.165f}};
constexpr float kReadRate = 5.5e6f;  // bytes of operands in a us that no tile exceeds where they are read once
struct Plan {
    Cut cut;
    int splits;
    float time;
};
// `fine`, for what the linear layer does not launch: a compute unit has two workgroups at a time of all tiles but the two that take its shared memory, so that
// of an odd number of them the last one works alone (losses, bf16: 300 x 4096 -> 32000 classes 135 us in tiles of 128, three a compute unit, 105 in
// tiles of 256; 333 x 1024 -> 32000 39 and 33; 2000 x 512 -> 5000 23.0 and 21.0); and a sum may be split into any number of parts (loss's
// step of 3630 x 1072 -> 38878 bf16 1445 us, 1580 with powers of two; gradients of gated 1500 x 2048 -> 2 x 5600 205 and 224).
inline Plan plan_product(int rows, int cols, int sum, int size, bool vectors, size_t workspace_bytes, Cut largest = CUT_256, bool fine = false) {
    const int steps = (int)(((long long)sum * size + kStepBytes - 1) / kStepBytes);
    const float read = ((float)rows + (float)cols) * (float)sum * (float)size / kReadRate;
    Plan best = {CUT_32, 1, 0.0f};
    for (int c = largest; c < CUTS; ++c) {
        CutCost cost = vectors ? (size == 4 ? kCuts32[c] : kCuts16[c]) : kCutsAnywhere[c];
        if (cost.size == 0) continue;
        if (!vectors && size == 4) cost.step = std::max(cost.step, kCuts32[c].step), cost.more = std::max(cost.more, kCuts32[c].more);
        const float tiles = (float)((rows + cost.size - 1) / cost.size) * (float)((cols + cost.size - 1) / cost.size);
        for (int k = 1; k <= kMaxSplits && (k == 1 || steps >= 4 * k); k = fine ? k + 1 : 2 * k) {
            const size_t partial = k > 1 ? (size_t)k * rows * cols * sizeof(float) : 0;
            if (partial > workspace_bytes) break;
            const float rounds = std::ceil(tiles * (float)k / (float)kComputeUnits);
            const bool alone = fine && rounds > 1.0f && std::fmod(rounds, 2.0f) == 1.0f && c != CUT_256 && c != CUT_128_DEEP;
            const float each = std::max(cost.step, rounds * cost.more) + (alone ? std::max(0.0f, cost.step - cost.more) : 0.0f);
            const float time = cost.start + (rounds - 1.0f) * cost.tile + std::max((float)((steps + k - 1) / k) * each, read) + (k > 1 ? (vectors ? 2.3f : 3.0f) + (float)partial * 2.0f / 4.0e6f : 0.0f);
            if (best.time == 0.0f || time < best.time) best = {(Cut)c, k, time};
        }
    }
    return best;
}

// The kernel for few rows instead: the wavefronts' shares of a sum, and the estimate to compare with a plan's.  A chunk of 64 bytes
// costs a wavefront a latency, and the compute unit its requests where several workgroups have one; the rows of x are read again by every
// workgroup.  Measured, this kernel / tiles, 16-bit types: 1 x 4096 x 4096 8.1 / 9.9, 16 x 4096 x 4096 10.3 / 10.5, 4 x 8192 x 28672 80 / 91,
// 16 x 8192 x 28672 108 / 89, 1 x 2048 x 8192 9.8 / 7.8, 1 x 16384 x 512 19.5 / 9.5; fp32: 1 x 4096 x 4096 15.8 / 21.3, 8 x 16384 x 64 47 / 21;
// rows that lie anywhere: 1 x 999 x 1001 4.9 / 5.6, 8 x 4095 x 4097 31 / 15, 4 x 8191 x 20001 182 / 109.
inline int few_shares(int cols, int sum, int size) { return sum * size <= 1024 && cols > 64 * (kComputeUnits - 1) ? 2 : 8; }
inline float few_time(int rows, int cols, int sum, int size, bool vectors) {
    const int shares = few_shares(cols, sum, size), outputs = kFewOutputs * kFewWaves / shares;
    const float blocks = (float)(cols / outputs + (cols % outputs != 0)) / (float)kComputeUnits;
    const float chunks = std::ceil((float)sum * (float)size / (64.0f * (float)shares)), n = (float)rows;
    const float latency = vectors ? 0.25f + 0.01f * n : 0.45f + 0.035f * n, more = vectors ? 0.2875f + 0.0095f * n : 0.85f + 0.1f * n;
    return 2.4f + chunks * std::max(latency, blocks * more) + blocks * (shares == 2 ? 0.7f : 1.4f);
}

// A product of few rows whose workgroups have `outputs` columns each: go(shares, grid, its parameters), columns beyond a launch's threads (2^27 with 16 a workgroup) in
// launches of their own.
template <typename F>
void by_few_columns(ProductParams p, int shares, int outputs, F&& go) {
    const int blocks = p.cols / outputs + (p.cols % outputs != 0), most = (int)(kMaxThreads / (64 * kFewWaves));
    for (int first = 0; first < blocks; first += most) {
        p.first = first * outputs;
        const dim3 grid((unsigned)std::min(most, blocks - first));
        if (shares == 8)
            go(std::integral_constant<int, 8>(), grid, p);
        else
            go(std::integral_constant<int, 2>(), grid, p);
    }
}

template <typename T, bool ACROSS_I, bool ACROSS_J>
Access access_of(const ProductParams& p) {
    auto of = [](const Operand& o, int rows, int sum, bool across, bool padded) {
        int row = across ? rows : sum;
        if (padded) row = (row + Elem<T>::kVec - 1) / Elem<T>::kVec * Elem<T>::kVec;
        if (row < Elem<T>::kVec || o.ld * 256 * (long long)sizeof(T) > 0x7fffffffLL) return ELEMENTS;
        return (uintptr_t)o.p % 16 == 0 && o.ld * sizeof(T) % 16 == 0 && row % Elem<T>::kVec == 0 ? WHOLE_PIECES : ANYWHERE;
    };
    return std::max(of(p.i, p.rows, p.sum, ACROSS_I, p.padded_i), of(p.j, p.cols, p.sum, ACROSS_J, p.padded_j));
}
// f(tile, wavefronts of i, of j, of the sum, stages, access, steps held, long sums) with the constants of a tile's kernel (product_sums)
// Short sums of many tiles: a tile's life is its launch, its first requests and what follows its sums rather than these, and so several workgroups a compute unit do more
// than steps under way.  Tiles of 128 with one step in LDS, four of them at a time (losses, bf16: 3043 x 32 -> 17021 classes 23 us, 32 in tiles
// of 256; 4096 x 512 -> 65536, 8 steps, 272 and 282; 8192 x 1024 -> 32768, 16 steps, 495 and 472; 200 x 512 -> 20000, 314 tiles, 16.7 and 16.1).
constexpr int kShortSteps = 8, kShortTiles = 3 * kComputeUnits / 2;
inline bool short_sum(Access access, int rows, int cols, int sum, int size, int steps = kShortSteps) {
    const long long tiles = ((rows - 1) / 128 + 1LL) * ((cols - 1) / 128 + 1);
    return access == WHOLE_PIECES && (long long)sum * size <= steps * kStepBytes && tiles >= kShortTiles;
}
constexpr int short_waves(int waves, int stages) { return stages == 1 ? 4 : (waves + 3) / 4; }  // wavefronts a SIMD that registers do for

template <typename F>
void by_tile(Access access, Cut cut, bool brief, F&& f) {
    constexpr std::integral_constant<int, 256> n256;
    constexpr std::integral_constant<int, 128> n128;
    constexpr std::integral_constant<int, 64> n64;
    constexpr std::integral_constant<int, 32> n32;
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 2> two;
    constexpr std::integral_constant<int, 4> four;
    constexpr std::integral_constant<int, 8> eight;
    constexpr std::true_type yes;
    constexpr std::false_type no;
    constexpr std::integral_constant<Access, WHOLE_PIECES> pieces;
    constexpr std::integral_constant<Access, ANYWHERE> anywhere;
    constexpr std::integral_constant<Access, ELEMENTS> elements;
    if (access == WHOLE_PIECES) {
        if (brief) return f(n128, two, two, one, one, pieces, one, no);
        switch (cut) {
            case CUT_256: return f(n256, two, four, one, two, pieces, one, no);
            case CUT_128: return f(n128, two, two, one, two, pieces, one, no);
            case CUT_128_DEEP: return f(n128, two, two, two, four, pieces, one, no);
            case CUT_64: return f(n64, two, two, two, four, pieces, one, no);
            default: return f(n32, one, one, four, eight, pieces, one, no);
        }
    }
    if (access == ELEMENTS) return f(n32, one, one, four, two, elements, one, no);
    switch (cut) {
        case CUT_128: return f(n128, two, two, one, two, anywhere, one, no);
        case CUT_64: return f(n64, two, two, two, two, anywhere, four, no);
        default: return f(n32, one, one, four, two, anywhere, four, yes);
    }
}
inline void cut_product(ProductParams& p, int size, int steps_size, int splits, float* workspace) {
    p.tiles_i = (p.rows + size - 1) / size;
    p.tiles_j = (p.cols + size - 1) / size;
    const int steps = p.plane ? 2 * p.plane / steps_size : (p.sum + steps_size - 1) / steps_size;
    p.split_sum = std::max(1, (steps + splits - 1) / splits) * steps_size;
    p.splits = std::max(1, ((p.plane ? 2 * p.plane : p.sum) + p.split_sum - 1) / p.split_sum);
    p.partial = workspace;
    p.partial_stride = (long long)p.rows * p.cols;
}

// The sums of wavefronts that shared a tile's sum, in those of share 0; all of the workgroup call it.
template <int WI, int WJ, int WS, int NI, int NJ>
__device__ __forceinline__ void join_shares(Acc (&acc)[NI][NJ], char* lds, const Spot& spot) {
    if constexpr (WS > 1) {
        float4* mine = reinterpret_cast<float4*>(lds) + spot.wave % (WI * WJ) * (4 * NI * NJ * 64) + spot.lane;
        constexpr int kShare = WI * WJ * 4 * NI * NJ * 64;
        if (spot.share > 0) {
#pragma unroll
            for (int a = 0; a < NI; ++a)
#pragma unroll
                for (int b = 0; b < NJ; ++b)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        mine[(spot.share - 1) * kShare + ((a * NJ + b) * 4 + q) * 64] =
                            make_float4(acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]);
        }
        __syncthreads();
        if (spot.share == 0) {
#pragma unroll
            for (int w = 0; w + 1 < WS; ++w)
#pragma unroll
                for (int a = 0; a < NI; ++a)
#pragma unroll
                    for (int b = 0; b < NJ; ++b)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float4 o = mine[w * kShare + ((a * NJ + b) * 4 + q) * 64];
                            acc[a][b][4 * q] += o.x, acc[a][b][4 * q + 1] += o.y, acc[a][b][4 * q + 2] += o.z, acc[a][b][4 * q + 3] += o.w;
                        }
        }
        __syncthreads();
    }
}

// ---- passes over an output's gradient (dz): a thread has one vector of 16 bytes of columns and goes down its share of the rows; the workgroups' column
// sums are joined afterwards, always in the same order.
constexpr int kDzThreads = 256;
// Rows that one thread takes, and the parts that a column's sum falls into (a part a workgroup).
inline int dz_lanes(int vectors) { return vectors >= kDzThreads ? kDzThreads : vectors; }  // of a workgroup, side by side
inline int dz_rows(int rows, int vectors, bool active) {
    const long long threads = 1024LL * kComputeUnits;  // four workgroups a compute unit
    const int each = (int)std::max(8LL, ((long long)rows * vectors + threads - 1) / threads), deep = kDzThreads / dz_lanes(vectors);
    // one part needs no join: 16 rows a thread with their activation's slopes, 32 without, take less time than that launch (one
    // workgroup with 32 rows of GELU a thread: gradients of 64 x 1024 -> 1024 30.5 us, 18.9 with a join; 36 x 860 -> 489
    // fp32 without an activation 13.3 in one part, 13.9 with a join, 32 x 512 -> 1024 bf16 11.8 and 13.1)
    return rows <= (active ? 16 : 32) * deep ? std::max(each, (rows + deep - 1) / deep) : each;
}
inline int dz_parts(int rows, int vectors, bool active) {
    const int deep = kDzThreads / dz_lanes(vectors) * dz_rows(rows, vectors, active);
    return (rows + deep - 1) / deep;
}
inline int out_vectors(int out_features, int dtype) { return (out_features + (int)(16 / dtype_bytes(dtype)) - 1) / (int)(16 / dtype_bytes(dtype)); }
inline size_t whole_lines(size_t bytes) { return (bytes + 255) / 256 * 256; }

// ---- copies of rows that lie anywhere.  A tile of such rows takes 1.6 times as long, so that a large product is faster on a copy at whole 16 bytes, zeros
// behind the rows' ends: a gated product bf16 8192 x 4095 -> 2 x 8191 951 us with both operands copied and 1588 without, 8192 x 4096 -> 2 x 4096 with rows
// 3 elements apart 464 and 676.  A copy moves 4 TB/s or more.
template <typename T>
bool lies_anywhere(const Operand& o, int n) { return n % Elem<T>::kVec != 0 || (uintptr_t)o.p % 16 != 0 || o.ld * (long long)sizeof(T) % 16 != 0; }
inline long long packed_ld(int n, int size) { return ((long long)n * size + 15) / 16 * 16 / size; }
inline size_t packed_bytes(long long rows, int n, int size) { return whole_lines((size_t)rows * packed_ld(n, size) * size); }
inline float pack_time(size_t bytes) { return 2.5f + (float)bytes * 2.0f / 4.0e6f; }
// (linear.hip)  the copy
Operand launch_pack(int dtype, const Operand& o, long long rows, int n, void* to, hipStream_t stream);

// ---- (linear.hip)  dx = d w and dw = d^T x, each where it has an `out`; with dx.carry its sum stays in its `partial`, whose number of splits is
// dx.splits.  The workspace is for split sums (gradient_product_bytes; without one none is split).
size_t gradient_product_bytes(int rows, int in_features, int out_features, int dtype, bool together = false);
// `together`: both in one launch of large tiles, wide tiles for few rows, tiles for short sums and fine plans, too, where these take less time.
int launch_gradient_products(int dtype, const ProductParams& dx, const ProductParams& dw, float* workspace, size_t workspace_bytes, hipStream_t stream,
                             bool together = false);
// ---- (few_gradients.hip)  the same for kFewGradientRows rows at most and d in fp32, [outs][kFewGradientRows] with zeros behind the last row; `partial` holds few_gradients_bytes
constexpr int kFewGradientRows = 4;
size_t few_gradients_bytes(int rows, int in_features, int outs, int dtype);
int launch_few_gradients(int dtype, const float* d, int rows, int in_features, int outs, const Operand& weight, const Operand& input, void* dx, long long dx_ld,
                         void* dw, long long dw_ld, float* partial, hipStream_t stream);

// ---- (linear.hip)  a carried sum -> dx.out
int launch_carried_sum(int dtype, const ProductParams& dx, hipStream_t stream);
// out[n] = the sums of `parts` rows of n, in one order
void launch_column_join(const float* sums, float* out, int parts, int n, hipStream_t stream);

}  // namespace head
}  // namespace tcbnn
