// Linear layers and their gradients (tcbnn_linear_forward / _backward):  z = x w^T + b,  y = act(z) + r;
// dz = dy act'(z),  dx = dz w,  dw = dz^T x,  db = column sums of dz.
//
// All three products are one kernel: c[i][j] = sum over s of I(i, s) J(j, s), where an operand lies in memory either along the
// sum (x and w of the forward product: rows of s) or across it (w of dx, dz and x of dw: a row for every s).
//
// Large products are bound by the matrix instructions, as far as power and the barriers between steps let them run: 8192 x 4096 x
// 4096 in bf16 takes 222 us (1.24 PFLOP/s), 254 with bias, GELU, residual and z kept, because 134 MB more of traffic and the
// activations follow the tiles' last steps; 8192^3 811 us (1.36 PFLOP/s); fp32 4096^3 949 us (145 TFLOP/s).  Of the gradients
// of 8192 x 4096 x 1024 dx takes 83 us and dw 86 (0.8 PFLOP/s): operands across the sum need twice the LDS requests.  Rows that lie
// anywhere go through registers, 348 us instead of 222.  Small products are bound by a launch and the latency of their steps,
// products of few rows by the weights' bytes.
#include <cmath>

#include "head.h"

namespace tcbnn {
namespace {

using namespace head;

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
constexpr int kStepBytes = 128;
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
template <typename T, int ROWS, bool ACROSS, Access ACCESS, int THREADS, int SLOTS, bool HIDDEN>
struct Tile {
    static constexpr int V = Elem<T>::kVec, kSteps = kStepBytes / (int)sizeof(T);
    static constexpr int kBytes = ROWS * kStepBytes, kPieces = kBytes / 16, kEach = kPieces / THREADS;
    static constexpr int kReads = !ACROSS ? 1 : (sizeof(T) == 2 ? 2 : 4);  // LDS requests of a fragment
    static constexpr int kRowPieces = ACROSS ? ROWS / V : 8;  // pieces of a row as LDS holds them
    static_assert(kEach * THREADS == kPieces, "whole pieces a thread");

    const T* base;
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
    // rows first .. of `total` rows (i or j).  What lies past the last row is some other row's: nothing of it is kept.
    __device__ __forceinline__ void init(const Operand& o, long long first, long long total) {
        ld = o.ld;
        valid = (int)min((long long)ROWS, total - first);
        // Across the sum, a tile's last piece is read as the row's last 16 bytes, which begin before the tile where it has fewer
        // columns than that: offsets count from there and are never negative.
        const int lead = ACROSS && ACCESS == ANYWHERE ? max(0, V - valid) : 0;
        base = (const T*)o.p + (ACROSS ? first - lead : first * ld);
        if constexpr (ACCESS != ELEMENTS) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                int row, piece;
                where(e, row, piece);
                if constexpr (ACROSS)  // (pieces past the last column: the last one)
                    offset[e] = (int)(row * ld + min(piece * V, valid - V) + lead) * (int)sizeof(T);
                else
                    offset[e] = (int)(min(row, valid - 1) * ld + piece * V) * (int)sizeof(T);
            }
        }
    }
    // requests a piece of the step that begins at `s` of `sum` into LDS
    __device__ __forceinline__ void request_piece(char* lds, int s, int sum, int e) {
        int row, piece;
        where(e, row, piece);
        const int at = s + (ACROSS ? row : piece * V) < sum ? offset[e] : kOutOfRange;
        char* to = lds + (e * THREADS + wave_first()) * 16;
        const T* from = ACROSS ? base + s * ld : base;
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
    __device__ __forceinline__ void request(char* lds, int s, int sum) {
        if constexpr (ACCESS == WHOLE_PIECES) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) request_piece(lds, s, sum, e);
        } else if constexpr (ACCESS == ANYWHERE) {
            // (no branches: then the requests of several steps can be told apart by their number)
            const char* from = reinterpret_cast<const char*>(ACROSS ? base + s * ld : base);
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                int row, piece;
                where(e, row, piece);
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
                const T* p = ACROSS ? base + (s + row) * ld + piece * V : base + min(row, valid - 1) * ld + s + piece * V;
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

struct ProductParams {
    Operand i, j;
    int rows, cols, sum;  // c is rows x cols
    int tiles_i, tiles_j, splits, split_sum;
    int activation;
    const float* bias;     // [cols], or NULL
    const void* residual;  // or NULL
    void* out;
    void* preact;          // or NULL
    long long residual_ld, out_ld, preact_ld;
    float* partial;        // splits > 1: [splits][rows][cols]
};

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
// their z -> the outputs
template <typename T, int C>
__device__ __forceinline__ void finish(const ProductParams& p, long long i, int j, int n, const float* bias, Columns<T, C> residual, float* z) {
#pragma unroll
    for (int e = 0; e < C; ++e) z[e] += bias[e];
    if (p.preact) put_columns<T, C>(p.preact, p.preact_ld, i, j, n, z);
    by_activation(p.activation, [&](auto act) {
#pragma unroll
        for (int e = 0; e < C; ++e) z[e] = activate<T, act.value>(z[e]);
    });
    if (p.residual) {
#pragma unroll
        for (int e = 0; e < C; ++e) z[e] += (float)residual[e];
    }
    put_columns<T, C>(p.out, p.out_ld, i, j, n, z);
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
template <typename T, int BI, int BJ, int WI, int WJ, int WS, int STAGES, Access ACCESS, int HOLD, bool LONG, bool ACROSS_I, bool ACROSS_J>
__device__ __forceinline__ void product(const ProductParams& p, int block, char* lds) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass leaves a kernel's stub out where it instantiates a tile's requests twice)
    constexpr int kThreads = 64 * WI * WJ * WS, NI = BI / WI / 32, NJ = BJ / WJ / 32, V = Elem<T>::kVec, kQuarters = 4 / WS;
    constexpr bool ALIGNED = ACCESS == WHOLE_PIECES;
    constexpr bool kHidden = ALIGNED && sizeof(T) == 2 && (ACROSS_I || ACROSS_J);  // transposing reads
    using TileI = Tile<T, BI, ACROSS_I, ACCESS, kThreads, HOLD, kHidden>;
    using TileJ = Tile<T, BJ, ACROSS_J, ACCESS, kThreads, HOLD, kHidden>;
    constexpr int kStage = TileI::kBytes + TileJ::kBytes;
    // a wavefront's 32 rows of c on their way out, 16 bytes between rows
    constexpr int kOutRow = 32 * NJ * 4 + 16, kOutWave = 32 * kOutRow;
    static_assert(ALIGNED || STAGES == 2, "what registers hold needs two tiles");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Workgroups go to the 8 XCDs in turn: each XCD gets a run of tiles, and a run covers 8 tiles of i after 8 tiles of i, so that what
    // runs at one time on an XCD shares its operands' tiles in that XCD's L2.
    const int tiles = p.tiles_i * p.tiles_j, units = tiles * p.splits;
    const int xcd = block % 8, nth = block / 8;
    const int unit = xcd * (units / 8) + min(xcd, units % 8) + nth;
    const int split = unit / tiles, tile = unit % tiles;
    const int band = tile / (8 * p.tiles_j), in_band = tile % (8 * p.tiles_j), high = min(8, p.tiles_i - 8 * band);
    const long long i0 = (long long)(8 * band + in_band % high) * BI, j0 = (long long)(in_band / high) * BJ;

    TileI ti;
    TileJ tj;
    ti.init(p.i, i0, p.rows);
    tj.init(p.j, j0, p.cols);
    const int s0 = split * p.split_sum, s1 = min(p.sum, s0 + p.split_sum);
    const int share = wave / (WI * WJ), wi = wave / WJ % WI * (32 * NI), wj = wave % WJ * (32 * NJ);

    Acc acc[NI][NJ];
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
    auto request_i = [&](int stage, int step, auto slot) { ti.template request<slot.value>(lds + stage * kStage, s0 + step * TileI::kSteps, s1); };
    auto request_j = [&](int stage, int step, auto slot) {
        tj.template request<slot.value>(lds + stage * kStage + TileI::kBytes, s0 + step * TileI::kSteps, s1);
    };
    // (registers only) a slot's step goes to LDS, for all to read
    auto hand_over = [&](int stage, int step, auto slot) {
        ti.template store<slot.value>(lds + stage * kStage, s0 + step * TileI::kSteps, s1);
        tj.template store<slot.value>(lds + stage * kStage + TileI::kBytes, s0 + step * TileI::kSteps, s1);
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
        if constexpr (ALIGNED) {
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
                    const int last = stage == 0 ? STAGES - 1 : stage - 1, s = s0 + (step + STAGES - 1) * TileI::kSteps;
                    if (kApart && k == 0 && !kHidden) request_i(last, step + STAGES - 1, slot0);
                    fragments((k + 1) & 1, stage, k + 1);
                    if (kApart && k == 0 && kHidden) {
                        multiply_and(0, requests_i, [&](int e) { ti.request_piece(lds + last * kStage, s, s1, e); });
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
                    multiply_and((kQuarters - 1) & 1, requests_j, [&](int e) {
                        tj.request_piece(lds + stage * kStage + TileI::kBytes, s0 + (step + STAGES) * TileI::kSteps, s1, e);
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

    // ---- out: 32 rows of the wavefront at a time through LDS, so that a row leaves in whole runs of 64 bytes or more.  Wavefronts
    // that shared the sum take a share of the rows each.
    char* mine = lds + wave * kOutWave;
    const char* first_share = lds + wave % (WI * WJ) * kOutWave;
    constexpr int kPerRow = 32 * NJ / V, kShareRows = 32 / WS;  // lanes to a row, rows of a wavefront
    constexpr int kRowsAtOnce = 64 / kPerRow < kShareRows ? 64 / kPerRow : kShareRows, kTimes = kShareRows / kRowsAtOnce;
    const int col = (lane % kPerRow) * V, j = (int)j0 + wj + col, n = lane / kPerRow < kRowsAtOnce ? min(V, p.cols - j) : 0;
    float bias[V];
#pragma unroll
    for (int e = 0; e < V; ++e) bias[e] = p.bias && e < n ? p.bias[j + e] : 0.0f;
#pragma unroll 1
    for (int a = 0; a < NI; ++a) {
        const int row0 = share * kShareRows + lane / kPerRow % kRowsAtOnce;
        const long long first = i0 + wi + 32 * a + row0;
        Vec<T> residual[kTimes];
        if (p.residual && p.splits == 1) {
#pragma unroll
            for (int r = 0; r < kTimes; ++r)
                if (first + r * kRowsAtOnce < p.rows) residual[r] = get_columns<T, V>(p.residual, p.residual_ld, first + r * kRowsAtOnce, j, n);
        }
#pragma unroll
        for (int k = 0; k < NI; ++k)  // (registers have no index: one of NI pieces of code)
            if (k == a) {
#pragma unroll
                for (int b = 0; b < NJ; ++b)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<float4*>(mine + (lane & 31) * kOutRow + (32 * b + 8 * g + 4 * (lane >> 5)) * 4) =
                            make_float4(acc[k][b][4 * g], acc[k][b][4 * g + 1], acc[k][b][4 * g + 2], acc[k][b][4 * g + 3]);
            }
        if constexpr (WS > 1)
            __syncthreads();
        else
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int r = 0; r < kTimes; ++r) {
            const long long i = first + r * kRowsAtOnce;
            const char* from = first_share + (row0 + r * kRowsAtOnce) * kOutRow + col * 4;
            float z[V];
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                float4 q = *reinterpret_cast<const float4*>(from + e * 4);
#pragma unroll
                for (int w = 1; w < WS; ++w) {
                    const float4 o = *reinterpret_cast<const float4*>(from + w * (WI * WJ * kOutWave) + e * 4);
                    q.x += o.x, q.y += o.y, q.z += o.z, q.w += o.w;
                }
                z[e] = q.x, z[e + 1] = q.y, z[e + 2] = q.z, z[e + 3] = q.w;
            }
            if (i < p.rows && n > 0) {
                if (p.splits > 1) {
#pragma unroll
                    for (int e = 0; e < V; e += 4) put_columns<float, 4>(p.partial + (size_t)split * p.rows * p.cols, p.cols, i, j + e, n - e, z + e);
                } else {
                    finish<T, V>(p, i, j, n, bias, residual[r], z);
                }
            }
        }
        if constexpr (WS > 1) {
            if (NI > 1) __syncthreads();
        } else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
#endif
}
template <typename T, int BI, int BJ, int WI, int WJ, int WS, int STAGES, Access ACCESS, int HOLD, bool LONG, bool ACROSS_I, bool ACROSS_J>
__global__ __launch_bounds__(64 * WI * WJ * WS) void product_kernel(const ProductParams p) {
    __shared__ __align__(1024) char lds[product_lds<BI, BJ, WI, WJ, WS, STAGES>()];
    product<T, BI, BJ, WI, WJ, WS, STAGES, ACCESS, HOLD, LONG, ACROSS_I, ACROSS_J>(p, blockIdx.x, lds);
}

// The sums of a split product's parts, always in the same order, and what follows them: four columns of a row a thread, all parts requested
// before the first is added (one after the other, 3 x 408 in 8 parts took 8.8 us).
constexpr int kMaxSplits = 8, kJoinVector = 4;
template <typename T>
__global__ __launch_bounds__(256) void product_join_kernel(const ProductParams p) {
    constexpr int C = kJoinVector;
    const int per_row = (p.cols + C - 1) / C;
    const long long v = (long long)blockIdx.x * 256 + threadIdx.x, i = v / per_row;
    if (i >= p.rows) return;
    const int j = (int)(v - i * per_row) * C, n = min(C, p.cols - j);
    Columns<float, C> part[kMaxSplits];
#pragma unroll
    for (int k = 0; k < kMaxSplits; ++k)
        if (k < p.splits) part[k] = get_columns<float, C>(p.partial, p.cols, (long long)k * p.rows + i, j, n);
    float z[C], bias[C];
#pragma unroll
    for (int e = 0; e < C; ++e) {
        z[e] = 0.0f;
        bias[e] = p.bias && e < n ? p.bias[j + e] : 0.0f;
    }
    Columns<T, C> residual = {};
    if (p.residual) residual = get_columns<T, C>(p.residual, p.residual_ld, i, j, n);
#pragma unroll
    for (int k = 0; k < kMaxSplits; ++k)
        if (k < p.splits) {
#pragma unroll
            for (int e = 0; e < C; ++e) z[e] += part[k][e];
        }
    finish<T, C>(p, i, j, n, bias, residual, z);
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

template <typename T, int SHARES>
__global__ __launch_bounds__(64 * kFewWaves) __attribute__((amdgpu_waves_per_eu(2, 4))) void few_rows_kernel(const ProductParams p) {
    constexpr int V = Elem<T>::kVec, kChunk = 4 * V;
    __shared__ Acc4 lds[kFewWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, share = wave % SHARES, start = (lane >> 4) * V;
    const int j0 = (blockIdx.x * (kFewWaves / SHARES) + wave / SHARES) * kFewOutputs;
    // rows past the last one are read as the last one; nothing of them is kept
    const T* w = (const T*)p.j.p + (long long)min(j0 + (lane & 15), p.cols - 1) * p.j.ld;
    const T* x = (const T*)p.i.p + (long long)min(lane & 15, p.rows - 1) * p.i.ld;
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
    if (share != 0) return;
    const int i = lane & 15, j = j0 + 4 * (lane >> 4), n = min(4, p.cols - j);
    if (i >= p.rows || n <= 0) return;
    float z[4], bias[4];
#pragma unroll
    for (int k = 1; k < SHARES; ++k) acc += lds[wave + k][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        z[e] = acc[e];
        bias[e] = p.bias && e < n ? p.bias[j + e] : 0.0f;
    }
    Columns<T, 4> residual = {};
    if (p.residual) residual = get_columns<T, 4>(p.residual, p.residual_ld, i, j, n);
    finish<T, 4>(p, i, j, n, bias, residual, z);
}

// ---- dz = dy act'(z) in the operands' type (nothing to write without an activation), and its column sums in fp32, unrounded.
// Bound by memory: a thread has one vector of 16 bytes of columns and goes down its share of the rows, four rows requested at
// a time; the workgroups' sums are joined afterwards, always in the same order.  8192 x 4096 bf16 with GELU: 42 us for 201 MB (4.8 TB/s)
// and 5 us for the join.  dz is rounded to the operands' type because that is what the matrix instructions of dx and dw take: each term
// of theirs then has two roundings of its own in place of one, which in 16 bits are sqrt 2 of the error that dw would have otherwise.
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

template <typename T, int ACT>
__global__ __launch_bounds__(kDzThreads) void dz_kernel(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ dz,
                                                        float* __restrict__ sums, int rows, int n, int lanes, int each,
                                                        long long dy_ld, long long z_ld) {
    constexpr int V = Elem<T>::kVec, kAtOnce = 4;
    __shared__ float lds[kDzThreads * V];
    const int deep = kDzThreads / lanes, lane = threadIdx.x % lanes, depth = threadIdx.x / lanes;
    const int j = (blockIdx.x * lanes + lane) * V, left = n - j;
    const long long first = (long long)blockIdx.y * deep * each;
    const long long last = min((long long)rows, first + (long long)deep * each);
    float s[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = 0.0f;
    if (depth < deep && left > 0) {
        auto get = [&](const T* p) {
            if (left >= V) return load_vec(p);
            Vec<T> v;
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = e < left ? p[e] : (T)0.0f;
            return v;
        };
        for (long long r = first + depth; r < last; r += kAtOnce * deep) {
            Vec<T> g[kAtOnce], x[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const long long at = min(r + u * deep, last - 1);  // (rows past the end are read once more and not used)
                g[u] = get(dy + at * dy_ld + j);
                if constexpr (ACT != TCBNN_ACT_NONE) x[u] = get(z + at * z_ld + j);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                if (r + u * deep >= last) break;
                float d[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    d[e] = (float)g[u][e];
                    if constexpr (ACT != TCBNN_ACT_NONE) d[e] *= slope<T, ACT>((float)x[u][e]);
                    s[e] += d[e];
                }
                if constexpr (ACT != TCBNN_ACT_NONE) {
                    T* to = dz + (r + u * deep) * n + j;
                    if (left >= V) {
                        Vec<T> v;
#pragma unroll
                        for (int e = 0; e < V; ++e) v[e] = (T)d[e];
                        store_vec(to, v);
                    } else {
#pragma unroll
                        for (int e = 0; e < V; ++e)
                            if (e < left) to[e] = (T)d[e];
                    }
                }
            }
        }
    }
    if (sums == nullptr) return;
#pragma unroll
    for (int e = 0; e < V; ++e) lds[e * kDzThreads + threadIdx.x] = s[e];
    __syncthreads();
    for (int c = threadIdx.x; c < lanes * V; c += kDzThreads) {
        const int l = c / V, e = c % V, col = (blockIdx.x * lanes + l) * V + e;
        float t = 0.0f;
        for (int d = 0; d < deep; ++d) t += lds[e * kDzThreads + d * lanes + l];
        if (col < n) sums[(size_t)blockIdx.y * n + col] = t;
    }
}

// the sums of all parts: 16 columns a workgroup (and 16 more where there are more than a launch has threads for), 16 threads to a column
constexpr int kJoinColumns = 16;
__global__ __launch_bounds__(kDzThreads) void column_join_kernel(const float* __restrict__ sums, float* __restrict__ db, int parts, int n) {
    constexpr int kStep = kDzThreads / kJoinColumns;
    __shared__ float lds[kStep][kJoinColumns];
    const int c = threadIdx.x % kJoinColumns, part = threadIdx.x / kJoinColumns;
    for (int j = blockIdx.x * kJoinColumns + c; j - c < n; j += gridDim.x * kJoinColumns) {
        float s = 0.0f;
        if (j < n)
            for (int k = part; k < parts; k += 8 * kStep) {
                float v[8];  // (requests of their own, one wait)
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = k + u * kStep < parts ? sums[(size_t)(k + u * kStep) * n + j] : 0.0f;
#pragma unroll
                for (int u = 0; u < 8; ++u) s += v[u];
            }
        lds[part][c] = s;
        __syncthreads();
        if (part == 0 && j < n) {
            s = 0.0f;
#pragma unroll
            for (int k = 0; k < kStep; ++k) s += lds[k][c];
            db[j] = s;
        }
        __syncthreads();
    }
}

// ---- both products of small gradients in one launch.  A launch more takes as long as these products do (102 x 24 -> 21 f16 with its dz:
// 13.0 us in three launches, 9.9 in two; 128 x 1024 -> 512 18.8 and 16.3).  The first `blocks` workgroups have the product with the longer sum:
// started last, they would run on alone (1024 x 1024 -> 10 bf16 15.1 us, 12.6 so).
template <typename T, Access ACCESS, int STAGES, int HOLD>
__global__ __launch_bounds__(256) void small_gradients_kernel(const ProductParams dx, const ProductParams dw, int blocks, bool dw_first) {
    __shared__ __align__(1024) char lds[product_lds<32, 32, 1, 1, 4, STAGES>()];
    const int second = (int)blockIdx.x >= blocks, block = (int)blockIdx.x - (second ? blocks : 0);
    if (second == dw_first)
        product<T, 32, 32, 1, 1, 4, STAGES, ACCESS, HOLD, ACCESS == ANYWHERE, false, true>(dx, block, lds);
    else
        product<T, 32, 32, 1, 1, 4, STAGES, ACCESS, HOLD, ACCESS == ANYWHERE, true, true>(dw, block, lds);
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
inline Plan plan_product(int rows, int cols, int sum, int size, bool vectors, size_t workspace_bytes, Cut largest = CUT_256) {
    const int steps = (int)(((long long)sum * size + kStepBytes - 1) / kStepBytes);
    const float read = ((float)rows + (float)cols) * (float)sum * (float)size / kReadRate;
    Plan best = {CUT_32, 1, 0.0f};
    for (int c = largest; c < CUTS; ++c) {
        CutCost cost = vectors ? (size == 4 ? kCuts32[c] : kCuts16[c]) : kCutsAnywhere[c];
        if (cost.size == 0) continue;
        if (!vectors && size == 4) cost.step = std::max(cost.step, kCuts32[c].step), cost.more = std::max(cost.more, kCuts32[c].more);
        const float tiles = (float)((rows + cost.size - 1) / cost.size) * (float)((cols + cost.size - 1) / cost.size);
        for (int k = 1; k <= kMaxSplits && (k == 1 || steps >= 4 * k); k *= 2) {
            const size_t partial = k > 1 ? (size_t)k * rows * cols * sizeof(float) : 0;
            if (partial > workspace_bytes) break;
            const float rounds = std::ceil(tiles * (float)k / (float)kComputeUnits), each = std::max(cost.step, rounds * cost.more);
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

template <typename T, bool ACROSS_I, bool ACROSS_J>
Access access_of(const ProductParams& p) {
    auto of = [](const Operand& o, int rows, int sum, bool across) {
        const int row = across ? rows : sum;
        if (row < Elem<T>::kVec || o.ld * 256 * (long long)sizeof(T) > 0x7fffffffLL) return ELEMENTS;
        return (uintptr_t)o.p % 16 == 0 && o.ld * sizeof(T) % 16 == 0 && row % Elem<T>::kVec == 0 ? WHOLE_PIECES : ANYWHERE;
    };
    return std::max(of(p.i, p.rows, p.sum, ACROSS_I), of(p.j, p.cols, p.sum, ACROSS_J));
}
inline void cut_product(ProductParams& p, int size, int steps_size, int splits, float* workspace) {
    p.tiles_i = (p.rows + size - 1) / size;
    p.tiles_j = (p.cols + size - 1) / size;
    const int steps = (p.sum + steps_size - 1) / steps_size;
    p.split_sum = std::max(1, (steps + splits - 1) / splits) * steps_size;
    p.splits = std::max(1, (p.sum + p.split_sum - 1) / p.split_sum);
    p.partial = workspace;
}

// dx and dw in one launch, where in tiles of 32 x 32, four a compute unit at most, they are estimated to take less time together than
// apart in tiles and splits of their own; false: nothing is launched
template <typename T>
bool launch_small_gradients(ProductParams dx, ProductParams dw, size_t workspace_bytes, hipStream_t stream) {
    const Access access_dx = access_of<T, false, true>(dx), access_dw = access_of<T, true, true>(dw), access = std::max(access_dx, access_dw);
    float together = -kCuts16[CUT_32].start, apart = 0.0f;
    for (const ProductParams* p : {&dx, &dw}) {
        if ((long long)((p->rows + 31) / 32) * ((p->cols + 31) / 32) > 4 * kComputeUnits) return false;
        together += plan_product(p->rows, p->cols, p->sum, (int)sizeof(T), access == WHOLE_PIECES, 0, CUT_32).time;
        apart += plan_product(p->rows, p->cols, p->sum, (int)sizeof(T), (p == &dx ? access_dx : access_dw) == WHOLE_PIECES, workspace_bytes).time;
    }
    if (access == ELEMENTS || together >= apart) return false;
    cut_product(dx, 32, kStepBytes / (int)sizeof(T), 1, nullptr);
    cut_product(dw, 32, kStepBytes / (int)sizeof(T), 1, nullptr);
    const int blocks_dx = dx.tiles_i * dx.tiles_j, blocks_dw = dw.tiles_i * dw.tiles_j;
    const bool dw_first = dw.sum > dx.sum;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks_dx + blocks_dw)), dim3(256), 0, stream, dx, dw, dw_first ? blocks_dw : blocks_dx, dw_first);
    };
    if (access == WHOLE_PIECES)
        go(small_gradients_kernel<T, WHOLE_PIECES, 8, 1>);
    else
        go(small_gradients_kernel<T, ANYWHERE, 2, 4>);
    return true;
}

// Tiles of 64 whose rows lie anywhere: the loop for long sums takes registers that a third workgroup of a compute unit would have
// (bf16, with that loop / without: 1000 x 1001 x 999, one tile a compute unit, 9.8 us / 13.5; 2000 x 777 x 1111, three, 24.4 / 19.6).
template <typename T>
bool long_sums(const ProductParams& p, const Plan& plan) {
    const long long tiles = (long long)((p.rows + 63) / 64) * ((p.cols + 63) / 64) * plan.splits;
    return tiles <= 2 * kComputeUnits && (long long)p.sum * sizeof(T) > (long long)kLongSteps * kStepBytes * plan.splits;
}

// (tiles of single elements are for memory where addresses do not fit; they are slower in any size)
template <typename T>
bool few_rows(const ProductParams& p, Access access, const Plan& plan) {
    return p.rows <= kFewRows && (access == ELEMENTS || few_time(p.rows, p.cols, p.sum, (int)sizeof(T), access == WHOLE_PIECES) < plan.time);
}

// the kernel that launch_product takes for a forward product, as a profiler lists it
template <typename T>
void product_name(const ProductParams& p, size_t workspace_bytes, char* buf, size_t len) {
    const char* type = std::is_same_v<T, float> ? "float" : (std::is_same_v<T, _Float16> ? "_Float16" : "__bf16");
    const Access access = access_of<T, false, false>(p);
    const Plan plan = plan_product(p.rows, p.cols, p.sum, (int)sizeof(T), access == WHOLE_PIECES, workspace_bytes);
    if (few_rows<T>(p, access, plan)) {
        snprintf(buf, len, "few_rows_kernel<%s, %d>", type, few_shares(p.cols, p.sum, (int)sizeof(T)));
        return;
    }
    static const char* const shape[3][CUTS] = {
        {"256, 256, 2, 4, 1, 2", "128, 128, 2, 2, 1, 2", "128, 128, 2, 2, 2, 4", "64, 64, 2, 2, 2, 4", "32, 32, 1, 1, 4, 8"},
        {"", "128, 128, 2, 2, 1, 2", "", "64, 64, 2, 2, 2, 2", "32, 32, 1, 1, 4, 2"},
        {"32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2", "32, 32, 1, 1, 4, 2"}};
    const int hold = access == ANYWHERE && plan.cut != CUT_128 ? 4 : 1;
    const bool keep = hold == 4 && (plan.cut != CUT_64 || long_sums<T>(p, plan));
    snprintf(buf, len, "product_kernel<%s, %s, (Access)%d, %d, %s, false, false>%s", type, shape[access][plan.cut], (int)access, hold, keep ? "true" : "false",
             plan.splits > 1 ? " + product_join_kernel" : "");
}

template <typename T, bool ACROSS_I, bool ACROSS_J>
int launch_product(ProductParams p, float* workspace, size_t workspace_bytes, hipStream_t stream) {
    const Access access = access_of<T, ACROSS_I, ACROSS_J>(p);
    const Plan plan = plan_product(p.rows, p.cols, p.sum, (int)sizeof(T), access == WHOLE_PIECES, workspace_bytes);
    if constexpr (!ACROSS_I && !ACROSS_J) {
        if (few_rows<T>(p, access, plan)) {
            const int shares = few_shares(p.cols, p.sum, (int)sizeof(T)), outputs = kFewOutputs * kFewWaves / shares;
            const dim3 grid((unsigned)(p.cols / outputs + (p.cols % outputs != 0)));
            if (shares == 8)
                hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_kernel<T, 8>), grid, dim3(64 * kFewWaves), 0, stream, p);
            else
                hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_kernel<T, 2>), grid, dim3(64 * kFewWaves), 0, stream, p);
            TCBNN_LAUNCH_CHECK("few_rows_kernel");
            return TCBNN_OK;
        }
    }
    auto go = [&](auto size, auto wi, auto wj, auto ws, auto stages, auto how, auto hold, auto keep) {
        constexpr int B = size.value, WI = wi.value, WJ = wj.value, WS = ws.value, S = stages.value, H = hold.value;
        constexpr bool L = keep.value;
        constexpr int kThreads = 64 * WI * WJ * WS;
        // rows beyond a launch's threads (2^29 rows, where they are too short for larger tiles than 32) have one of their own
        cut_product(p, B, kStepBytes / (int)sizeof(T), plan.splits, workspace);
        const long long at_once = kMaxThreads / kThreads / ((long long)p.tiles_j * p.splits) * B;
        for (long long first = 0; first < p.rows; first += at_once) {
            ProductParams q = p;
            q.rows = (int)std::min(at_once, p.rows - first);
            q.i.p = (const T*)p.i.p + (ACROSS_I ? first : first * p.i.ld);
            q.residual = p.residual ? (const T*)p.residual + first * p.residual_ld : nullptr;
            q.out = (T*)p.out + first * p.out_ld;
            q.preact = p.preact ? (T*)p.preact + first * p.preact_ld : nullptr;
            cut_product(q, B, kStepBytes / (int)sizeof(T), plan.splits, workspace);
            hipLaunchKernelGGL(HIP_KERNEL_NAME(product_kernel<T, B, B, WI, WJ, WS, S, how.value, H, L, ACROSS_I, ACROSS_J>),
                               dim3((unsigned)((long long)q.tiles_i * q.tiles_j * q.splits)), dim3(kThreads), 0, stream, q);
            if (q.splits > 1) {
                const long long vectors_out = (long long)q.rows * ((q.cols + kJoinVector - 1) / kJoinVector);
                hipLaunchKernelGGL(product_join_kernel<T>, dim3((unsigned)((vectors_out + 255) / 256)), dim3(256), 0, stream, q);
            }
        }
    };
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
        switch (plan.cut) {
            case CUT_256: go(n256, two, four, one, two, pieces, one, no); break;
            case CUT_128: go(n128, two, two, one, two, pieces, one, no); break;
            case CUT_128_DEEP: go(n128, two, two, two, four, pieces, one, no); break;
            case CUT_64: go(n64, two, two, two, four, pieces, one, no); break;
            default: go(n32, one, one, four, eight, pieces, one, no); break;
        }
    } else if (access == ANYWHERE) {
        switch (plan.cut) {
            case CUT_128: go(n128, two, two, one, two, anywhere, one, no); break;
            case CUT_64:
                if (long_sums<T>(p, plan))
                    go(n64, two, two, two, two, anywhere, four, yes);
                else
                    go(n64, two, two, two, two, anywhere, four, no);
                break;
            default: go(n32, one, one, four, two, anywhere, four, yes); break;
        }
    } else {
        go(n32, one, one, four, two, elements, one, no);
    }
    TCBNN_LAUNCH_CHECK("product_kernel");
    return TCBNN_OK;
}

}  // namespace
}  // namespace tcbnn

using namespace tcbnn;
using namespace tcbnn::head;

static int check_linear(int rows, int in_features, int out_features, int dtype, int activation) {
    TCBNN_REQUIRE(dtype_known(dtype), "linear: unknown dtype");
    TCBNN_REQUIRE(activation >= TCBNN_ACT_NONE && activation <= TCBNN_ACT_SILU, "linear: unknown activation");
    TCBNN_REQUIRE(rows >= 0 && in_features > 0 && out_features > 0, "linear: bad shape");
    TCBNN_REQUIRE(rows <= kMaxRows, "linear: at most %d rows", kMaxRows);
    TCBNN_REQUIRE(in_features <= kMaxIn, "linear: at most %d inputs", kMaxIn);
    TCBNN_REQUIRE(out_features <= kMaxOut, "linear: at most %d outputs", kMaxOut);
    return TCBNN_OK;
}

// the partial sums of a split product
static size_t split_bytes(int rows, int cols, int sum, int dtype, bool forward) {
    const int size = (int)dtype_bytes(dtype);
    int splits = 1;
    for (bool vectors : {false, true}) {  // (where the operands will lie is not known here)
        const Plan plan = plan_product(rows, cols, sum, size, vectors, ~(size_t)0);
        if (!forward || rows > kFewRows || few_time(rows, cols, sum, size, vectors) >= plan.time) splits = std::max(splits, plan.splits);
    }
    return splits > 1 ? (size_t)splits * rows * cols * sizeof(float) : 0;
}

extern "C" size_t tcbnn_linear_workspace_bytes(int rows, int in_features, int out_features, int dtype) {
    if (rows <= 0 || rows > kMaxRows || in_features <= 0 || out_features <= 0 || !dtype_known(dtype)) return 0;
    return split_bytes(rows, out_features, in_features, dtype, true);
}

static ProductParams forward_product(const tcbnn_linear_desc* d) {
    ProductParams p = {};
    p.i = {d->input, row_stride(d->input_ld, d->in_features)};
    p.j = {d->weight, row_stride(d->weight_ld, d->in_features)};
    p.rows = d->rows;
    p.cols = d->out_features;
    p.sum = d->in_features;
    p.activation = d->activation;
    p.bias = d->bias;
    p.residual = d->residual;
    p.out = d->output;
    p.preact = d->preact;
    p.residual_ld = row_stride(d->residual_ld, d->out_features);
    p.out_ld = row_stride(d->output_ld, d->out_features);
    p.preact_ld = row_stride(d->preact_ld, d->out_features);
    return p;
}

extern "C" int tcbnn_linear_kernel_name(const tcbnn_linear_desc* d, char* buf, size_t len) {
    TCBNN_NOTNULL(d);
    TCBNN_NOTNULL(buf);
    if (int rc = check_linear(d->rows, d->in_features, d->out_features, d->dtype, d->activation)) return rc;
    by_dtype(d->dtype, [&](auto t) { product_name<decltype(t)>(forward_product(d), d->workspace ? d->workspace_bytes : 0, buf, len); });
    return TCBNN_OK;
}

extern "C" int tcbnn_linear_forward(const tcbnn_linear_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_linear(d->rows, d->in_features, d->out_features, d->dtype, d->activation)) return rc;
    const long long x_ld = row_stride(d->input_ld, d->in_features), w_ld = row_stride(d->weight_ld, d->in_features),
                    r_ld = row_stride(d->residual_ld, d->out_features), y_ld = row_stride(d->output_ld, d->out_features),
                    z_ld = row_stride(d->preact_ld, d->out_features);
    TCBNN_REQUIRE(x_ld > 0 && w_ld > 0 && r_ld > 0 && y_ld > 0 && z_ld > 0, "linear: rows overlap");
    if (d->rows == 0) return TCBNN_OK;
    TCBNN_NOTNULL(d->input);
    TCBNN_NOTNULL(d->weight);
    TCBNN_NOTNULL(d->output);
    TCBNN_REQUIRE(d->output != d->residual || d->rows == 1 || y_ld == r_ld, "linear: an output over its residual has the residual's stride");
    const ProductParams p = forward_product(d);
    return by_dtype(d->dtype, [&](auto t) { return launch_product<decltype(t), false, false>(p, (float*)d->workspace, d->workspace ? d->workspace_bytes : 0, (hipStream_t)stream); });
}

// What the gradients need of a workspace: dz in dtype, then the parts of the column sums (whole 256 bytes each).
static size_t whole_lines(size_t bytes) { return (bytes + 255) / 256 * 256; }
static size_t dz_bytes(int rows, int out_features, int dtype) { return whole_lines((size_t)rows * out_features * dtype_bytes(dtype)); }
static int out_vectors(int out_features, int dtype) { return (out_features + (int)(16 / dtype_bytes(dtype)) - 1) / (int)(16 / dtype_bytes(dtype)); }

static size_t sum_bytes(int rows, int out_features, int dtype) {
    return rows == 0 ? 0 : whole_lines(sizeof(float) * dz_parts(rows, out_vectors(out_features, dtype), true) * (size_t)out_features);
}
extern "C" size_t tcbnn_linear_grad_workspace_bytes(int rows, int in_features, int out_features, int dtype) {
    if (rows <= 0 || rows > kMaxRows || in_features <= 0 || out_features <= 0 || !dtype_known(dtype)) return 0;
    return dz_bytes(rows, out_features, dtype) + sum_bytes(rows, out_features, dtype) +
           std::max(split_bytes(rows, in_features, out_features, dtype, false), split_bytes(out_features, in_features, rows, dtype, false));
}

extern "C" int tcbnn_linear_backward(const tcbnn_linear_grad_desc* d, void* stream) {
    TCBNN_NOTNULL(d);
    if (int rc = check_linear(d->rows, d->in_features, d->out_features, d->dtype, d->activation)) return rc;
    const long long x_ld = row_stride(d->input_ld, d->in_features), w_ld = row_stride(d->weight_ld, d->in_features),
                    z_ld = row_stride(d->preact_ld, d->out_features), dy_ld = row_stride(d->grad_output_ld, d->out_features),
                    dx_ld = row_stride(d->grad_input_ld, d->in_features), dw_ld = row_stride(d->grad_weight_ld, d->in_features);
    TCBNN_REQUIRE(x_ld > 0 && w_ld > 0 && z_ld > 0 && dy_ld > 0 && dx_ld > 0 && dw_ld > 0, "linear: rows overlap");
    const bool active = d->activation != TCBNN_ACT_NONE;
    if (d->rows > 0) {
        TCBNN_NOTNULL(d->grad_output);
        if (active) TCBNN_NOTNULL(d->preact);
        if (d->grad_weight) TCBNN_NOTNULL(d->input);
        if (d->grad_input) TCBNN_NOTNULL(d->weight);
        TCBNN_NOTNULL(d->workspace);
        TCBNN_REQUIRE((uintptr_t)d->workspace % 16 == 0, "linear: the workspace is not aligned to 16 bytes");
        TCBNN_REQUIRE(d->workspace_bytes >= tcbnn_linear_grad_workspace_bytes(d->rows, d->in_features, d->out_features, d->dtype),
                      "linear: workspace too small");
    }
    return by_dtype(d->dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (active || d->grad_bias) {
            const int vectors = out_vectors(d->out_features, d->dtype), lanes = dz_lanes(vectors), parts = dz_parts(d->rows, vectors, active);
            float* sums = d->grad_bias ? (float*)((char*)d->workspace + dz_bytes(d->rows, d->out_features, d->dtype)) : nullptr;
            if (d->grad_bias && parts == 1 && d->rows > 0) sums = d->grad_bias;
            if (d->rows > 0)
                by_activation(d->activation, [&](auto act) {
                    hipLaunchKernelGGL(HIP_KERNEL_NAME(dz_kernel<T, act.value>), dim3((unsigned)((vectors + lanes - 1) / lanes), (unsigned)parts),
                                       dim3(kDzThreads), 0, (hipStream_t)stream, (const T*)d->grad_output, (const T*)d->preact,
                                       (T*)d->workspace, sums, d->rows, d->out_features, lanes, dz_rows(d->rows, vectors, active), dy_ld, z_ld);
                });
            if (d->grad_bias && sums != d->grad_bias)
                hipLaunchKernelGGL(column_join_kernel, dim3((unsigned)std::min((d->out_features + kJoinColumns - 1LL) / kJoinColumns, kMaxThreads / kDzThreads)),
                                   dim3(kDzThreads), 0, (hipStream_t)stream, sums, d->grad_bias, d->rows > 0 ? parts : 0, d->out_features);
        }
        TCBNN_LAUNCH_CHECK("dz_kernel");
        const size_t before = dz_bytes(d->rows, d->out_features, d->dtype) + sum_bytes(d->rows, d->out_features, d->dtype);
        float* partials = d->rows > 0 ? (float*)((char*)d->workspace + before) : nullptr;
        const size_t partial_bytes = d->rows > 0 ? d->workspace_bytes - before : 0;
        const Operand dz = active ? Operand{d->workspace, d->out_features} : Operand{d->grad_output, dy_ld};
        ProductParams dx = {}, dw = {};
        dx.i = dw.i = dz;
        dx.j = {d->weight, w_ld};
        dx.rows = d->rows;
        dx.cols = d->in_features;
        dx.sum = d->out_features;
        dx.out = d->grad_input;
        dx.out_ld = dx_ld;
        dw.j = {d->input, x_ld};
        dw.rows = d->out_features;
        dw.cols = d->in_features;
        dw.sum = d->rows;
        dw.out = d->grad_weight;
        dw.out_ld = dw_ld;
        if (d->grad_input && d->grad_weight && d->rows > 0 && launch_small_gradients<T>(dx, dw, partial_bytes, (hipStream_t)stream)) {
            TCBNN_LAUNCH_CHECK("small_gradients_kernel");
            return TCBNN_OK;
        }
        if (d->grad_input && d->rows > 0)
            if (int rc = launch_product<T, false, true>(dx, partials, partial_bytes, (hipStream_t)stream)) return rc;
        if (d->grad_weight)
            if (int rc = launch_product<T, true, true>(dw, partials, partial_bytes, (hipStream_t)stream)) return rc;
        return TCBNN_OK;
    });
}
