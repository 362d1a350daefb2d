// Losses of the move-scoring head and their gradients.
//
// A board's features X [32][64] and the logit kernel W [32][73] give the logits l[f][s] = sum_c W[c][f] X[c][s] of its
// move vocabulary (73 filters x 64 from-squares = 4 672).  With target t and weight w of the board,
//
//     loss  = log sum exp l - l[t]                         d = w (softmax(l) - onehot(t))
//     dX[c][s] = sum_f W[c][f] d[f][s]                     dW[c][f] = sum over boards and s of X[c][s] d[f][s]
//
// where the softmax runs over the whole vocabulary (k_policy_loss) or over the board's own list of moves
// (k_policy_move_loss).  A board without a target has loss 0 and no part in the gradients.  Both keep one board in one
// wave, so that its result does not depend on its place in the batch, and sum dW over a wave's boards, then over a
// workgroup's waves, then over the workgroups (k_sum_parts), each in fixed order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/batchfirst.h"
#include "bf_train.h"

namespace bf {
namespace {

constexpr int kC = 32, kS = 64, kF = 73, kVocab = kF * kS, kXW = kC * kF;

// ---- arithmetic, and what both losses share --------------------------------------------------------------------------
//
// 16x16x32 MFMAs with float32 sums.  Lane l = (col = l & 15, q = l >> 4) of an operand holds eight k (8 q ... 8 q + 7) of row or
// column col, of a result the rows 4 q ... 4 q + 3 of column col.
//
// float32 operands travel as two float16 terms (22 bits), scaled by a power of two so that the larger term stays normal
// down to 2^-27 of the largest: over the vocabulary the kernel's by its largest element and the features' by the board's,
// over moves by the filter's and by the square's; of the four products of terms the least is left out (2^-22).  (float32
// MFMAs alone would take 384 us for the 65 536 boards below that take 276.)  Where the largest may take no part in a sum and
// the bits below it count, the sum is float32 throughout: kWide below.  bfloat16 and float16 operands are exact as they are.
// The logits' gradients d (before the weight) travel as two terms: float16 ones, scaled like the features, or for bfloat16
// features bfloat16 ones (16 bits, 2^-17 of d beside the 2^-8 of their result's rounding).  Their largest is the target's,
// which is the negative sum of all the others.

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((__vector_size__(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Arith {                                   // float32 and float16 features: float16 terms
    static constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;
    static constexpr bool kScaled = true;         // the gradients' terms need scaling
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    }
    // (a, b) = terms hi + lo, each packed with a in the low half.  Rounded to nearest: towards zero (which packs in one
    // instruction as well) both terms and the product that is left out err to one side, 8e-7 of a gradient in place of 1e-7.
    static __device__ __forceinline__ void split(float a, float b, unsigned& hi, unsigned& lo) {
        hi = __builtin_bit_cast(unsigned, half2v{(_Float16)a, (_Float16)b});
        asm("" : "+v"(hi));                      // one rounding for both uses: a product a may be contracted into either
        const half2v h = __builtin_bit_cast(half2v, hi);
        float ra = a - (float)h[0], rb = b - (float)h[1];
        asm("" : "+v"(ra));                      // packed together: rounded in the subtraction they cost 1 % of the call
        asm("" : "+v"(rb));
        lo = __builtin_bit_cast(unsigned, half2v{(_Float16)ra, (_Float16)rb});
    }
};
template <>
struct Arith<__bf16> {
    static constexpr int kTerms = 1;
    static constexpr bool kScaled = false;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void split(float a, float b, unsigned& hi, unsigned& lo) {
        hi = __builtin_bit_cast(unsigned, bf2{(__bf16)a, (__bf16)b});
        asm("" : "+v"(hi));
        lo = __builtin_bit_cast(unsigned, bf2{(__bf16)(a - __uint_as_float(hi << 16)), (__bf16)(b - __uint_as_float(hi & 0xffff0000u))});
    }
};

template <typename T>
struct Raw;                                      // four neighbours as they lie
template <> struct Raw<float> { typedef f32x4 type; };
template <> struct Raw<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(4))); };
template <> struct Raw<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(4))); };

__device__ __forceinline__ void lds_fence() {    // orders a wave's own LDS accesses for the compiler; the hardware keeps order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The larger, or NaN if either is: one instruction of three operands, without the quieting that fmaxf's takes each.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Over the 64 lanes, in fixed order; the result is uniform.
template <bool MAX>
__device__ __forceinline__ float lanes_reduce(float v) {
    auto step = [](float a, float b) { return MAX ? larger(a, b) : a + b; };
#define BF_DPP(ctrl) v = step(v, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), ctrl, 0xf, 0xf, true)))
    BF_DPP(0xb1);    // quad_perm [1, 0, 3, 2]
    BF_DPP(0x4e);    // quad_perm [2, 3, 0, 1]
    BF_DPP(0x141);   // row_half_mirror
    BF_DPP(0x140);   // row_mirror
#undef BF_DPP
    auto at = [&](int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane)); };
    return step(step(at(0), at(16)), step(at(32), at(48)));
}

// The largest over the four lanes of a column, NaN if one is, the same in all four.
__device__ __forceinline__ float rows_max(float v) {
    auto step = [](auto pair) { return larger(__uint_as_float(pair[0]), __uint_as_float(pair[1])); };
    v = step(__builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return step(__builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
}

// 2^(13 - e) for a largest magnitude in [2^e, 2^(e+1)), and its reciprocal; magnitudes below 2^least count as that, infinity
// and NaN as 2^128.
__device__ __forceinline__ void scale_of(float largest, int least, float& scale, float& back) {
    const int e = max((int)(__float_as_uint(largest) >> 23 & 255u) - 127, least);
    scale = __uint_as_float((unsigned)(127 + 13 - e) << 23);
    back = __uint_as_float((unsigned)(127 - 13 + e) << 23);
}

// From the lanes' largest magnitudes to the largest of all (infinity or NaN where one is not finite); whether one that is
// not zero lies more than 2^16 below it.
__device__ __forceinline__ bool range_of(float& largest) {
    const float mine = largest;
    largest = lanes_reduce<true>(mine);
    return __ballot(mine > 0.0f && mine < largest * 0x1p-16f) != 0;
}

constexpr int kTiles = 5;                        // of 16 filters
constexpr int kRow = 40;                         // 16-bit elements of a row of 32 in LDS: 16 rows start in 16 different bank groups
constexpr int kTerm = kS * kRow;                 // elements of 64 rows
constexpr int kPart = kC * 16 * kTiles;          // elements of a part of the kernel's gradient: [32][80], 73 of 80 in use
constexpr int kPartBytes = kPart * 4;            // a wave's in LDS, when its boards are done

// A board's features: a lane holds channels 8 q ... 8 q + 7 of squares 4 col ... 4 col + 3 and turns them into operands
// of columns square (4 col + j), k channel.
template <typename T>
struct Features {
    static constexpr int kTerms = Arith<T>::kTerms;
    typename Raw<T>::type raw[8];
    u32x4 column[4][kTerms];
    float back;
    bool uneven;

    __device__ __forceinline__ void load(const T* board, int col, int q) {
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = *reinterpret_cast<const typename Raw<T>::type*>(board + (8 * q + i) * kS + 4 * col);
    }
    // One scale for the board.
    __device__ __forceinline__ void convert() {
        back = 1.0f;
        uneven = false;
        float scale[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (kTerms == 2) {
            float largest = 0.0f;
#pragma unroll
            for (int i = 0; i < 32; ++i) largest = larger(largest, fabsf(raw[i >> 2][i & 3]));
            uneven = range_of(largest);
            scale_of(largest, -100, scale[0], back);
            scale[1] = scale[2] = scale[3] = scale[0];
        }
        terms(scale);
    }
    // One for each square, by its own largest: squares that a list of moves leaves out may hold anything, and one whose
    // moves are out of the question costs the others nothing.
    __device__ __forceinline__ void convert_squares(f32x4& squares_back) {
        float scale[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (kTerms == 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float largest = fabsf(raw[0][j]), b;
#pragma unroll
                for (int i = 1; i < 8; ++i) largest = larger(largest, fabsf(raw[i][j]));
                scale_of(rows_max(largest), -100, scale[j], b);
                squares_back[j] = b;
            }
        }
        terms(scale);
    }
    __device__ __forceinline__ void terms(const float (&scale)[4]) {
        u32x2 rows[kTerms][8];                   // pairs of squares
        if constexpr (kTerms == 2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int j = 2 * (i & 1);
                unsigned hi, lo;
                Arith<T>::split(raw[i >> 1][j] * scale[j], raw[i >> 1][j + 1] * scale[j + 1], hi, lo);
                rows[0][i >> 1][i & 1] = hi;
                rows[1][i >> 1][i & 1] = lo;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) rows[0][i] = __builtin_bit_cast(u32x2, raw[i]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int k = 0; k < kTerms; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    column[j][k][i] = __builtin_amdgcn_perm(rows[k][2 * i + 1][j >> 1], rows[k][2 * i][j >> 1],
                                                            j & 1 ? 0x07060302u : 0x05040100u);
    }
};

// Square 4 col + j is row 16 j + col of 64 rows of channels or filters in LDS.
template <int TERMS>
__device__ __forceinline__ void write_rows(short* rows, int col, int q, const u32x4 (&v)[4][TERMS]) {
#pragma unroll
    for (int i = 0; i < 4 * TERMS; ++i)
        *reinterpret_cast<u32x4*>(rows + (i % TERMS) * kTerm + (16 * (i / TERMS) + col) * kRow + 8 * q) = v[i / TERMS][i % TERMS];
}

// A transposed read: a lane names four elements of one row (group of 16 lanes: four rows) and gets one column's element of
// the four rows.  Two make the eight k of an operand of 16 rows or columns; lo and hi are the lane's row of the first and
// of the second four.
__device__ __forceinline__ u32x4 transposed(const short* lo, const short* hi) {
    typedef __attribute__((address_space(3))) short4v* lds_short4;
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4)lo));
    const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4)hi));
    return u32x4{a[0], a[1], b[0], b[1]};
}

// Boards without a target: loss 0, gradient 0.
template <typename T>
__device__ __forceinline__ void zero_features_grad(T* board, int lane) {
    u32x4* out = reinterpret_cast<u32x4*>(board);
#pragma unroll
    for (int i = 0; i < (int)(kC * kS * sizeof(T) / 1024); ++i) out[i * 64 + lane] = u32x4{0, 0, 0, 0};
}

// g[4 a + j]: rows channel 16 a + 4 q + r, columns square 4 col + j
template <typename T>
__device__ __forceinline__ void store_features_grad(T* board, int col, int q, const f32x4 (&g)[8], float back) {
    typedef typename Raw<T>::type raw_t;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int a = i >> 2, r = i & 3;
        *reinterpret_cast<raw_t*>(board + (16 * a + 4 * q + r) * kS + 4 * col) =
            raw_t{(T)(g[4 * a][r] * back), (T)(g[4 * a + 1][r] * back), (T)(g[4 * a + 2][r] * back), (T)(g[4 * a + 3][r] * back)};
    }
}

// The workgroup's part of the kernel's gradient: dw[a][t] of every wave, rows channel 16 a + 4 q + r, columns the filters
// that filter_of(t, col) says; the waves' LDS lies `stride` bytes apart.
template <typename F>
__device__ __forceinline__ void store_part(const f32x4 (&dw)[2][kTiles], unsigned char* first, int stride, int wave, int waves,
                                           int col, int q, float* __restrict__ part, F&& filter_of) {
    float* mine = reinterpret_cast<float*>(first + wave * stride);
#pragma unroll
    for (int i = 0; i < 8 * kTiles; ++i) {
        const int a = i / (4 * kTiles), t = i / 4 % kTiles, r = i & 3;
        mine[(16 * a + 4 * q + r) * (16 * kTiles) + filter_of(t, col)] = dw[a][t][r];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kPart / 4; i += blockDim.x) {
        f32x4 a = {0, 0, 0, 0};
#pragma unroll 4
        for (int k = 0; k < waves; ++k) a += reinterpret_cast<const f32x4*>(first + k * stride)[i];
        reinterpret_cast<f32x4*>(part)[i] = a;
    }
}

// The kernel's scale, by its largest element.  Every wave looks at all of it (9 KB out of the cache, loads that are
// in flight beside those of its operands), which spares a pass through LDS and a barrier.
template <typename T>
__device__ __forceinline__ bool head_scale(const T* __restrict__ w, int lane, float& scale, float& back) {
    scale = back = 1.0f;
    bool uneven = false;
    if constexpr (Arith<T>::kTerms == 2) {
        constexpr int kPieces = kXW / 4, kLoads = (kPieces + 63) / 64;
        f32x4 v[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) v[i] = reinterpret_cast<const f32x4*>(w)[min(i * 64 + lane, kPieces - 1)];
        float largest = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * kLoads; ++i) largest = larger(largest, fabsf(v[i >> 2][i & 3]));
        uneven = range_of(largest);
        scale_of(largest, -100, scale, back);
    }
    return uneven;
}

// Eight values as an operand.
template <typename T>
__device__ __forceinline__ void operand(const float (&v)[8], float scale, u32x4 (&out)[Arith<T>::kTerms]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (Arith<T>::kTerms == 2) {
            unsigned hi, lo;
            Arith<T>::split(v[2 * i] * scale, v[2 * i + 1] * scale, hi, lo);
            out[0][i] = hi;
            out[1][i] = lo;
        } else {
            typedef T pair __attribute__((ext_vector_type(2)));
            out[0][i] = __builtin_bit_cast(unsigned, pair{(T)v[2 * i], (T)v[2 * i + 1]});
        }
    }
}

// c[i] += a(i) b(i) for products of operands of one or two terms each, the least of four left out.  An MFMA that waits for
// the one before it takes twice as long, so the N sums take turns; the barriers keep the compiler from undoing that.
template <typename T, int TA, int TB, int N, typename A, typename B>
__device__ __forceinline__ void products(f32x4 (&c)[N], A&& a, B&& b) {
#pragma unroll
    for (int k = (TA - 1) + (TB - 1); k >= 0; --k) {
        const int ka = k == 2 ? 1 : TB == 1 ? k : 0, kb = k == 2 ? 0 : TB == 1 ? 0 : k;
#pragma unroll
        for (int i = 0; i < N; ++i) c[i] = Arith<T>::mfma(a(i, ka), b(i, kb), c[i]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// What a call asks for beside the loss.
enum { kFeaturesGrad = 1, kKernelGrad = 2 };

// ---- the whole vocabulary --------------------------------------------------------------------------------------------
//
// One wave a board, everything between the features and the gradients in its registers.
//
//   logits   rows filter (five tiles of 16, 73 padded to 80), columns square, k channel.  Column col of tile j is square
//            4 col + j, so that a lane's features are four neighbours in memory.
//   dX       rows channel, columns square, k filter.  k is numbered so that a lane's eight are the filters whose logits
//            it holds already: the probabilities become an operand where they are.
//   dW       rows channel, columns filter, k square: features and probabilities are written to LDS a square's channels
//            or filters at a time, as they lie in the lanes, and read transposed (32 filters at a time); the sums stay
//            in registers over all the wave's boards.
//
// Loss and both gradients of 65 536 float32 boards: 274 to 283 us, 3.9 TB/s of features and gradients (a copy reaches
// 4.75), 322 on average from a cold start; of 32 768 bfloat16 boards 97 us.  Bound by issue: of a board's 5 600 cycles a
// SIMD the 765 (bfloat16; float32 895) vector instructions take 3 400 and the 108 (192) MFMAs 1 700 (3 100), with two
// waves of 220 to 256 registers a SIMD to overlap them.  The loss alone reads 65 536 float32 boards in 119 us, 4.5 TB/s.

template <typename T>
struct HeadLds {                                 // the kernel as operands, 16 bytes a lane
    // five for the logits: rows filter, k channel; 2 u + a: rows channel, k filter as the logits' results hold them
    u32x4 operand[kTiles + 6][Arith<T>::kTerms][64];
};
constexpr int kWaveLds = 2 * kTerm * 2;          // bytes a wave: the crossing
static_assert(kWaveLds >= kPartBytes, "at the end it takes the wave's kernel gradient");

// Two float16 terms lose 2^-38 of the largest factor.  That shows where the largest takes no part: in logits, where a filter
// that a column of -1e30 takes out of the softmax makes the others' products small beside it, in gradients too where the
// products are ordinary.  So a float32 board goes by float32 MFMAs, three times as long (65 536 in 1.16 ms), if its largest
// feature and the kernel's largest element make 2^12 or more or are not finite, or if features or kernel are uneven:
// some lane's 32 and more have a largest 2^16 below the largest of all.
constexpr float kWide = 0x1p-16f;                // 2^(12 - 2) by the scales' reciprocals, 2^-13 each

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// v as the main path has it, in units of 1: rows filter, columns square, k channel 8 q + i in step i
template <typename T>
__device__ __forceinline__ void wide_logits(const T* __restrict__ board, const T* __restrict__ w, int col, int q, f32x16 (&v)[kTiles]) {
    Features<T> f;
    f.load(board, col, q);
    asm volatile("" : "+v"(col), "+v"(q));       // addresses worked out here, not kept through the main path
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        f32x4 l[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
        const T* filter = w + 8 * q * kF + min(16 * t + col, kF - 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = (float)filter[i * kF];
#pragma unroll
            for (int j = 0; j < 4; ++j) l[j] = mfma_f32(a, (float)f.raw[i][j], l[j]);
            __builtin_amdgcn_sched_barrier(0);       // no loads ahead: the registers are the main path's
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) v[t][k] = l[k >> 2][k & 3];
    }
}

// The filter of column `col` of tile t of the kernel's gradient: c of a pair of tiles is 16 (c >> 2 & 1) + 4 (c >> 3) + (c & 3)
// of the pair's 32.
__device__ __forceinline__ int filter_of(int t, int col) {
    const int c = 16 * (t & 1) + col;
    return t == kTiles - 1 ? 64 + col : 32 * (t >> 1) + 16 * (c >> 2 & 1) + 4 * (c >> 3) + (c & 3);
}

// Both gradients from v = the logits' gradients times z.
template <int WANT, typename T>
__device__ __forceinline__ void wide_gradients(const T* __restrict__ board, const T* __restrict__ w, float* crossing, int lane, float rz,
                                               float weight, f32x16 (&v)[kTiles], T* __restrict__ dx, f32x4 (&dw)[2][kTiles]) {
    asm volatile("" : "+v"(lane));
    const int col = lane & 15, q = lane >> 4;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int k = 0; k < 16; ++k) v[t][k] *= rz;
    if (WANT & kFeaturesGrad) {                  // k filter: a step takes row r of the four lanes' results where it is
        f32x4 g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int f = 16 * t + 4 * q + r;
                const T* channel = w + col * kF + min(f, kF - 1);
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const float e = (float)channel[16 * a * kF], k = f < kF ? e : 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) g[4 * a + j] = mfma_f32(k, v[t][4 * j + r], g[4 * a + j]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        store_features_grad(dx, col, q, g, weight);
    }
    if (WANT & kKernelGrad) {                    // k square: a pair of tiles crosses the lanes by LDS, a square's 32 filters a row
        constexpr int kPitch = 36;
        static_assert(kS * kPitch * 4 <= kWaveLds, "a pair of tiles");
#pragma unroll
        for (int u = 0; u < 3; ++u) {
            const int tiles = u < 2 ? 2 : 1;
#pragma unroll
            for (int i = 0; i < 4 * tiles; ++i) {
                const f32x16& p = v[2 * u + (i >> 2)];
                const int j = i & 3;
                *reinterpret_cast<f32x4*>(crossing + (4 * col + j) * kPitch + 16 * (i >> 2) + 4 * q) =
                    f32x4{p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]};
            }
            lds_fence();
            f32x4 s[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll 1
            for (int k = q; k < kS; k += 4) {
                const float a[2] = {(float)board[col * kS + k], (float)board[(16 + col) * kS + k]};
#pragma unroll
                for (int i = 0; i < 2 * tiles; ++i)
                    s[i] = mfma_f32(a[i & 1], crossing[k * kPitch + (filter_of(2 * u + (i >> 1), col) - 32 * u)], s[i]);
            }
#pragma unroll
            for (int i = 0; i < 2 * tiles; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) dw[i & 1][2 * u + (i >> 1)][r] = fmaf(s[i][r], weight, dw[i & 1][2 * u + (i >> 1)][r]);
            lds_fence();
        }
    }
}

template <typename T, int WANT>
__global__ __launch_bounds__(512, WANT ? 2 : 3) void k_policy_loss(const T* __restrict__ x, const T* __restrict__ w, size_t n,
                                                     const int64_t* __restrict__ targets, const float* __restrict__ weights,
                                                     unsigned weight_step, float* __restrict__ loss, T* __restrict__ dx,
                                                     float* __restrict__ dw_part, int* __restrict__ err) {
    constexpr int NT = Arith<T>::kTerms;
    extern __shared__ __align__(16) unsigned char smem[];
    HeadLds<T>& lds = *reinterpret_cast<HeadLds<T>*>(smem);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int col = lane & 15, q = lane >> 4;
    short* mine = reinterpret_cast<short*>(smem + sizeof(HeadLds<T>) + wave * kWaveLds);   // kernel gradients only
    const short* read_at = mine + (8 * q + (col >> 2)) * kRow + 4 * (col & 3);
    auto crossed = [&](int term, int h, int tile) {      // columns 16 tile ..., k the rows 32 h + 8 q ...
        const short* p = read_at + term * kTerm + 32 * h * kRow + 16 * tile;
        return transposed(p, p + 4 * kRow);
    };

    Features<T> features;
    const size_t step = (size_t)gridDim.x * waves;
    size_t base = (size_t)wave * gridDim.x + blockIdx.x; // lane i looks after board base + i step
    int64_t t64;
    float my_weight;
    auto look_up = [&](int lane) {
        const size_t b = base + lane * step;
        t64 = b < n ? targets[b] : -1;
        my_weight = WANT && b < n ? weights[b * weight_step] : 0.0f;
    };
    // the first board's loads are under way while the kernel is prepared
    look_up(lane);
    if (base < n) features.load(x + base * (kC * kS), col, q);

    float w_back;
    bool w_uneven;
    {
        // an operand a wave at a time: five for the logits, six for the way back; all of a wave's are read at once
        constexpr int kOperands = kTiles + (WANT & kFeaturesGrad ? 6 : 0), kRounds = (kOperands + 3) / 4;
        T v[kRounds][8];
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int i = min(wave + r * waves, kOperands - 1), j = i - kTiles;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int c = i < kTiles ? 8 * q + k : 16 * (j & 1) + col;
                const int f = i < kTiles ? 16 * i + col : 32 * (j >> 1) + 16 * (k >> 2) + 4 * q + (k & 3);
                v[r][k] = w[c * kF + min(f, kF - 1)];
            }
        }
        float w_scale;
        w_uneven = head_scale<T>(w, lane, w_scale, w_back);
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int i = wave + r * waves, j = i - kTiles;
            float e[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)          // the padding's filters are zero
                e[k] = (i < kTiles ? 16 * i + col : 32 * (j >> 1) + 16 * (k >> 2) + 4 * q + (k & 3)) < kF ? (float)v[r][k] : 0.0f;
            u32x4 out[NT];
            operand<T>(e, w_scale, out);
            if (i < kOperands)
#pragma unroll
                for (int k = 0; k < NT; ++k) lds.operand[i][k][lane] = out[k];
        }
        __syncthreads();
    }

    f32x4 dw[2][kTiles];
    if (WANT & kKernelGrad)
#pragma unroll
        for (int i = 0; i < 2 * kTiles; ++i) dw[i / kTiles][i % kTiles] = f32x4{0, 0, 0, 0};

    for (bool loaded = true; base < n; base += 64 * step, loaded = false) {
        int mine_at = lane;
        asm volatile("" : "+v"(mine_at));        // worked out here, not kept in registers through the loop
        if (!loaded) look_up(mine_at);
        const bool in = base + mine_at * step < n, valid = t64 >= 0 && t64 < kVocab;
        const int my_target = (int)t64;
        if (in && !valid) {                      // no part in anything, whatever the features hold
            if (t64 != -1) atomicOr(err, 1);
            if (loss) loss[base + mine_at * step] = 0.0f;
        }
        if (WANT & kFeaturesGrad)
            for (uint64_t left = __ballot(in && !valid); left; left &= left - 1)
                zero_features_grad(dx + (base + __builtin_ctzll(left) * step) * (kC * kS), lane);
        uint64_t left = __ballot(valid);
        if (left && !(loaded && (left & 1))) features.load(x + (base + __builtin_ctzll(left) * step) * (kC * kS), col, q);
        while (left) {
            const int who = __builtin_ctzll(left);
            const size_t b = base + who * step;
            left &= left - 1;
            const T* next = x + (base + (left ? __builtin_ctzll(left) : 0) * step) * (kC * kS);   // read ahead; after the last, in vain
            const int target = __builtin_amdgcn_readlane(my_target, who);

            features.convert();
            const u32x4 (&xc)[4][NT] = features.column;
            const float x_back = features.back;
            // From logits in units of `unit` to the loss and v = the logits' gradients times z; the others' come from
            // the target's, d_target.
            auto solve = [&](f32x16 (&v)[kTiles], float unit, float& rz, float& d_target) __attribute__((always_inline)) {
                // the padding's filters 73 ... 79
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (64 + 4 * q + r >= kF) v[kTiles - 1][4 * j + r] = -INFINITY;

                // the target's place: tile, register and lane are uniform
                const int tf = target >> 6, ts = target & 63;
                const int t_tile = tf >> 4, t_reg = (ts & 3) * 4 + (tf & 3), t_lane = (tf >> 2 & 3) * 16 + (ts >> 2);
                auto at_target = [&](auto&& change) {    // returns what the target's lane then holds
                    float e = 0.0f;
#pragma unroll
                    for (int t = 0; t < kTiles; ++t)
                        if (t == t_tile) {
                            e = change(v[t][t_reg]);
                            v[t][t_reg] = e;
                            asm volatile("" : "+v"(e));  // keeps the branch
                        }
                    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e), t_lane));
                };
                float l_target = at_target([&](float e) { return e; });

                float top = -INFINITY;
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
#pragma unroll
                    for (int k = 0; k < 16; k += 2) top = larger(top, larger(v[t][k], v[t][k + 1]));
                top = lanes_reduce<true>(top);
                // exp(l - top) = 2^(l unit - top unit); an error of the rounded second product is common to all of the board.
                // Where the products pass float32's range, or their rounding shows, the largest is subtracted first.
                if (fabsf(top) * unit > 4096.0f) {
#pragma unroll
                    for (int t = 0; t < kTiles; ++t)
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[t][k] -= top;
                    l_target -= top;
                    top = 0.0f;
                }
                const float unit2 = unit * 1.44269504088896341f, top2 = -(top * unit2);
                float z4[4] = {};
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        v[t][k] = __builtin_amdgcn_exp2f(fmaf(v[t][k], unit2, top2));
                        z4[k & 3] += v[t][k];
                    }
                const float z = lanes_reduce<false>((z4[0] + z4[1]) + (z4[2] + z4[3]));
                if (loss && lane == 0) loss[b] = fmaf(__builtin_amdgcn_logf(z), 0.693147180559945309f, (top - l_target) * unit);
                if (!WANT) return;
                // the logits' gradients times z: exponentials, less z at the target.  The target's is the largest but for
                // rounding: z's own, up to 90 * 2^-24, can make the target's smaller than another by as much, which the least
                // scale covers.
                rz = __builtin_amdgcn_rcpf(z);
                d_target = at_target([&](float e) { return e - (lane == t_lane ? z : 0.0f); }) * rz;
            };
            if (NT == 2 && __builtin_expect(!(w_back * x_back <= kWide) || w_uneven || features.uneven, 0)) {
                const T* board = x + b * (kC * kS);
                f32x16 v[kTiles];
                wide_logits(board, w, col, q, v);
                float rz, d_target;
                solve(v, 1.0f, rz, d_target);
                const float weight = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_weight), who));
                if (WANT) wide_gradients<WANT>(board, w, reinterpret_cast<float*>(mine), lane, rz, weight, v, dx + b * (kC * kS), dw);
                features.load(next, col, q);
                continue;
            }
            if (WANT == 0) features.load(next, col, q);
            u32x4 xr[2][2][NT];                      // and as rows (channel, k square) for dW
            if (WANT & kKernelGrad) {
                write_rows<NT>(mine, col, q, xc);
                lds_fence();
#pragma unroll
                for (int i = 0; i < 4 * NT; ++i) xr[i / NT >> 1][i / NT & 1][i % NT] = crossed(i % NT, i / NT & 1, i / NT >> 1);
                lds_fence();
            }

            // logits, in units of 2^-(scales)
            f32x16 v[kTiles];                        // [tile of filters][4 * square + row]
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                u32x4 a[NT];
#pragma unroll
                for (int k = 0; k < NT; ++k) a[k] = lds.operand[t][k][lane];
                f32x4 l[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
                products<T, NT, NT>(l, [&](int, int k) { return a[k]; }, [&](int j, int k) { return xc[j][k]; });
#pragma unroll
                for (int k = 0; k < 16; ++k) v[t][k] = l[k >> 2][k & 3];
            }
            float rz, d_target;
            solve(v, fmaxf(w_back * x_back, 1e-36f), rz, d_target);
            if (!WANT) continue;
            float inv = 1.0f, wb = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_weight), who));
            if constexpr (Arith<T>::kScaled) {
                float d_scale, d_back;
                scale_of(fabsf(d_target), -17, d_scale, d_back);
                inv = d_scale * rz;
                wb *= d_back;
            } else {
                wb *= rz;
            }

            f32x4 g[8];                              // [4 * half of channels + square of four]
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = f32x4{0, 0, 0, 0};
            const float w_scale = wb * x_back;
#pragma unroll
            for (int u = 0; u < 3; ++u) {
                const int tiles = u < 2 ? 2 : 1;
                u32x4 d[4][2];                       // [square of four][term]: eight filters
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        unsigned hi = 0, lo = 0;
                        if (i < 2 * tiles) {
                            const f32x16& p = v[2 * u + (i >> 1)];
                            const int k = 4 * j + 2 * (i & 1);
                            if constexpr (Arith<T>::kScaled) Arith<T>::split(p[k] * inv, p[k + 1] * inv, hi, lo);
                            else Arith<T>::split(p[k], p[k + 1], hi, lo);
                        }
                        d[j][0][i] = hi;
                        d[j][1][i] = lo;
                    }
                if (u == 0) features.load(next, col, q);   // the first two tiles' registers are free
                if (WANT & kKernelGrad) {
                    if (tiles == 2) write_rows<2>(mine, col, q, d);
                    else
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<u32x2*>(mine + (i & 1) * kTerm + (16 * (i >> 1) + col) * kRow + 4 * q) =
                                u32x2{d[i >> 1][i & 1][0], d[i >> 1][i & 1][1]};
                    lds_fence();
                }
                if (WANT & kFeaturesGrad) {
                    u32x4 wk[2][NT];
#pragma unroll
                    for (int i = 0; i < 2 * NT; ++i) wk[i / NT][i % NT] = lds.operand[kTiles + 2 * u + i / NT][i % NT][lane];
                    products<T, NT, 2>(g, [&](int i, int k) { return wk[i >> 2][k]; }, [&](int i, int k) { return d[i & 3][k]; });
                }
                if (WANT & kKernelGrad) {
                    auto sums = [&](auto& s) {       // [2 * tile + half of channels]
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            u32x4 dk[2][2];
#pragma unroll
                            for (int i = 0; i < 2 * tiles; ++i)
                                dk[i >> 1][i & 1] = crossed(i & 1, h, i >> 1);
                            products<T, NT, 2>(s, [&](int i, int k) { return xr[i & 1][h][k]; }, [&](int i, int k) { return dk[i >> 1][k]; });
                        }
#pragma unroll
                        for (int i = 0; i < 2 * tiles; ++i)
#pragma unroll
                            for (int r = 0; r < 4; ++r) dw[i & 1][2 * u + (i >> 1)][r] = fmaf(s[i][r], w_scale, dw[i & 1][2 * u + (i >> 1)][r]);
                    };
                    if (tiles == 2) {
                        f32x4 s[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
                        sums(s);
                    } else {
                        f32x4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
                        sums(s);
                    }
                    lds_fence();
                }
            }
            if (WANT & kFeaturesGrad) store_features_grad(dx + b * (kC * kS), col, q, g, wb * w_back);
        }
    }
    if (WANT & kKernelGrad)
        store_part(dw, smem + sizeof(HeadLds<T>), kWaveLds, wave, waves, col, q, dw_part + (size_t)blockIdx.x * kPart, filter_of);
}

// ---- the boards' own moves -------------------------------------------------------------------------------------------
//
// One wave a board again.  A list of 32 moves needs a hundredth of the vocabulary's products, and MFMAs make them nearly
// free where the operands are cheap to gather: the features lie in LDS as rows of a square's channels, the kernel as rows of a
// filter's, and a move names one of each.
//
//   logits   16 moves' features times the same 16 moves' filters: the diagonal
//   dX       rows channel, columns square, k move: the filters' rows by a transposed read, the gradients of the logits
//            each in the column of its move's square, zero in the others
//   dW       rows channel, columns filter, k move: the squares' rows, the gradients in the columns of their filters
//
// float32: every filter and every square has a scale of its own, so that what the list leaves out, or what the softmax
// does, takes no bits from the rest.  The logits' gradients then carry the filters' units into dX and the squares' into dW,
// as two pairs of terms, each scaled by its own largest (one scale a board and kernel: 239 in place of 245 us, and wrong
// where an unlisted square was 1e5 times larger).
//
// What bounds it is reading the features and writing their gradient: 65 536 float32 boards with lists of 32 moves in 245 us,
// 4.4 TB/s (a copy reaches 4.75), 8 191 bfloat16 boards in 30 us, the loss alone of 65 536 float32 boards in 109 us.  (One
// float32 sum a move, with the gradients added up in LDS, took 342 us: its chains of reads and writes left the memory
// idle; LDS's own float adds take 200 cycles each and 880 us.)  A wave's boards are neighbours: it finds where its
// lists begin by adding up the counts of all boards before its own, and needs no pass over them beforehand: a byte a
// board for every workgroup after it, out of the caches, 128 (gradients) to 512 (16-bit losses) a board on average beside the
// board's own 4 to 16 KB.  At 2^20 boards it does not show: 4.7 (gradients) and 4.9 TB/s (loss, bfloat16), 5.2 (float32).

template <typename T>
struct MoveHeadLds {
    short rows[Arith<T>::kTerms][kF][kRow];      // [filter][channel]
    float back[Arith<T>::kTerms == 2 ? (kF + 3) / 4 * 4 : 4];   // float32: one over the filter's scale
    uint64_t sum[8];
};
static_assert(sizeof(MoveHeadLds<float>) % 16 == 0 && sizeof(MoveHeadLds<__bf16>) % 16 == 0, "the waves' parts are aligned");
template <typename T>
struct __attribute__((aligned(16))) MoveList {   // a board's moves, up to a multiple of 32; beyond its last, that again
    static constexpr int kGradients = Arith<T>::kTerms;
    float logit[256];
    // terms of the logits' gradients; float32: times one over the scale of the move's filter, for dX, and of its square, for dW
    unsigned short hi[kGradients][256], lo[kGradients][256];
    float back[Arith<T>::kTerms == 2 ? kS : 4];  // float32: one over the square's scale
    unsigned char square[256], filter[256];      // square: its row of features
    unsigned square_tile[4][16];                 // for 32 moves, a pair a word: which of the pair is in the tile of columns
    unsigned filter_tile[kTiles][16];
};
template <typename T>
constexpr unsigned move_wave_bytes(int want) {
    const unsigned rows = Arith<T>::kTerms * kTerm * 2, most = rows + sizeof(MoveList<T>);
    return (want & kKernelGrad) && most < (unsigned)kPartBytes ? kPartBytes : most;
}

struct __attribute__((packed)) Bytes16 { unsigned v[4]; };

__device__ __forceinline__ unsigned lanes_add(unsigned v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// 0xffff in the half of each that is set
__device__ __forceinline__ unsigned halves(bool low, bool high) { return (low ? 0xffffu : 0u) | (high ? 0xffff0000u : 0u); }

template <typename T, int WANT>
__global__ __launch_bounds__(512) void k_policy_move_loss(const T* __restrict__ x, const T* __restrict__ w, size_t n,
                                                          const uint8_t* __restrict__ from, const uint8_t* __restrict__ filter,
                                                          const uint8_t* __restrict__ per, size_t n_moves,
                                                          const int64_t* __restrict__ targets, const float* __restrict__ weights,
                                                          unsigned weight_step, float* __restrict__ loss, T* __restrict__ dx,
                                                          float* __restrict__ dw_part, int* __restrict__ err) {
    constexpr int NT = Arith<T>::kTerms;
    extern __shared__ __align__(16) unsigned char smem[];
    MoveHeadLds<T>& head = *reinterpret_cast<MoveHeadLds<T>*>(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
    const int col = lane & 15, q = lane >> 4;
    unsigned char* const first_wave = smem + sizeof(MoveHeadLds<T>);
    short* rows = reinterpret_cast<short*>(first_wave + wave * move_wave_bytes<T>(WANT));
    MoveList<T>& list = *reinterpret_cast<MoveList<T>*>(rows + NT * kTerm);

    // the wave's boards [lo, hi)
    const size_t all = (size_t)gridDim.x * waves, me = (size_t)blockIdx.x * waves + wave;
    const size_t lo = n * me / all, hi = n * (me + 1) / all, group_lo = n * (me - wave) / all;
    Features<T> features;
    size_t base = lo;                            // lane i looks after board base + i
    unsigned listed;
    int64_t t64;
    float my_weight;
    auto look_up = [&] {
        const size_t b = base + lane;
        listed = b < hi ? per[b] : 0u;
        t64 = b < hi ? targets[b] : -1;
        my_weight = WANT && b < hi ? weights[b * weight_step] : 0.0f;
    };
    // the first board's loads are under way while the kernel is prepared
    look_up();
    if (base < hi) features.load(x + base * (kC * kS), col, q);

    {
        constexpr int kRounds = 2;               // (filter, eight channels) a thread; at least 256 threads
        T v[kRounds][8];
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int i = min(tid + r * (int)blockDim.x, kF * 4 - 1);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[r][k] = w[(8 * (i & 3) + k) * kF + (i >> 2)];
        }
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int i = tid + r * (int)blockDim.x;
            float e[8], w_scale = 1.0f, w_back = 1.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = (float)v[r][k];
            if constexpr (NT == 2) {             // the filter's scale, by its four threads
                float largest = fabsf(e[0]);
#pragma unroll
                for (int k = 1; k < 8; ++k) largest = larger(largest, fabsf(e[k]));
                largest = larger(largest, __shfl_xor(largest, 1));
                largest = larger(largest, __shfl_xor(largest, 2));
                scale_of(largest, -100, w_scale, w_back);
            }
            u32x4 out[NT];
            operand<T>(e, w_scale, out);
            if (i < kF * 4) {
#pragma unroll
                for (int k = 0; k < NT; ++k) *reinterpret_cast<u32x4*>(&head.rows[k][i >> 2][8 * (i & 3)]) = out[k];
                if (NT == 2 && (i & 3) == 0) head.back[i >> 2] = w_back;
            }
        }
        static_assert(kF * 4 <= kRounds * 256, "every element");
    }

    // where their lists begin
    unsigned before = 0;
    for (size_t i = (size_t)tid * 16; i < group_lo; i += (size_t)blockDim.x * 16) {
        if (i + 16 <= group_lo) {
            const Bytes16 p = *reinterpret_cast<const Bytes16*>(per + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) before = __builtin_amdgcn_sad_u8(p.v[k], 0u, before);
        } else {
            for (size_t k = i; k < group_lo; ++k) before += per[k];
        }
    }
    before = lanes_add(before);
    if (lane == 0) head.sum[wave] = before;
    before = 0;
    for (size_t i = group_lo + lane; i < lo; i += 64) before += per[i];
    uint64_t start = lanes_add(before);
    __syncthreads();
    for (int i = 0; i < waves; ++i) start += head.sum[i];

    f32x4 dw[2][kTiles];
    if (WANT & kKernelGrad)
#pragma unroll
        for (int i = 0; i < 2 * kTiles; ++i) dw[i / kTiles][i % kTiles] = f32x4{0, 0, 0, 0};

    for (bool loaded = true; base < hi; base += 64, loaded = false) {
        if (!loaded) look_up();
        const bool in = base + lane < hi;
        unsigned upto = listed;                          // inclusive sum over the lanes
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned v = __shfl_up(upto, o);
            upto += lane >= o ? v : 0u;
        }
        const uint64_t my_first = min(start + upto - listed, (uint64_t)n_moves);
        const int my_count = (int)min((uint64_t)listed, n_moves - my_first);
        start += (unsigned)__builtin_amdgcn_readlane(upto, 63);
        const bool valid = t64 >= 0 && t64 < my_count;
        const int my_target = (int)t64;
        if (in && !valid) {                      // no part in anything, whatever the features hold
            if (t64 != -1) atomicOr(err, 1);
            if (loss) loss[base + lane] = 0.0f;
        }
        for (uint64_t left = __ballot(in && !valid); left; left &= left - 1) {
            const int who = __builtin_ctzll(left);
            if (WANT & kFeaturesGrad) zero_features_grad(dx + (base + who) * (kC * kS), lane);
            // its moves are looked over all the same
            const uint64_t first = (uint64_t)(unsigned)__builtin_amdgcn_readlane((unsigned)my_first, who) |
                                   (uint64_t)(unsigned)__builtin_amdgcn_readlane((unsigned)(my_first >> 32), who) << 32;
            for (int m = lane; m < __builtin_amdgcn_readlane(my_count, who); m += 64)
                if (from[first + m] >= kS || filter[first + m] >= kF) atomicOr(err, 1);
        }
        uint64_t left = __ballot(valid);
        if (!left) continue;

        uint64_t first;                          // of the board at hand
        int cnt;
        unsigned square, filt;                   // its first 64 moves
        auto fetch = [&](int who, bool loaded) {
            first = (uint64_t)(unsigned)__builtin_amdgcn_readlane((unsigned)my_first, who) |
                    (uint64_t)(unsigned)__builtin_amdgcn_readlane((unsigned)(my_first >> 32), who) << 32;
            cnt = __builtin_amdgcn_readlane(my_count, who);
            square = from[first + min(lane, cnt - 1)];
            filt = filter[first + min(lane, cnt - 1)];
            if (!loaded) features.load(x + (base + who) * (kC * kS), col, q);
        };
        int who = __builtin_ctzll(left);
        fetch(who, loaded && who == 0);
        while (true) {
            const size_t b = base + who;
            const int target = __builtin_amdgcn_readlane(my_target, who), count = cnt;
            const float weight = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_weight), who));
            f32x4 x_back;
            features.convert_squares(x_back);
            write_rows<NT>(rows, col, q, features.column);
            if (NT == 2 && q == 0) *reinterpret_cast<f32x4*>(&list.back[4 * col]) = x_back;
            const T* const board = x + b * (kC * kS);
            unsigned move[4];                        // [pass of 64 moves]: square, filter
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                if (64 * p >= count) continue;
                if (p) {
                    square = from[first + min(64 * p + lane, count - 1)];
                    filt = filter[first + min(64 * p + lane, count - 1)];
                }
                if (square >= kS || filt >= kF) atomicOr(err, 1);
                square = min(square, kS - 1u);
                filt = min(filt, kF - 1u);
                list.square[64 * p + lane] = (unsigned char)(16 * (square & 3) + (square >> 2));
                list.filter[64 * p + lane] = (unsigned char)filt;
                move[p] = square | filt << 8;
            }
            left &= left - 1;
            if (left) {
                who = __builtin_ctzll(left);
                fetch(who, false);
            }
            lds_fence();

            auto square_back = [&](int p) { return list.back[move[p] & 255u]; };
            auto filter_back = [&](int p) { return head.back[move[p] >> 8]; };
            // logits, float32 ones in units of their squares' and filters'
            for (int m = 0; m < count; m += 32) {
                u32x4 a[2][NT], f[2][NT];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int sq = list.square[m + 16 * i + col], fl = list.filter[m + 16 * i + col];
#pragma unroll
                    for (int k = 0; k < NT; ++k) {
                        a[i][k] = *reinterpret_cast<const u32x4*>(rows + k * kTerm + sq * kRow + 8 * q);
                        f[i][k] = *reinterpret_cast<const u32x4*>(&head.rows[k][fl][8 * q]);
                    }
                }
                f32x4 l[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
                products<T, NT, NT>(l, [&](int i, int k) { return a[i][k]; }, [&](int i, int k) { return f[i][k]; });
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float even = col & 2 ? l[i][2] : l[i][0], odd = col & 2 ? l[i][3] : l[i][1];
                    if (q == col >> 2) list.logit[m + 16 * i + col] = col & 1 ? odd : even;
                }
            }
            lds_fence();
            float v[4], top = -INFINITY;             // [pass of 64 moves]
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                v[p] = -INFINITY;
                if (64 * p >= count) continue;
                if (64 * p + lane < count) {
                    v[p] = list.logit[64 * p + lane];
                    if constexpr (NT == 2) {
                        const float unit = square_back(p) * filter_back(p);
                        v[p] *= unit;
                        if (!(unit <= kWide)) {      // as over the vocabulary: not finite, or wide
                            v[p] = 0.0f;
                            for (int c = 0; c < kC; ++c)
                                v[p] = fmaf((float)board[c * kS + (move[p] & 255u)], (float)w[c * kF + (move[p] >> 8)], v[p]);
                        }
                    }
                }
                top = larger(top, v[p]);
            }
            top = lanes_reduce<true>(top);
            float l_target = 0.0f, z = 0.0f;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                if (64 * p >= count) continue;
                if (p == target >> 6) l_target = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v[p]), target & 63));
                v[p] = __builtin_amdgcn_exp2f((v[p] - top) * 1.44269504088896341f);
                z += v[p];
            }
            z = lanes_reduce<false>(z);
            if (loss && lane == 0) loss[b] = fmaf(__builtin_amdgcn_logf(z), 0.693147180559945309f, top - l_target);

            if (WANT) {
                // the logits' gradients times z, as over the vocabulary
                const float rz = __builtin_amdgcn_rcpf(z);
                float inv = 1.0f, wb = weight;
                if constexpr (NT == 1) {
                    if constexpr (Arith<T>::kScaled) {
                        const float e_target = __builtin_amdgcn_exp2f((l_target - top) * 1.44269504088896341f);
                        float d_scale, d_back;
                        scale_of(fabsf(e_target - z) * rz, -17, d_scale, d_back);
                        inv = d_scale * rz;
                        wb *= d_back;
                    } else {
                        wb *= rz;
                    }
                }
                float wb_x = wb, wb_w = wb;          // what dX and dW are multiplied by
                // float32: each takes them in the units of its factor, scaled by the largest
                auto gradients = [&](int of, auto&& unit, float& back) {
                    float largest = 0.0f, scale = 1.0f, scale_back;
                    if constexpr (NT == 2) {
#pragma unroll
                        for (int p = 0; p < 4; ++p)
                            if (64 * p < count) largest = larger(largest, fabsf((v[p] - (64 * p + lane == target ? z : 0.0f)) * rz * unit(p)));
                        scale_of(lanes_reduce<true>(largest), -113, scale, scale_back);
                        back *= scale_back;
                    }
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        if (64 * p >= count) continue;
                        float d = v[p] - (64 * p + lane == target ? z : 0.0f);
                        if constexpr (NT == 2) d = d * rz * unit(p) * scale;
                        else d *= inv;
                        unsigned hi, lo;
                        Arith<T>::split(d, 0.0f, hi, lo);
                        list.hi[of][64 * p + lane] = (unsigned short)hi;
                        list.lo[of][64 * p + lane] = (unsigned short)lo;
                    }
                };
                constexpr int kOfX = 0, kOfW = NT - 1;
                if ((WANT & kFeaturesGrad) || NT == 1) gradients(kOfX, filter_back, wb_x);
                if ((WANT & kKernelGrad) && NT == 2) gradients(kOfW, square_back, wb_w);
                f32x4 g[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] = f32x4{0, 0, 0, 0};
                for (int m = 0; m < count; m += 32) {
                    {                                // pair `col`, tile q
                        const unsigned s2 = *reinterpret_cast<const unsigned short*>(&list.square[m + 2 * col]);
                        const unsigned f2 = *reinterpret_cast<const unsigned short*>(&list.filter[m + 2 * col]);
                        list.square_tile[q][col] = halves((s2 >> 4 & 15) == (unsigned)q, s2 >> 12 == (unsigned)q);
                        list.filter_tile[q][col] = halves((f2 >> 4 & 15) == (unsigned)q, f2 >> 12 == (unsigned)q);
                        if (q == 0) list.filter_tile[4][col] = halves((f2 >> 4 & 15) == 4, f2 >> 12 == 4);
                    }
                    lds_fence();
                    // the lane's eight moves m + 8 q ...: the terms, kept where the move's square or filter is in the lane's column
                    const int row_lo = m + 8 * q + (col >> 2), row_hi = row_lo + 4;   // whose row the lane names in a transposed read
                    auto in_column = [&](int term, const unsigned char* of, u32x4 (&out)[2]) {
                        const u32x4 d[2] = {*reinterpret_cast<const u32x4*>(&list.hi[term][m + 8 * q]),
                                            *reinterpret_cast<const u32x4*>(&list.lo[term][m + 8 * q])};
                        const u32x2 s8 = *reinterpret_cast<const u32x2*>(of + m + 8 * q);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const unsigned pair = s8[i >> 1] >> 16 * (i & 1);
                            const unsigned keep = halves((pair & 15) == (unsigned)col, (pair >> 8 & 15) == (unsigned)col);
                            out[0][i] = d[0][i] & keep;
                            out[1][i] = d[1][i] & keep;
                        }
                    };
                    if (WANT & kFeaturesGrad) {
                        u32x4 a[2][NT], mine[2], s[4][2];
                        const short* w_lo = &head.rows[0][list.filter[row_lo]][4 * (col & 3)];
                        const short* w_hi = &head.rows[0][list.filter[row_hi]][4 * (col & 3)];
#pragma unroll
                        for (int i = 0; i < 2 * NT; ++i) {
                            const int at = (i % NT) * kF * kRow + 16 * (i / NT);
                            a[i / NT][i % NT] = transposed(w_lo + at, w_hi + at);
                        }
                        in_column(kOfX, list.square, mine);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const u32x4 keep = *reinterpret_cast<const u32x4*>(&list.square_tile[j][4 * q]);
                            s[j][0] = mine[0] & keep;
                            s[j][1] = mine[1] & keep;
                        }
                        products<T, NT, 2>(g, [&](int i, int k) { return a[i >> 2][k]; }, [&](int i, int k) { return s[i & 3][k]; });
                    }
                    if (WANT & kKernelGrad) {
                        u32x4 a[2][NT], mine[2];
                        const short* x_lo = rows + list.square[row_lo] * kRow + 4 * (col & 3);
                        const short* x_hi = rows + list.square[row_hi] * kRow + 4 * (col & 3);
#pragma unroll
                        for (int i = 0; i < 2 * NT; ++i) {
                            const int at = (i % NT) * kTerm + 16 * (i / NT);
                            a[i / NT][i % NT] = transposed(x_lo + at, x_hi + at);
                        }
                        in_column(kOfW, list.filter, mine);
                        // float32's in two turns: all five tiles' operands and sums beside a[2][2] pass the registers
                        auto tiles = [&](auto first, auto end) {
                            constexpr int t0 = decltype(first)::value, N = decltype(end)::value - t0;
                            f32x4 sum[2 * N];
                            u32x4 f[N][2];
#pragma unroll
                            for (int t = 0; t < N; ++t) {
                                const u32x4 keep = *reinterpret_cast<const u32x4*>(&list.filter_tile[t0 + t][4 * q]);
                                f[t][0] = mine[0] & keep;
                                f[t][1] = mine[1] & keep;
                            }
#pragma unroll
                            for (int i = 0; i < 2 * N; ++i) sum[i] = f32x4{0, 0, 0, 0};
                            products<T, NT, 2>(sum, [&](int i, int k) { return a[i & 1][k]; }, [&](int i, int k) { return f[i >> 1][k]; });
#pragma unroll
                            for (int i = 0; i < 8 * N; ++i)
                                dw[i >> 2 & 1][t0 + (i >> 3)][i & 3] = fmaf(sum[i >> 2][i & 3], wb_w, dw[i >> 2 & 1][t0 + (i >> 3)][i & 3]);
                        };
                        constexpr int kTurn = NT == 2 ? 3 : kTiles;
                        tiles(std::integral_constant<int, 0>{}, std::integral_constant<int, kTurn>{});
                        if constexpr (kTurn < kTiles) tiles(std::integral_constant<int, kTurn>{}, std::integral_constant<int, kTiles>{});
                    }
                    lds_fence();
                }
                if (WANT & kFeaturesGrad) store_features_grad(dx + b * (kC * kS), col, q, g, wb_x);
            }
            lds_fence();
            if (!left) break;
        }
    }
    if (lo < hi && hi == n && lane == 0 && start != n_moves) atomicOr(err, 1);
    if (WANT & kKernelGrad) {
        __syncthreads();
        store_part(dw, first_wave, move_wave_bytes<T>(WANT), wave, waves, col, q, dw_part + (size_t)blockIdx.x * kPart,
                   [](int t, int col) { return 16 * t + col; });
    }
}

// The partial kernel gradients of the workgroups, added up in fixed order: a workgroup 32 elements, 32 threads each, whose
// loads are all in flight at once.
constexpr unsigned kGroups = 256;   // workgroups of a gradient call: one a compute unit, each with a part of the kernel's gradient
template <typename T>
__global__ __launch_bounds__(1024) void k_sum_parts(const float* __restrict__ part, unsigned parts, T* __restrict__ dw) {
    __shared__ double sums[32][33];
    const int i = threadIdx.x & 31, j = threadIdx.x >> 5;
    double a = 0.0;
#pragma unroll
    for (unsigned k = 0; k < kGroups / 32; ++k) {
        const unsigned p = j + 32 * k;
        a += p < parts ? part[(size_t)p * kPart + blockIdx.x * 32 + i] : 0.0f;
    }
    sums[i][j] = a;
    __syncthreads();
    a = sums[j][i];
#pragma unroll
    for (int o = 16; o; o >>= 1) a += __shfl_xor(a, o);
    const int e = blockIdx.x * 32 + j, c = e / (16 * kTiles), f = e % (16 * kTiles);
    if (i == 0 && f < kF) dw[c * kF + f] = (T)(float)a;
}
static_assert(kPart % 32 == 0, "k_sum_parts needs no bounds check");

template <typename T, int WANT>
hipError_t launch(const PolicyLossArgs& a, hipStream_t s) {
    const T *x = static_cast<const T*>(a.features), *w = static_cast<const T*>(a.kernel);
    T* dx = static_cast<T*>(a.d_features);
    float* part = static_cast<float*>(a.workspace);
    // At least four waves a workgroup, which share the work on the kernel's operands.  (Spreading a small call's boards over all
    // compute units, one or two a workgroup, leaves more parts to add up: 17.6 in place of 16.4 us for 512 boards.)
    // Without gradients more workgroups fit a compute unit, and as many are launched: of float32 three (registers) over the
    // vocabulary and two (LDS) over moves, else four.  One more that has to wait costs more than it brings: 40 000 boards
    // of float32 over moves in 62 us with two, 77 with three; 5 000 over the vocabulary in 14.2 us with three, 17.5 with four.
    const unsigned waves = WANT && a.n > 4 * kGroups ? 8 : 4, step = a.n_weights > 1 ? 1u : 0u;
    const unsigned most = WANT ? kGroups : (sizeof(T) == 2 ? 4 : a.per_board ? 2 : 3) * kGroups;
    const unsigned grid = (unsigned)std::min<size_t>((a.n + waves - 1) / waves, most);
    if (grid && a.per_board)
        hipLaunchKernelGGL((k_policy_move_loss<T, WANT>), dim3(grid), dim3(waves * 64),
                           sizeof(MoveHeadLds<T>) + waves * move_wave_bytes<T>(WANT), s, x, w, a.n,
                           a.from, a.filter, a.per_board, a.n_moves, a.targets, a.weights, step, a.loss, dx, part, a.err);
    else if (grid)
        hipLaunchKernelGGL((k_policy_loss<T, WANT>), dim3(grid), dim3(waves * 64),
                           sizeof(HeadLds<T>) + (WANT & kKernelGrad ? waves * kWaveLds : 0), s, x, w,
                           a.n, a.targets, a.weights, step, a.loss, dx, part, a.err);
    if (hipError_t e = hipGetLastError()) return e;
    if (WANT & kKernelGrad) hipLaunchKernelGGL(k_sum_parts<T>, dim3(kPart / 32), dim3(1024), 0, s, part, grid, static_cast<T*>(a.d_kernel));
    return hipGetLastError();
}

template <typename T>
hipError_t launch(const PolicyLossArgs& a, hipStream_t s) {
    if (a.d_features) return a.d_kernel ? launch<T, kFeaturesGrad | kKernelGrad>(a, s) : launch<T, kFeaturesGrad>(a, s);
    return a.d_kernel ? launch<T, kKernelGrad>(a, s) : launch<T, 0>(a, s);
}

}  // namespace

size_t policy_loss_workspace(size_t n) { return std::min<size_t>(n, kGroups) * kPartBytes; }

hipError_t launch_policy_loss(const PolicyLossArgs& a, hipStream_t stream) {
    if (a.type == BF_TYPE_F32) return launch<float>(a, stream);
    if (a.type == BF_TYPE_BF16) return launch<__bf16>(a, stream);
    return launch<_Float16>(a, stream);
}

}  // namespace bf
