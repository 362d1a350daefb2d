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

#include "../../include/batchfirst.h"
#include "bf_train.h"

namespace bf {
namespace {

constexpr int kC = 32, kS = 64, kF = 73, kVocab = kF * kS, kXW = kC * kF;
// ---- the whole vocabulary --------------------------------------------------------------------------------------------
//
// One wave a board, everything between the features and the gradients in its registers, on 16x16x32 MFMAs with float32
// sums.  Lane l = (n = l & 15, q = l >> 4) of an operand holds eight k (8 q ... 8 q + 7) of row or column n, of a result
// the rows 4 q ... 4 q + 3 of column n.
//
//   logits   rows filter (five tiles of 16, 73 padded to 80), columns square, k channel.  Column n of tile j is square
//            4 n + j, so that a lane's features are four neighbours in memory.
//   dX       rows channel, columns square, k filter.  k is numbered so that a lane's eight are the filters whose logits
//            it holds already: the probabilities become an operand where they are.
//   dW       rows channel, columns filter, k square: features and probabilities are written to LDS a square's channels
//            or filters at a time, as they lie in the lanes, and read transposed (32 filters at a time); the sums stay
//            in registers over all the wave's boards.
//
// float32 operands travel as two float16 terms (22 bits), scaled by a power of two, the kernel's by its largest element
// and the features' by the board's, so that the larger term stays normal down to 2^-29 of the largest; of the four products of terms the
// least is left out (2^-22).  bfloat16 and float16 operands are exact as they are.  The logits' gradients d (before the
// weight) travel as two terms: bfloat16 ones for bfloat16 features, else float16 ones, scaled like the features.  Their
// largest is the target's, which is the negative sum of all the others.

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
    // (a, b) = terms hi + lo, each packed with a in the low half; rounded towards zero, so lo has hi's sign
    static __device__ __forceinline__ void split(float a, float b, unsigned& hi, unsigned& lo) {
        const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
        hi = __builtin_bit_cast(unsigned, h);
        lo = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a - (float)h[0], b - (float)h[1]));
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

// 2^(13 - e) for a largest magnitude in [2^e, 2^(e+1)), and its reciprocal; magnitudes below 2^least count as that.
__device__ __forceinline__ void scale_of(float largest, int least, float& scale, float& back) {
    const int e = max((int)(__float_as_uint(largest) >> 23 & 255u) - 127, least);
    scale = __uint_as_float((unsigned)(127 + 13 - e) << 23);
    back = __uint_as_float((unsigned)(127 - 13 + e) << 23);
}

constexpr int kTiles = 5;                        // of filters
constexpr int kRow = 40;                         // 16-bit elements a square of the crossing: 32, and 16 rows in 16 different bank groups
constexpr int kTerm = kS * kRow;                 // elements a term
constexpr int kWaveLds = 2 * kTerm * 2;          // bytes a wave
static_assert(kWaveLds >= 64 * 40 * 4, "at the end it takes the wave's kernel gradient");

template <typename T>
struct HeadLds {                                 // the kernel as operands, 16 bytes a lane
    u32x4 logit[kTiles][Arith<T>::kTerms][64];   // rows filter, k channel
    u32x4 back[3][2][Arith<T>::kTerms][64];      // rows channel, k filter as the logits' results hold them
    float red[8];
};

// Eight values as an operand of one or two terms.
template <typename T>
__device__ __forceinline__ void operand(const float (&v)[8], float scale, u32x4 (&out)[Arith<T>::kTerms]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (Arith<T>::kTerms == 2) {
            unsigned hi, lo;
            Arith<T>::split(v[2 * i] * scale, v[2 * i + 1] * scale, hi, lo);
            out[0][i] = hi;
            out[1][i] = lo;
        } else if constexpr (sizeof(T) == 2) {
            typedef T pair __attribute__((ext_vector_type(2)));
            out[0][i] = __builtin_bit_cast(unsigned, pair{(T)v[2 * i], (T)v[2 * i + 1]});
        }
    }
}

// Fills the kernel's operands; returns the factor that takes a product of scaled operands' kernel part back.
template <typename T, bool GRAD>
__device__ __forceinline__ float load_head(const T* __restrict__ w, HeadLds<T>& lds) {
    float scale = 1.0f, back = 1.0f;
    const int tid = threadIdx.x, waves = blockDim.x >> 6;
    if constexpr (Arith<T>::kTerms == 2) {
        float largest = 0.0f;
        for (int i = tid; i < kXW; i += blockDim.x) largest = fmaxf(largest, fabsf((float)w[i]));
        largest = lanes_reduce<true>(largest);
        if ((tid & 63) == 0) lds.red[tid >> 6] = largest;
        __syncthreads();
        for (int i = 0; i < waves; ++i) largest = fmaxf(largest, lds.red[i]);
        scale_of(largest, -100, scale, back);
    }
    for (int i = tid; i < kTiles * 64; i += blockDim.x) {
        const int f = (i >> 6) * 16 + (i & 15), q = i >> 4 & 3;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = f < kF ? (float)w[(8 * q + k) * kF + f] : 0.0f;
        u32x4 out[Arith<T>::kTerms];
        operand<T>(v, scale, out);
#pragma unroll
        for (int k = 0; k < Arith<T>::kTerms; ++k) lds.logit[i >> 6][k][i & 63] = out[k];
    }
    if (GRAD)
        for (int i = tid; i < 6 * 64; i += blockDim.x) {
            const int u = i >> 7, a = i >> 6 & 1, c = a * 16 + (i & 15), q = i >> 4 & 3;
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int f = 32 * u + 16 * (k >> 2) + 4 * q + (k & 3);
                v[k] = f < kF ? (float)w[c * kF + f] : 0.0f;
            }
            u32x4 out[Arith<T>::kTerms];
            operand<T>(v, scale, out);
#pragma unroll
            for (int k = 0; k < Arith<T>::kTerms; ++k) lds.back[u][a][k][i & 63] = out[k];
        }
    __syncthreads();
    return back;
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

template <typename T, int WANT>
__global__ __launch_bounds__(512) void k_policy_loss(const T* __restrict__ x, const T* __restrict__ w, size_t n,
                                                     const int64_t* __restrict__ targets, const float* __restrict__ weights,
                                                     unsigned weight_step, float* __restrict__ loss, T* __restrict__ dx,
                                                     float* __restrict__ dw_part, int* __restrict__ err) {
    constexpr int NT = Arith<T>::kTerms;
    typedef typename Raw<T>::type raw_t;
    extern __shared__ __align__(16) unsigned char smem[];
    HeadLds<T>& lds = *reinterpret_cast<HeadLds<T>*>(smem);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int col = lane & 15, q = lane >> 4;
    // Crossing: square 4 col + j is row 16 j + col.  A lane of a transposed read names four elements of one row and gets
    // one column's element of four rows; two make an operand's eight k.
    typedef __attribute__((address_space(3))) short4v* lds_short4;
    short* mine = reinterpret_cast<short*>(smem + sizeof(HeadLds<T>) + wave * kWaveLds);   // kernel gradients only
    short* write_at = mine + col * kRow + 8 * q;
    short* read_at = mine + (8 * q + (col >> 2)) * kRow + 4 * (col & 3);
    auto transposed = [&](int term, int h, int tile) {   // columns 16 tile ..., rows 32 h + 8 q ...
        short* p = read_at + term * kTerm + 32 * h * kRow + 16 * tile;
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4)p));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4)(p + 4 * kRow)));
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };

    const size_t step = (size_t)gridDim.x * waves;
    size_t base = (size_t)blockIdx.x * waves + wave;     // lane i looks after board base + i step
    const float w_back = load_head<T, (WANT & kFeaturesGrad) != 0>(w, lds);
    raw_t raw[8];                                // channels 8 q ... 8 q + 7, squares 4 col ... 4 col + 3
    auto load = [&](size_t board) {
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = *reinterpret_cast<const raw_t*>(x + board * (kC * kS) + (8 * q + i) * kS + 4 * col);
    };

    f32x4 dw[2][kTiles];
    if (WANT & kKernelGrad)
#pragma unroll
        for (int i = 0; i < 2 * kTiles; ++i) dw[i / kTiles][i % kTiles] = f32x4{0, 0, 0, 0};

    for (; base < n; base += 64 * step) {
        const bool in = base + lane * step < n;
        const int64_t t64 = in ? targets[base + lane * step] : 0;
        const bool valid = in && t64 >= 0 && t64 < kVocab;
        const float my_weight = WANT && valid ? weights[(base + lane * step) * weight_step] : 0.0f;
        const int my_target = (int)t64;
        if (in && !valid) {                      // no part in anything, whatever the features hold
            if (t64 != -1) atomicOr(err, 8);
            if (loss) loss[base + lane * step] = 0.0f;
        }
        if (WANT & kFeaturesGrad)
            for (uint64_t left = __ballot(in && !valid); left; left &= left - 1) {
                u32x4* out = reinterpret_cast<u32x4*>(dx + (base + __builtin_ctzll(left) * step) * (kC * kS));
#pragma unroll
                for (int i = 0; i < (int)(kC * kS * sizeof(T) / 1024); ++i) out[i * 64 + lane] = u32x4{0, 0, 0, 0};
            }
        uint64_t left = __ballot(valid);
        if (left) load(base + __builtin_ctzll(left) * step);
      while (left) {
        const int who = __builtin_ctzll(left);
        const size_t b = base + who * step;
        left &= left - 1;
        const size_t next = base + (left ? __builtin_ctzll(left) : 0) * step;   // read ahead; after the last, in vain
        const int target = __builtin_amdgcn_readlane(my_target, who);

        // features in their terms, pairs of squares packed
        u32x2 rows[NT][8];
        float x_scale = 1.0f, x_back = 1.0f;
        if constexpr (sizeof(T) == 4) {
            float largest = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) largest = larger(largest, fabsf(raw[i][j]));
            scale_of(lanes_reduce<true>(largest), -100, x_scale, x_back);
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    unsigned hi, lo;
                    Arith<T>::split(raw[i][2 * j] * x_scale, raw[i][2 * j + 1] * x_scale, hi, lo);
                    rows[0][i][j] = hi;
                    rows[1][i][j] = lo;
                }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) rows[0][i] = __builtin_bit_cast(u32x2, raw[i]);
        }
        if (WANT == 0) load(next);

        // as columns (square 4 col + j, channels 8 q ... 8 q + 7)
        u32x4 xc[4][NT];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int k = 0; k < NT; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    xc[j][k][i] = __builtin_amdgcn_perm(rows[k][2 * i + 1][j >> 1], rows[k][2 * i][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);

        // and as rows (channel, squares by row of the crossing) for dW
        u32x4 xr[2][2][NT];
        if (WANT & kKernelGrad) {
#pragma unroll
            for (int i = 0; i < 4 * NT; ++i) *reinterpret_cast<u32x4*>(write_at + (i % NT) * kTerm + 16 * (i / NT) * kRow) = xc[i / NT][i % NT];
            lds_fence();
#pragma unroll
            for (int i = 0; i < 4 * NT; ++i) xr[i / NT >> 1][i / NT & 1][i % NT] = transposed(i % NT, i / NT & 1, i / NT >> 1);
            lds_fence();
        }

        // logits, in units of 2^-(scales)
        f32x16 v[kTiles];                        // [tile of filters][4 * square + row]
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            u32x4 a[NT];
#pragma unroll
            for (int k = 0; k < NT; ++k) a[k] = lds.logit[t][k][lane];
            f32x4 l[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
            products<T, NT, NT>(l, [&](int, int k) { return a[k]; }, [&](int j, int k) { return xc[j][k]; });
#pragma unroll
            for (int k = 0; k < 16; ++k) v[t][k] = l[k >> 2][k & 3];
        }
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
        const float l_target = at_target([&](float e) { return e; });

        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int k = 0; k < 16; k += 2) top = larger(top, larger(v[t][k], v[t][k + 1]));
        top = lanes_reduce<true>(top);
        // exp(l - top) = 2^(l unit - top unit); an error of the rounded second product is common to all of the board
        const float unit = fminf(fmaxf(w_back * x_back, 1e-36f), 1e38f);
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
        if (!WANT) continue;

        // the logits' gradients times z: exponentials, less z at the target.  The target's is the largest but for
        // rounding: z's own, up to 90 * 2^-24, can make the target's smaller than another by as much, which the least
        // scale covers.
        const float rz = __builtin_amdgcn_rcpf(z);
        const float d_target = at_target([&](float e) { return e - (lane == t_lane ? z : 0.0f); }) * rz;
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
            if (u == 0) load(next);              // the first two tiles' registers are free
            if (WANT & kKernelGrad) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    short* p = write_at + (i & 1) * kTerm + 16 * (i >> 1) * kRow;
                    if (tiles == 2) *reinterpret_cast<u32x4*>(p) = d[i >> 1][i & 1];
                    else *reinterpret_cast<u32x2*>(p - 4 * q) = u32x2{d[i >> 1][i & 1][0], d[i >> 1][i & 1][1]};
                }
                lds_fence();
            }
            if (WANT & kFeaturesGrad) {
                u32x4 wk[2][NT];
#pragma unroll
                for (int i = 0; i < 2 * NT; ++i) wk[i / NT][i % NT] = lds.back[u][i / NT][i % NT][lane];
                products<T, NT, 2>(g, [&](int i, int k) { return wk[i >> 2][k]; }, [&](int i, int k) { return d[i & 3][k]; });
            }
            if (WANT & kKernelGrad) {
                auto sums = [&](auto& s) {       // [2 * tile + half of channels]
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        u32x4 dk[2][2];
#pragma unroll
                        for (int i = 0; i < 2 * tiles; ++i)
                            dk[i >> 1][i & 1] = transposed(i & 1, h, i >> 1);
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
        if (WANT & kFeaturesGrad) {
            const float back = wb * w_back;
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const raw_t out = {(T)(g[4 * a][r] * back), (T)(g[4 * a + 1][r] * back), (T)(g[4 * a + 2][r] * back), (T)(g[4 * a + 3][r] * back)};
                    *reinterpret_cast<raw_t*>(dx + b * (kC * kS) + (16 * a + 4 * q + r) * kS + 4 * col) = out;
                }
        }
      }
    }

    if (WANT & kKernelGrad) {
        float* part = reinterpret_cast<float*>(mine);
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    // column c of a pair of tiles is filter 16 (c >> 2 & 1) + 4 (c >> 3) + (c & 3) of the pair's 32
                    const int c = 16 * (t & 1) + col, f = t == 4 ? 64 + col : 32 * (t >> 1) + 16 * (c >> 2 & 1) + 4 * (c >> 3) + (c & 3);
                    part[(16 * a + 4 * q + r) * (16 * kTiles) + f] = dw[a][t][r];
                }
        __syncthreads();
        const float* all = reinterpret_cast<const float*>(smem + sizeof(HeadLds<T>));
        for (int i = threadIdx.x; i < kXW; i += blockDim.x) {
            const int c = i / kF, f = i % kF;
            float a = 0.0f;
            for (int k = 0; k < waves; ++k) a += all[k * (kWaveLds / 4) + c * 80 + f];
            dw_part[(size_t)blockIdx.x * kXW + i] = a;
        }
    }
}

// ---- the boards' own moves -------------------------------------------------------------------------------------------
//
// One wave a board, one lane a move (64 at a time), the board's features and the kernel in LDS.  A list of 32 moves needs
// a hundredth of the vocabulary's products, so they are plain float32 sums; what bounds the kernel is reading the features and
// writing their gradient, and next to it LDS.  A lane holds a move's logit; then 32 lanes a move, two moves at a time,
// add the move's part to the kernel's gradient (kept in LDS over all the wave's boards) and to the features' gradient
// (which takes the features' place).  Two moves that would meet take turns, so the sums are the same
// every time.  (LDS's own float adds do the same in one instruction, but take 200 cycles each: 0.88 ms in place of
// 0.35 for 65 536 boards.)
//
// A wave's boards are neighbours: it finds where its lists begin by adding up the counts of all boards before it, a
// byte a board beside the 8 to 16 KB that each board costs, and needs no pass over them beforehand.

constexpr int kHeadRow = 36;                     // floats a filter of the kernel in LDS
constexpr int kXRow = 68;                        // floats a channel of the features, from square to square
constexpr int kGRow = 33;                        // floats a square of their gradient, from channel to channel
constexpr int kMoveHeadBytes = kF * kHeadRow * 4 + 16 * 8;
constexpr int kMoveWaveBytes = kC * kXRow * 4 + 64 * 8;
constexpr int kMoveGradBytes = kMoveWaveBytes + kF * kC * 4;
static_assert(kS * kGRow <= kC * kXRow, "the gradient takes the features' place");

struct __attribute__((packed)) Bytes16 { unsigned v[4]; };

__device__ __forceinline__ unsigned lanes_add(unsigned v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
template <typename T, int WANT>
__global__ __launch_bounds__(512) void k_policy_move_loss(const T* __restrict__ x, const T* __restrict__ w, size_t n,
                                                          const uint8_t* __restrict__ from, const uint8_t* __restrict__ filter,
                                                          const uint8_t* __restrict__ per, size_t n_moves,
                                                          const int64_t* __restrict__ targets, const float* __restrict__ weights,
                                                          unsigned weight_step, float* __restrict__ loss, T* __restrict__ dx,
                                                          float* __restrict__ dw_part, int* __restrict__ err) {
    typedef typename Raw<T>::type raw_t;
    extern __shared__ __align__(16) unsigned char smem[];
    float* head = reinterpret_cast<float*>(smem);
    uint64_t* red = reinterpret_cast<uint64_t*>(smem + kF * kHeadRow * 4);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
    const int col = lane & 15, q = lane >> 4, chan = lane & 31, half = lane >> 5;
    unsigned char* mine = smem + kMoveHeadBytes + wave * (WANT & kKernelGrad ? kMoveGradBytes : kMoveWaveBytes);
    float* xs = reinterpret_cast<float*>(mine);                                  // [32][68]
    u32x2* entry = reinterpret_cast<u32x2*>(mine + kC * kXRow * 4);              // [64] (square | filter << 8, gradient)
    float* dws = reinterpret_cast<float*>(mine + kMoveWaveBytes);                // [73][32], gradient calls only

    const size_t all = (size_t)gridDim.x * waves, me = (size_t)blockIdx.x * waves + wave;
    const size_t lo = n * me / all, hi = n * (me + 1) / all, group_lo = n * (me - wave) / all;

    for (int i = tid; i < kXW; i += blockDim.x) head[(i % kF) * kHeadRow + i / kF] = (float)w[i];
    if (WANT & kKernelGrad)
        for (int i = lane; i < kF * kC; i += 64) dws[i] = 0.0f;
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
    if (lane == 0) red[wave] = before;
    before = 0;
    for (size_t i = group_lo + lane; i < lo; i += 64) before += per[i];
    uint64_t start = lanes_add(before);
    __syncthreads();
    for (int i = 0; i < waves; ++i) start += red[i];

    raw_t raw[8];
    auto load = [&](size_t b) {
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = *reinterpret_cast<const raw_t*>(x + b * (kC * kS) + (4 * i + q) * kS + 4 * col);
    };
    if (lo < hi) load(lo);
    unsigned counts = 0;
    for (size_t b = lo; b < hi; ++b) {
        if (((b - lo) & 63) == 0) counts = b + lane < hi ? per[b + lane] : 0u;
        const unsigned listed = __builtin_amdgcn_readlane(counts, (int)((b - lo) & 63));
        const uint64_t first = min(start, (uint64_t)n_moves);
        const int cnt = (int)min((uint64_t)listed, n_moves - first);
        start += listed;
        const int64_t t64 = targets[b];
        const int target = __builtin_amdgcn_readfirstlane(t64 >= 0 && t64 < cnt ? (int)t64 : -1);

#pragma unroll
        for (int i = 0; i < 8; ++i)
            *reinterpret_cast<f32x4*>(xs + (4 * i + q) * kXRow + 4 * col) = f32x4{(float)raw[i][0], (float)raw[i][1], (float)raw[i][2], (float)raw[i][3]};
        if (b + 1 < hi) load(b + 1);
        lds_fence();

        float l[4];                              // [pass of 64 moves]
        unsigned place[4];
        float top = -INFINITY, l_target = 0.0f;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            l[p] = -INFINITY;
            place[p] = 0;
            if (64 * p >= cnt) continue;
            if (64 * p + lane < cnt) {
                unsigned s = from[first + 64 * p + lane], f = filter[first + 64 * p + lane];
                if (s >= kS || f >= kF) atomicOr(err, 8);
                s = min(s, kS - 1u);
                f = min(f, kF - 1u);
                place[p] = s | f << 8;
                float a = 0.0f;
#pragma unroll
                for (int c = 0; c < kC; c += 4) {
                    const f32x4 k = *reinterpret_cast<const f32x4*>(head + f * kHeadRow + c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) a = fmaf(k[i], xs[(c + i) * kXRow + s], a);
                }
                l[p] = a;
            }
            top = larger(top, l[p]);
            if (target >> 6 == p) l_target = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(l[p]), target & 63));
        }
        if (target < 0) {                        // no part in anything, whatever the features hold
            if (lane == 0) {
                if (t64 != -1) atomicOr(err, 8);
                if (loss) loss[b] = 0.0f;
            }
            if (WANT & kFeaturesGrad) {
                u32x4* out = reinterpret_cast<u32x4*>(dx + b * (kC * kS));
#pragma unroll
                for (int i = 0; i < (int)(kC * kS * sizeof(T) / 1024); ++i) out[i * 64 + lane] = u32x4{0, 0, 0, 0};
            }
            lds_fence();
            continue;
        }
        top = lanes_reduce<true>(top);
        float z = 0.0f;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            if (64 * p >= cnt) continue;
            l[p] = __builtin_amdgcn_exp2f((l[p] - top) * 1.44269504088896341f);
            z += l[p];
        }
        z = lanes_reduce<false>(z);
        if (loss && lane == 0) loss[b] = fmaf(__builtin_amdgcn_logf(z), 0.693147180559945309f, top - l_target);
        if (!WANT) {
            lds_fence();
            continue;
        }

        const float wb = weights[b * weight_step], rz = __builtin_amdgcn_rcpf(z);
        // One pass's moves, two at a time: move k by the lower lanes, move k + pairs by the upper ones.  to(place) is where
        // a lane adds to, of(place) what of times the logit's gradient it adds; meet(a, b): two moves add to the same.
        auto add_up = [&](int p, auto&& to, auto&& of, auto&& meet) {
            const int here = min(cnt - 64 * p, 64), pairs = (here + 1) >> 1;
            const float one = target == 64 * p + lane ? z : 0.0f;
            lds_fence();
            entry[lane] = u32x2{place[p], __float_as_uint((l[p] - one) * rz * wb)};
            lds_fence();
            const uint64_t turns = __ballot(lane + pairs < here && meet(entry[(lane + pairs) & 63][0], place[p]));
            u32x2 e = entry[half * pairs];
            float v = of(e[0]) * __uint_as_float(e[1]);
            for (int k = 0; k < pairs; ++k) {
                float* at = to(e[0]);
                const float was = *at;
                e = entry[min(k + 1 + half * pairs, 63)];
                const float next = of(e[0]) * __uint_as_float(e[1]);   // in flight while this one is added
                if (turns >> k & 1) {
                    if (half == 0) *at = was + v;
                    lds_fence();
                    if (half == 1) *at += v;
                } else if (k + half * pairs < here) {
                    *at = was + v;
                }
                lds_fence();
                v = next;
            }
        };
        if (WANT & kKernelGrad)
#pragma unroll
            for (int p = 0; p < 4; ++p)
                if (64 * p < cnt)
                    add_up(p, [&](unsigned m) { return dws + (m >> 8) * kC + chan; }, [&](unsigned m) { return xs[chan * kXRow + (m & 0xff)]; },
                           [](unsigned a, unsigned b) { return a >> 8 == b >> 8; });
        if (WANT & kFeaturesGrad) {
            lds_fence();
            float* g = xs;                       // [64][33]
            for (int i = lane; i < kS * kGRow; i += 64) g[i] = 0.0f;
#pragma unroll
            for (int p = 0; p < 4; ++p)
                if (64 * p < cnt)
                    add_up(p, [&](unsigned m) { return g + (m & 0xff) * kGRow + chan; }, [&](unsigned m) { return head[(m >> 8) * kHeadRow + chan]; },
                           [](unsigned a, unsigned b) { return (a & 0xff) == (b & 0xff); });
            lds_fence();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                raw_t out;
#pragma unroll
                for (int j = 0; j < 4; ++j) out[j] = (T)g[(4 * col + j) * kGRow + 4 * i + q];
                *reinterpret_cast<raw_t*>(dx + b * (kC * kS) + (4 * i + q) * kS + 4 * col) = out;
            }
        }
        lds_fence();
    }
    if (lo < hi && hi == n && lane == 0 && start != n_moves) atomicOr(err, 8);

    if (WANT & kKernelGrad) {
        __syncthreads();
        for (int i = tid; i < kXW; i += blockDim.x) {
            const int c = i / kF, f = i % kF;
            float a = 0.0f;
            for (int k = 0; k < waves; ++k)
                a += reinterpret_cast<const float*>(smem + kMoveHeadBytes + k * kMoveGradBytes + kMoveWaveBytes)[f * kC + c];
            dw_part[(size_t)blockIdx.x * kXW + i] = a;
        }
    }
}

// The partial kernel gradients of the workgroups, added up in fixed order: a workgroup 32 elements, eight threads each.
template <typename T>
__global__ __launch_bounds__(256) void k_sum_parts(const float* __restrict__ part, unsigned parts, T* __restrict__ dw) {
    __shared__ double sums[8][32];
    const int i = blockIdx.x * 32 + (threadIdx.x & 31), j = threadIdx.x >> 5;
    double a = 0.0;
#pragma unroll 8
    for (unsigned p = j; p < parts; p += 8) a += part[(size_t)p * kXW + i];
    sums[j][threadIdx.x & 31] = a;
    __syncthreads();
    if (j == 0) {
        for (int k = 1; k < 8; ++k) a += sums[k][threadIdx.x];
        dw[i] = (T)(float)a;
    }
}
static_assert(kXW % 32 == 0, "k_sum_parts needs no bounds check");

constexpr unsigned kGroups = 256;   // workgroups of a gradient call: one a compute unit, each with a part of the kernel's gradient

// Waves a workgroup: small calls are spread over the compute units.
unsigned waves_for(size_t n, unsigned most) {
    unsigned waves = 1;
    while (waves < most && (size_t)waves * kGroups < n) waves *= 2;
    return waves;
}

template <typename T, int WANT>
hipError_t launch(const PolicyLossArgs& a, hipStream_t s) {
    const T *x = static_cast<const T*>(a.features), *w = static_cast<const T*>(a.kernel);
    T* dx = static_cast<T*>(a.d_features);
    float* part = static_cast<float*>(a.workspace);
    const unsigned waves = waves_for(a.n, WANT ? 8 : 4), step = a.n_weights > 1 ? 1u : 0u;
    const unsigned grid = (unsigned)std::min<size_t>((a.n + waves - 1) / waves, WANT ? kGroups : 4 * kGroups);
    if (grid && a.per_board)
        hipLaunchKernelGGL((k_policy_move_loss<T, WANT>), dim3(grid), dim3(waves * 64),
                           kMoveHeadBytes + waves * (WANT & kKernelGrad ? kMoveGradBytes : kMoveWaveBytes), s, x, w, a.n, a.from,
                           a.filter, a.per_board, a.n_moves, a.targets, a.weights, step, a.loss, dx, part, a.err);
    else if (grid)
        hipLaunchKernelGGL((k_policy_loss<T, WANT>), dim3(grid), dim3(waves * 64),
                           sizeof(HeadLds<T>) + (WANT & kKernelGrad ? waves * kWaveLds : 0), s, x, w, a.n, a.targets, a.weights, step,
                           a.loss, dx, part, a.err);
    if (hipError_t e = hipGetLastError()) return e;
    if (WANT & kKernelGrad) hipLaunchKernelGGL(k_sum_parts<T>, dim3(kXW / 32), dim3(256), 0, s, part, grid, static_cast<T*>(a.d_kernel));
    return hipGetLastError();
}

template <typename T>
hipError_t launch(const PolicyLossArgs& a, hipStream_t s) {
    if (a.d_features) return a.d_kernel ? launch<T, kFeaturesGrad | kKernelGrad>(a, s) : launch<T, kFeaturesGrad>(a, s);
    return a.d_kernel ? launch<T, kKernelGrad>(a, s) : launch<T, 0>(a, s);
}

}  // namespace

size_t policy_loss_workspace(size_t n) { return std::min<size_t>(n, kGroups) * kXW * sizeof(float); }

hipError_t launch_policy_loss(const PolicyLossArgs& a, hipStream_t stream) {
    if (a.type == BF_TYPE_F32) return launch<float>(a, stream);
    if (a.type == BF_TYPE_BF16) return launch<__bf16>(a, stream);
    return launch<_Float16>(a, stream);
}

}  // namespace bf
