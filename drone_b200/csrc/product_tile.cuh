// C[M, N] = A[M, K] B[K, N] on the tensor cores: one block an SM walks tiles of 128 rows and BN columns, with two sets of accumulators in
// tensor memory, so that a tile's way to global memory and the next one's products overlap.
//
// Its warps: 4 to 16 take finished tiles out (bias, activation, residual), one issues the matrix instructions, one the asynchronous copies, and
// where floats have to be split on their way 8 or 16 more bring them.  Operands come in one of three ways:
//   kCopied    16-bit: tensor copies, tiles lie in shared memory as they do in global memory (along K or not).  Rows that are not on 16 bytes
//              (features of 602 or 47 values), which no tensor map takes, are copied to rows that are by pad_rows_kernel first
//   kImage     floats: A through registers, from any address; B from an image of it, split, that image_kernel has written, a copy a step
//   kThrough   floats: both through registers
//
// Floats are split into three bfloat16 of 8 bits each, x = h + m + l exactly (but for values below 2^-110), and six of the nine products are added:
// h h' in one accumulator, h m' + m h' + m m' + h l' + l h' in a second one that is 2^-7 of it, so that neither loses bits of the other.
// The rest is below 2^-22 of |x y|, and 2^-25 in the mean.  The accumulators cut off what they cannot hold, half a unit an addition in the mean and always
// towards 0: after every 256 of K they are added up in shared memory, rounding to nearest, and begin anew.  Products of 16 bits run through all of K, which is
// 32768 at most.  Where all terms have one sign that loses 2^-14.3 of a sum of 8192 (measured, in the mean) and 2^-12.3 of one of 32768, beside the half
// step of 2^-11 or 2^-8 that the result is rounded by.  A weight gradient, whose K are rows without end (2^-8.6 of 400,003), adds what it has up in its
// share after every 8192 of them: 2^-14.4; 400,003 x 2048 x 1280 with the gradient of the rows 4.55 ms, 4.40 without.  h is cut off, so that a finite x has
// a finite one.  Infinities and NaN have themselves for h (and NaN for m): where the first accumulator is not finite it is the result.
//
// All waits end after two seconds; a block whose wait did leaves NaN in its outputs.
//
// us: 232,965 x 602 x 128 floats with bias and ReLU 276 among other inputs, 252 on the same again (floor 128, of six bfloat16 products; 305 as two blocks an SM that bring,
// multiply and take out in turn; matrix instructions alone about 180: of 128 columns they read operands from shared memory at its rate); the weight gradient of the
// same 310, 349 with 8 warps that bring; 2.4 M x 256 x 256 bfloat16 with GELU, residual and the values before it 1074 (72 % of the copy
// rate; 2363 with 8 warps that take out, 1393 without the residual ahead and 8 bytes a lane).
#pragma once

#include "dense_types.cuh"

#include <cuda.h>

#include <algorithm>
#include <type_traits>

namespace drone {

// Where a product's tiles go: through the epilogue to Y (and pre), or as float shares of the sum.
template <typename T>
struct LinearOut {
    const float *bias;
    int activation;
    const T *residual;
    long long ldr;
    T *y;
    long long ldy;
    T *pre;
    long long ldp;
    float *shares;      // not NULL: [share][M][N]
    int at_once;        // columns of every operand that can be read and written at once: 16 bytes of them, 4, or 1
};

// An operand: values `ld` apart along one dimension and side by side along the other; read `bytes` at a time.
template <typename T>
struct Operand {
    const T *at;
    long long ld;
    int bytes;
};

enum Bring { kCopied, kImage, kThrough };

template <typename T> struct TileShape {
    static constexpr int PLANES = sizeof(T) == 4 ? 3 : 1;
    static constexpr int ROWS = 128, BN = sizeof(T) == 4 ? 128 : 256;
    static constexpr int KS = sizeof(T) == 4 ? 32 : 64;          // of K in a step
    static constexpr int STAGES = 3;                             // at most
    static constexpr int chunk(bool shares) { return sizeof(T) == 4 ? 256 / KS : shares ? 8192 / KS : 1 << 30; }      // steps until the accumulators are added up
    static constexpr int A_PLANE = ROWS * KS * 2, B_PLANE = BN * KS * 2, A_BYTES = PLANES * A_PLANE, B_BYTES = PLANES * B_PLANE, STAGE = A_BYTES + B_BYTES;
    static constexpr int SET = (sizeof(T) == 4 ? 2 : 1) * BN;    // columns of tensor memory of a set of accumulators, of which there are two
    // floats between the rows on their way out: of a whole tile whose sums are kept there, or of a warp's piece of 32 x 32
    static constexpr int PITCH = sizeof(T) == 4 ? BN + 4 : 36;
    static constexpr int shared(int stages, int out_warps) { return 1024 + stages * STAGE + (sizeof(T) == 4 ? ROWS : out_warps * 32) * PITCH * 4; }
};
// Warps that take tiles out, threads that bring operands.
template <Bring BRING> constexpr int kOutWarps = BRING == kCopied ? 16 : BRING == kImage ? 8 : 4;
template <Bring BRING> constexpr int kBringThreads = BRING == kCopied ? 0 : BRING == kImage ? 256 : 512;
template <Bring BRING> constexpr int kBringFrom = (kOutWarps<BRING> + 2) * 32;
template <Bring BRING> constexpr int kProductThreads = kBringFrom<BRING> + kBringThreads<BRING>;

__device__ __forceinline__ unsigned shared_address(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void barrier_init(unsigned bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count)); }
__device__ __forceinline__ void barrier_arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory"); }
// Waits for a phase of a barrier, two seconds at most: false if it did not end.  (The clock is looked at every 256 polls: a look takes longer than
// most waits.)
__device__ __forceinline__ bool barrier_wait(unsigned bar, unsigned parity) {
    unsigned long long began = 0;
    for (unsigned polls = 1;; ++polls) {
        unsigned done;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
        if ((polls & 255) == 0) {
            unsigned long long now;
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
            if (began == 0) began = now;
            else if (now - began > 2000000000ull) return false;
        }
    }
}

// Shared memory as the matrix instructions take it: 16 bytes hold 8 values along the dimension in which they lie side by side.
// ALONG_K: rows of KS values (64 or 128 bytes), 8 of them a swizzle pattern; else KS rows of 64 values for each 64 of the other dimension.
template <int KS, bool ALONG_K>
struct SharedLayout {
    static constexpr int UNITS_ALONG = KS / 8;
    __device__ static unsigned offset(int row, int unit) {      // ALONG_K: row of the tile, unit along K; else: row of K, unit along the tile
        if (ALONG_K) return KS == 64 ? row * 128 + ((unit ^ (row & 7)) << 4) : row * 64 + ((unit ^ ((row >> 1) & 3)) << 4);
        return (unit >> 3) * (KS * 128) + row * 128 + (((unit & 7) ^ (row & 7)) << 4);
    }
    // descriptor of the operand that starts at this address, for the 16 of K that start at k (start address, strides between
    // 64 values along the tile and between 8 rows, version, swizzle of 128 or 64 bytes)
    __device__ static unsigned long long descriptor(unsigned address, int k) {
        const unsigned at = address + (ALONG_K ? k * 2 : k * 128);
        const unsigned long long leading = ALONG_K ? 1 : (KS * 128) >> 4, stride = ALONG_K ? (KS * 16) >> 4 : 1024 >> 4, swizzle = ALONG_K && KS == 32 ? 4 : 2;
        return (unsigned long long)((at >> 4) & 0x3fff) | leading << 16 | stride << 32 | 1ull << 46 | swizzle << 61;
    }
};

// V values side by side, that can be read at once or (PAIR = false) one by one.
template <int V, bool PAIR>
__device__ __forceinline__ void load_whole(const float *p, float *v) {
    if constexpr (V == 4) {
        const float4 a = __ldg((const float4 *)p);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else if constexpr (PAIR) {
        const float2 a = __ldg((const float2 *)p);
        v[0] = a.x, v[1] = a.y;
    } else {
        v[0] = __ldg(p), v[1] = __ldg(p + 1);
    }
}
// V values side by side, of which `live` exist (the others are 0); `bytes` can be read at once.
template <int V>
__device__ __forceinline__ void load_values(const float *p, int live, int bytes, float *v) {
    if constexpr (V == 4) {
        float4 a = make_float4(0, 0, 0, 0);
        if (live >= 4) {
            a = __ldg((const float4 *)p);
        } else if (live > 0) {
            a.x = __ldg(p);
            if (live > 1) a.y = __ldg(p + 1);
            if (live > 2) a.z = __ldg(p + 2);
        }
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
        float2 a = make_float2(0, 0);
        if (live >= 2 && bytes >= 8) {
            a = __ldg((const float2 *)p);
        } else {
            if (live > 0) a.x = __ldg(p);
            if (live > 1) a.y = __ldg(p + 1);
        }
        v[0] = a.x, v[1] = a.y;
    }
}
template <int WORDS>
__device__ __forceinline__ void store_shared(unsigned at, const unsigned *v) {
    if constexpr (WORDS == 1) asm volatile("st.shared.b32 [%0], %1;" :: "r"(at), "r"(v[0]) : "memory");
    else if constexpr (WORDS == 2) asm volatile("st.shared.v2.b32 [%0], {%1, %2};" :: "r"(at), "r"(v[0]), "r"(v[1]) : "memory");
    else asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ unsigned bf16_pair(float low, float high) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(low, high);
    return reinterpret_cast<const unsigned &>(p);
}
__device__ __forceinline__ unsigned bf16_pair_cut(float low, float high) {      // towards 0
    unsigned pair;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(pair) : "f"(high), "f"(low));
    return pair;
}
// Pairs of floats in three pairs of bfloat16.
template <int V>
__device__ __forceinline__ void split_values(const float *v, unsigned (&planes)[3][V / 2]) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        unsigned a = __float_as_uint(v[2 * i]), b = __float_as_uint(v[2 * i + 1]);
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const unsigned pair = planes[q][i] = q == 0 ? bf16_pair_cut(__uint_as_float(a), __uint_as_float(b)) : bf16_pair(__uint_as_float(a), __uint_as_float(b));
            if (q == 2) break;
            // what is left of both, in one instruction (the products with -1 are exact)
            asm("{\n.reg .b64 x, y, m;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %3};\nmov.b64 m, 0xbf800000bf800000;\nfma.rn.f32x2 x, y, m, x;\nmov.b64 {%0, %1}, x;\n}"
                : "+r"(a), "+r"(b) : "r"(pair << 16), "r"(pair & 0xffff0000u));
        }
    }
}
template <int V>
__device__ __forceinline__ void store_values(unsigned at, unsigned plane_bytes, const float *v) {
    unsigned planes[3][V / 2];
    split_values<V>(v, planes);
#pragma unroll
    for (int q = 0; q < 3; ++q) store_shared<V / 2>(at + q * plane_bytes, planes[q]);
}

// What a thread brings of an operand's tile in each step.  Neighbouring threads have neighbouring values: 16 bytes each where rows allow it,
// else pairs (lanes with 32 bytes each of rows that are not on 16 bytes touch four times the lines with every load).
template <int THREADS, int R, bool ALONG_K>
struct Share {
    using S = TileShape<float>;
    using L = SharedLayout<S::KS, ALONG_K>;
    static constexpr int WIDTH = ALONG_K ? S::KS : R, VALUES = R * S::KS / THREADS;
    static constexpr unsigned PLANE = R * S::KS * 2;
    struct Values { float v[VALUES]; };
    Operand<float> from;
    template <int V> static constexpr int APART = THREADS / (WIDTH / V);      // rows between a thread's values
    int row, column;                  // of its first
    const float *at = nullptr;
    int limit = 0, k = 0;             // rows or columns of the tile that exist; of K until the share's end

    __device__ Share(const Operand<float> &o, int thread) : from(o) {
        const int v = o.bytes == 16 ? 4 : 2;
        row = thread / (WIDTH / v), column = thread % (WIDTH / v) * v;
    }
    __device__ void begin(long long start, int size, int k0, int k1) {
        at = ALONG_K ? from.at + (start + row) * from.ld + k0 + column : from.at + (long long)(k0 + row) * from.ld + start + column;
        limit = size, k = k1 - k0;
    }
    // WHOLE: the step lies inside the operand; its loads follow one another without a condition, so that all of them are in flight
    template <int V, bool WHOLE, bool PAIR = true>
    __device__ __forceinline__ void load_each(Values &to) {
        const float *p = at;
#pragma unroll
        for (int u = 0; u < VALUES / V; ++u, p += APART<V> * from.ld) {
            float *const v = to.v + u * V;
            if constexpr (WHOLE) {
                load_whole<V, PAIR>(p, v);
            } else {
                const int r = row + u * APART<V>;
                const bool in_row = ALONG_K ? r < limit : r < k;
                load_values<V>(p, in_row ? (ALONG_K ? k : limit) - column : 0, from.bytes, v);
            }
        }
    }
    __device__ __forceinline__ void load(Values &to) {
        const bool whole = limit >= R && k >= S::KS;
        if (from.bytes == 16) {
            if (whole) load_each<4, true>(to);
            else load_each<4, false>(to);
        } else {
            if (whole && from.bytes >= 8) load_each<2, true>(to);
            else if (whole) load_each<2, true, false>(to);
            else load_each<2, false>(to);
        }
        k -= S::KS;
        at += ALONG_K ? S::KS : S::KS * from.ld;
    }
    template <int V>
    __device__ void store_each(unsigned to, const Values &v) const {
#pragma unroll
        for (int u = 0; u < VALUES / V; ++u) {
            // rows 8 apart, and with them all values of a thread but the first, have the same place in the swizzle pattern
            constexpr bool SAME = APART<V> % 8 == 0;
            const unsigned at = SAME ? L::offset(row, column >> 3) + u * (L::offset(APART<V>, 0) - L::offset(0, 0)) : L::offset(row + u * APART<V>, column >> 3);
            store_values<V>(to + at + (column & 7) * 2, PLANE, v.v + u * V);
        }
    }
    __device__ void store(unsigned to, const Values &v) const {
        if (from.bytes == 16) store_each<4>(to, v);
        else store_each<2>(to, v);
    }
};

__device__ __forceinline__ void mma(unsigned accumulator, unsigned long long a, unsigned long long b, unsigned instruction, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(accumulator), "l"(a), "l"(b),
                 "r"(instruction), "r"((unsigned)add) : "memory");
}
__device__ __forceinline__ void mma_commit(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void load_accumulators(unsigned at, float *v) {
    unsigned r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
                 "%23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
                   "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void load_accumulators16(unsigned at, float *v) {
    unsigned r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// One lane of a warp whose lanes go the same way.  (A branch of one thread by its number would leave the compiler without uniform registers, in
// which these instructions take their operands: a matrix instruction then took about as long to issue as to run.)
__device__ __forceinline__ bool elected() {
    unsigned mine;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(mine));
    return mine != 0;
}
__device__ __forceinline__ void expect_bytes(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_tile(unsigned to, const CUtensorMap *map, int x, int y, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(to), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void copy_bytes(unsigned to, const void *from, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" :: "r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}

// A block's stages in turn.  The barriers' phases: `filled` ends with the stage's filling at hand, `emptied` with the use before it (there is none
// before the first: that phase counts as over).
struct Ring {
    int stages, stage = 0;
    unsigned filled = 0;
    __device__ explicit Ring(int n) : stages(n) {}
    __device__ unsigned emptied() const { return filled ^ 1; }
    __device__ void next() {
        if (++stage == stages) stage = 0, filled ^= 1;
    }
};

// The tiles of a block, in turn: columns first, so that blocks at work at the same time share their rows, then rows, then shares of K.
struct TileWalk {
    int tiles_n, tiles_m, M, N, K, share, bn, ks;
    long long tile, count;
    long long m0;
    int n0, k0, k1, steps, index;      // index: of the share
    __device__ TileWalk(int M_, int N_, int K_, int share_, int shares, int bn_, int ks_)
        : tiles_n((N_ + bn_ - 1) / bn_), tiles_m((M_ + 127) / 128), M(M_), N(N_), K(K_), share(share_), bn(bn_), ks(ks_), tile(blockIdx.x) {
        count = (long long)tiles_n * tiles_m * shares;
        place();
    }
    __device__ bool valid() const { return tile < count; }
    __device__ void next() {
        tile += gridDim.x;
        place();
    }
    __device__ void place() {
        if (tile >= count) return;
        const long long a_share = (long long)tiles_n * tiles_m, in_share = tile % a_share;
        index = (int)(tile / a_share);
        m0 = in_share / tiles_n * 128;
        n0 = (int)(in_share % tiles_n) * bn;
        k0 = index * share;
        k1 = min(K, k0 + share);
        steps = (k1 - k0 + ks - 1) / ks;
    }
    __device__ int rows() const { return (int)min(128LL, M - m0); }
    __device__ int width() const { return min(bn, N - n0); }
    __device__ int columns() const { return (width() + 15) / 16 * 16; }      // that the instructions compute
};

template <typename T, Bring BRING, bool A_ALONG_K, bool B_ALONG_K>
struct ProductArgs {
    Operand<T> A, B;
    CUtensorMap map_a, map_b;      // kCopied
    const char *image;             // kImage
    int M, N, K, share, shares, stages;
    LinearOut<T> out;
};

// The residual of 32 x 32 values, W of a row a lane: of 16-bit ones read before the accumulators are waited for, of floats (32 registers) when it
// is added.
template <typename T>
struct Residual {
    static constexpr bool AHEAD = sizeof(T) == 2;
    unsigned v[AHEAD ? 16 : 1];      // 0 where there is no residual
    template <int W>
    __device__ __forceinline__ void read_each(const LinearOut<T> &out, long long row0, int rows, int col0, int width) {
        constexpr int LANES = 32 / W, STEP = 32 / LANES;      // of a row; rows at once
        const int lane = threadIdx.x & 31, c = lane % LANES * W;
        if (c >= width) return;
        const T *from = out.residual + (row0 + lane / LANES) * out.ldr + col0 + c;
#pragma unroll
        for (int i = 0; i < LANES; ++i)
            if (lane / LANES + i * STEP < rows) {
                if constexpr (W == 8) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(from + (long long)(i * STEP) * out.ldr);
                    v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2 *>(from + (long long)(i * STEP) * out.ldr);
                    v[2 * i] = x.x, v[2 * i + 1] = x.y;
                }
            }
    }
    __device__ __forceinline__ void read(const LinearOut<T> &out, long long row0, int rows, int col0, int width) {
        if constexpr (AHEAD) {
            if (!out.residual) return;
            if (out.at_once == 8) read_each<8>(out, row0, rows, col0, width);
            else if (out.at_once == 4) read_each<4>(out, row0, rows, col0, width);
        }
    }
    template <int W>
    __device__ __forceinline__ Values<T, W> at(const LinearOut<T> &out, int i, long long row, int column) const {
        Values<T, W> x = {};
        if constexpr (AHEAD) memcpy(&x, &v[i * W / 2], W * 2);
        else if (out.residual) x = *reinterpret_cast<const Values<T, W> *>(out.residual + row * out.ldr + column);
        return x;
    }
};

// 32 x 32 values of a finished tile, of which the warp has written a row a lane to shared memory, to the outputs with neighbouring columns in
// neighbouring lanes.
template <typename T, int PITCH, int ACTIVATION, int W>
__device__ __forceinline__ void put_vectors(const LinearOut<T> &out, const float *piece, const Residual<T> &residual, long long row0, int rows, int col0, int width) {
    constexpr int LANES = 32 / W, STEP = 32 / LANES;
    const int lane = threadIdx.x & 31, c = lane % LANES * W;
    if (c >= width) return;
    float b[W];
#pragma unroll
    for (int i = 0; i < W; ++i) b[i] = 0;
    if (out.bias) {
#pragma unroll
        for (int i = 0; i < W; i += 4) *reinterpret_cast<float4 *>(b + i) = __ldg((const float4 *)(out.bias + col0 + c + i));
    }
#pragma unroll(Residual<T>::AHEAD ? LANES : 2)
    for (int step = 0; step < LANES; ++step) {
        const int r = lane / LANES + step * STEP;
        if (r >= rows) break;
        const long long row = row0 + r;
        float z[W], w[W], added[W];
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const float4 acc = *reinterpret_cast<const float4 *>(piece + r * PITCH + c + i);
            z[i] = acc.x + b[i], z[i + 1] = acc.y + b[i + 1], z[i + 2] = acc.z + b[i + 2], z[i + 3] = acc.w + b[i + 3];
        }
        residual.template at<W>(out, step, row, col0 + c).get(added);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            w[i] = activate<T, ACTIVATION>(z[i], added[i]);      // 0 where there is no residual
        }
        Values<T, W> y;
        if (out.pre) {
            y.set(z);
            *reinterpret_cast<Values<T, W> *>(out.pre + row * out.ldp + col0 + c) = y;
        }
        y.set(w);
        *reinterpret_cast<Values<T, W> *>(out.y + row * out.ldy + col0 + c) = y;
    }
}
// The same a value a lane: a row at a time with a lane for each column, or, of at most 16 columns of 16 bits, rows one after the other over the lanes (606,060 x 19 x 47
// half, GELU, residual 203 us, 253 without; floats gain as much, 333,333 x 108 x 12 100 and 134, but where the kernel holds that code too wide products are slower, 232,965 x 128 x
// 602 270 and 257).  What four values of a lane add is on its way at once.
// Before, and before the warps with the same rows shared a narrow tile: 606,060 x 19 x 47 half 588, floats 575 and now 213; 200,000 x 128 x 301 bfloat16 179 and now 111.
template <typename T, int PITCH, int ACTIVATION, bool SHORT>
__device__ __forceinline__ void put_values(const LinearOut<T> &out, const float *piece, long long row0, int rows, int col0, int width) {
    const int lane = threadIdx.x & 31;
    int r = SHORT ? lane / width : 0, c = SHORT ? lane % width : lane;
    if (c >= width) return;
    const int down = SHORT ? 32 / width : 1, along = SHORT ? 32 % width : 0;
    float b = !SHORT && out.bias ? __ldg(out.bias + col0 + c) : 0.f;
    auto put = [&](int r, int c, float added) {
        const long long row = row0 + r;
        const float z = piece[r * PITCH + c] + (SHORT && out.bias ? __ldg(out.bias + col0 + c) : b);
        const float w = activate<T, ACTIVATION>(z, added);
        if (out.pre) out.pre[row * out.ldp + col0 + c] = from_float<T>(z);
        out.y[row * out.ldy + col0 + c] = from_float<T>(w);
    };
    auto next = [&](int &r, int &c) {
        r += down, c += along;
        if (SHORT && c >= width) c -= width, ++r;
    };
    if (!out.residual) {
#pragma unroll 4
        for (; r < rows; next(r, c)) put(r, c, -0.f);      // no addition
        return;
    }
    constexpr int AT_ONCE = 4;
#pragma unroll 1
    while (r < rows) {
        float added[AT_ONCE];
        int ahead = r, column = c;
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (ahead < rows) added[u] = to_float(out.residual[(row0 + ahead) * out.ldr + col0 + column]);
            next(ahead, column);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (r >= rows) break;
            put(r, c, added[u]);
            next(r, c);
        }
    }
}
template <typename T, int PITCH, int ACTIVATION>
__device__ __forceinline__ void put_piece(const LinearOut<T> &out, const float *piece, const Residual<T> &residual, long long row0, int rows, int col0, int width) {
    if (sizeof(T) == 2 && out.at_once == 8) {
        if constexpr (sizeof(T) == 2) put_vectors<T, PITCH, ACTIVATION, 8>(out, piece, residual, row0, rows, col0, width);
    } else if (out.at_once == 4) {
        put_vectors<T, PITCH, ACTIVATION, 4>(out, piece, residual, row0, rows, col0, width);
    } else {
        bool is_short = false;
        if constexpr (sizeof(T) == 2) {
            is_short = width <= 16;
            if (is_short) put_values<T, PITCH, ACTIVATION, true>(out, piece, row0, rows, col0, width);
        }
        if (!is_short) put_values<T, PITCH, ACTIVATION, false>(out, piece, row0, rows, col0, width);
    }
}

template <typename T, Bring BRING, bool A_ALONG_K, bool B_ALONG_K>
__global__ void __launch_bounds__(kProductThreads<BRING>, 1)
product_tile_kernel(const __grid_constant__ ProductArgs<T, BRING, A_ALONG_K, B_ALONG_K> p) {
    using S = TileShape<T>;
    constexpr int OUT = kOutWarps<BRING>;
    constexpr bool SHARES = !A_ALONG_K;      // a weight gradient, in shares of K; else everything goes through the epilogue
    constexpr int CHUNK = S::chunk(SHARES);
    constexpr bool B_SHARED_ALONG_K = BRING == kImage || B_ALONG_K;
    using LA = SharedLayout<S::KS, A_ALONG_K>;
    using LB = SharedLayout<S::KS, B_SHARED_ALONG_K>;
    extern __shared__ char bytes[];
    __shared__ __align__(8) unsigned long long bars[2 * S::STAGES + 5];
    __shared__ unsigned tensor_memory;
    char *const shared = bytes + ((1024 - (shared_address(bytes) & 1023)) & 1023);
    const unsigned stages = shared_address(shared), full = shared_address(bars), empty = full + 8 * S::STAGES, done = full + 16 * S::STAGES, taken = done + 16,
                   last = taken + 16;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);      // the same in all lanes, for the compiler too

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            barrier_init(full + 8 * s, kBringThreads<BRING> / 32 + (BRING == kThrough ? 0 : 1));
            barrier_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            barrier_init(done + 8 * b, 1);
            barrier_init(taken + 8 * b, OUT);
        }
        barrier_init(last, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == OUT) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(shared_address(&tensor_memory)), "n"(2 * S::SET) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned accumulators = tensor_memory;
    TileWalk walk(p.M, p.N, p.K, p.share, p.shares, S::BN, S::KS);

    if (warp < OUT) {
        // Takes tiles out: a quarter of the rows (the lanes of tensor memory that the warp can read) and some of the columns.
        // Of a tile of few columns each of the warps that read the same rows has some.
        constexpr int GROUPS = OUT / 4, COLUMNS = S::BN / GROUPS;
        const int lane_row = (warp & 3) * 32, group = warp >> 2;
        const auto columns_each = [](const TileWalk &of) { return (of.columns() / 16 + GROUPS - 1) / GROUPS * 16; };
        float *const piece = reinterpret_cast<float *>(shared + p.stages * S::STAGE) + (S::PLANES > 1 ? lane_row * S::PITCH + group * COLUMNS : warp * 32 * S::PITCH);
        float *const row = piece + (threadIdx.x & 31) * S::PITCH;      // this lane's
        bool ended = true;      // no wait was given up
        unsigned chunk = 0;     // of the block, over all tiles
        auto take_out = [&](auto act) {
            [[maybe_unused]] constexpr int ACTIVATION = decltype(act)::value;
            // The residual of the tile after the one at work, on its way to L2.
            auto prefetch = [&](const TileWalk &of) {
                const int r = threadIdx.x & 31;
                if (!p.out.residual || !of.valid() || lane_row + r >= of.rows()) return;
                const int each = columns_each(of), first = group * each;
                const T *at = p.out.residual + (of.m0 + lane_row + r) * p.out.ldr + of.n0 + first;
                for (int c = 0; c < min(each, of.width() - first); c += 128 / (int)sizeof(T)) asm volatile("prefetch.global.L2 [%0];" :: "l"(at + c));
            };
            TileWalk upcoming = walk;
            prefetch(upcoming);
            for (; walk.valid(); walk.next()) {
                const int each = columns_each(walk), first = group * each;
                const int rows = min(32, walk.rows() - lane_row), width = min(each, walk.width() - first);
                upcoming.next();
                prefetch(upcoming);
                const long long row0 = walk.m0 + lane_row;
                const int col0 = walk.n0 + first;
                [[maybe_unused]] Residual<T> residual = {};
                auto put = [&](const float *from, int c, [[maybe_unused]] bool more) {      // 32 columns from c on; more: to what the share has already
                    if (rows <= 0 || width - c <= 0) return;
                    if constexpr (SHARES) {
                        LinearOut<float> to = {};
                        to.y = p.out.shares + (long long)walk.index * p.M * p.N;
                        to.ldy = to.ldr = p.N;
                        if (more) to.residual = to.y;      // what the same thread has written
                        to.at_once = p.N % 4 == 0 ? 4 : 1;
                        put_piece<float, S::PITCH, DRONE_ACT_NONE>(to, from, Residual<float>(), row0, rows, col0 + c, min(32, width - c));
                    } else {
                        put_piece<T, S::PITCH, ACTIVATION>(p.out, from, residual, row0, rows, col0 + c, min(32, width - c));
                    }
                };
                if constexpr (S::PLANES > 1) {
                    for (int s = 0; s < walk.steps; s += CHUNK, ++chunk) {
                        const unsigned set = chunk & 1, at = accumulators + ((unsigned)lane_row << 16) + set * S::SET + first;
                        ended = ended && barrier_wait(done + 8 * set, (chunk >> 1) & 1);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                        for (int c = 0; c < width; c += 16) {
                            float a[16], b[16];
                            load_accumulators16(at + c, a);
                            load_accumulators16(at + S::BN + c, b);
#pragma unroll
                            for (int i = 0; i < 16; ++i) a[i] += fabsf(a[i]) < INFINITY ? b[i] : 0.f;
#pragma unroll
                            for (int i = 0; i < 16; i += 4) {
                                float4 *const to = reinterpret_cast<float4 *>(row + c + i);
                                float4 v = make_float4(a[i], a[i + 1], a[i + 2], a[i + 3]);
                                if (s > 0) {
                                    const float4 before = *to;
                                    v = make_float4(before.x + v.x, before.y + v.y, before.z + v.z, before.w + v.w);
                                }
                                if (!ended) v = make_float4(NAN, NAN, NAN, NAN);      // a wait was given up: nothing plausible comes out
                                *to = v;
                            }
                        }
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if ((threadIdx.x & 31) == 0) barrier_arrive(taken + 8 * set);
                    }
#pragma unroll 1
                    for (int c = 0; c < width; c += 32) put(piece + c, c, false);
                    __syncwarp();      // the tile has been read
                } else {
                    for (int s = 0; s < walk.steps; s += CHUNK, ++chunk) {
                        const unsigned set = chunk & 1, at = accumulators + ((unsigned)lane_row << 16) + set * S::SET + first;
                        ended = ended && barrier_wait(done + 8 * set, (chunk >> 1) & 1);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                        for (int c = 0; c < width; c += 32) {
                            if (!SHARES) residual.read(p.out, row0, rows, col0 + c, width - c);
                            float v[32];
                            load_accumulators(at + c, v);
                            __syncwarp();      // the piece before has been read
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                float4 w = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                                if (!ended) w = make_float4(NAN, NAN, NAN, NAN);
                                *reinterpret_cast<float4 *>(row + i) = w;
                            }
                            __syncwarp();
                            put(piece, c, s > 0);
                        }
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if ((threadIdx.x & 31) == 0) barrier_arrive(taken + 8 * set);
                    }
                }
            }
        };
        if constexpr (SHARES) take_out(std::integral_constant<int, DRONE_ACT_NONE>());
        else with_activation(p.out.activation, take_out);
    } else if (warp == OUT) {
        // Issues the matrix instructions.
        constexpr unsigned TYPE = std::is_same_v<T, __half> ? 0 : 1;
        bool ended = true;
        Ring ring(p.stages);
        unsigned chunk = 0;      // of the block, over all tiles
        for (; walk.valid() && ended; walk.next()) {
            // float accumulators, both operands of this type, lying along K (0) or not (1), columns / 8, rows / 16
            const unsigned instruction = 1u << 4 | TYPE << 7 | TYPE << 10 | (A_ALONG_K ? 0u : 1u) << 15 | (B_SHARED_ALONG_K ? 0u : 1u) << 16 |
                                         (unsigned)(walk.columns() / 8) << 17 | (unsigned)(S::ROWS / 16) << 24;
            // Where the tile is full the parts h' and m' of B are one operand of twice the columns, as are the accumulators: A is read once for both.
            const unsigned both = walk.columns() == S::BN ? instruction + ((unsigned)(S::BN / 8) << 17) : 0;
            for (int s = 0; s < walk.steps && ended; ++s, ring.next()) {
                const bool begins = s % CHUNK == 0;
                const unsigned set = chunk & 1, to = accumulators + set * S::SET;
                if (begins && chunk >= 2) ended = barrier_wait(taken + 8 * set, ((chunk >> 1) - 1) & 1);
                const int stage = ring.stage;
                ended = ended && barrier_wait(full + 8 * stage, ring.filled);
                if (!ended) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned a = stages + stage * S::STAGE, b = a + S::A_BYTES;
                if (elected()) {
#pragma unroll
                    for (int k = 0; k < S::KS; k += 16) {
                        const bool add = !begins || k > 0;
                        if (S::PLANES == 1) {
                            mma(to, LA::descriptor(a, k), LB::descriptor(b, k), instruction, add);
                        } else {
                            const unsigned long long ah = LA::descriptor(a, k), am = LA::descriptor(a + S::A_PLANE, k), al = LA::descriptor(a + 2 * S::A_PLANE, k);
                            const unsigned long long bh = LB::descriptor(b, k), bm = LB::descriptor(b + S::B_PLANE, k), bl = LB::descriptor(b + 2 * S::B_PLANE, k);
                            if (both) {      // h h' and h m' at once
                                mma(to, ah, bh, both, add);
                            } else {
                                mma(to, ah, bh, instruction, add);
                                mma(to + S::BN, ah, bm, instruction, add);
                            }
                            mma(to + S::BN, am, bh, instruction, true);
                            mma(to + S::BN, am, bm, instruction, true);
                            mma(to + S::BN, ah, bl, instruction, true);
                            mma(to + S::BN, al, bh, instruction, true);
                        }
                    }
                    mma_commit(empty + 8 * stage);
                    if (s + 1 == walk.steps || (s + 1) % CHUNK == 0) mma_commit(done + 8 * set);
                }
                __syncwarp();
                if (s + 1 == walk.steps || (s + 1) % CHUNK == 0) ++chunk;
            }
        }
        if (elected()) mma_commit(last);
    } else if (warp == OUT + 1) {
        // Issues the copies.
        bool ended = true;
        Ring ring(p.stages);
        int used = 0;      // stages
        if (BRING != kThrough)
            for (; walk.valid() && ended; walk.next()) {
                const int pieces = (walk.columns() + 63) / 64;      // of 64 columns, of B along N
                const unsigned a_bytes = BRING == kCopied ? S::A_BYTES : 0, b_bytes = BRING == kCopied && !B_ALONG_K ? pieces * (S::KS * 128) : S::B_BYTES;
                for (int s = 0; s < walk.steps; ++s, ring.next()) {
                    const int stage = ring.stage, k = walk.k0 + s * S::KS;
                    ended = barrier_wait(empty + 8 * stage, ring.emptied());
                    if (!ended) break;
                    used = max(used, stage + 1);
                    const unsigned bar = full + 8 * stage, a = stages + stage * S::STAGE, b = a + S::A_BYTES;
                    if (elected()) {
                        expect_bytes(bar, a_bytes + b_bytes);
                        if constexpr (BRING == kCopied) {
                            if (A_ALONG_K) {
                                copy_tile(a, &p.map_a, k, (int)walk.m0, bar);
                            } else {
                                for (int i = 0; i < S::ROWS / 64; ++i) copy_tile(a + i * (S::KS * 128), &p.map_a, (int)walk.m0 + i * 64, k, bar);
                            }
                            if (B_ALONG_K) {
                                copy_tile(b, &p.map_b, k, walk.n0, bar);
                            } else {
                                for (int i = 0; i < pieces; ++i) copy_tile(b + i * (S::KS * 128), &p.map_b, walk.n0 + i * 64, k, bar);
                            }
                        } else {
                            copy_bytes(b, p.image + ((long long)(walk.n0 / S::BN) * walk.steps + s) * S::B_BYTES, S::B_BYTES, bar);
                        }
                    }
                    __syncwarp();
                }
            }
        if (!ended)      // copies in flight land before the block goes
            for (int stage = 0; stage < used; ++stage) barrier_wait(full + 8 * stage, stage < ring.stage ? ring.filled : ring.emptied());
    } else if constexpr (BRING != kCopied) {
        // Bring what goes through registers, DEPTH steps ahead.
        constexpr int DEPTH = BRING == kImage ? 3 : 2;      // by the registers that a step takes: 16 or 32
        const int thread = threadIdx.x - kBringFrom<BRING>;
        Share<kBringThreads<BRING>, S::ROWS, A_ALONG_K> a(p.A, thread);
        Share<kBringThreads<BRING>, S::BN, B_ALONG_K> b(p.B, thread);
        typename decltype(a)::Values va[DEPTH];
        typename decltype(b)::Values vb[BRING == kThrough ? DEPTH : 1];
        int s = 0;
        unsigned asked = 0, step = 0;
        Ring ring(p.stages);
        auto begin = [&] {
            if (!walk.valid()) return;
            a.begin(walk.m0, walk.rows(), walk.k0, walk.k1);
            if (BRING == kThrough) b.begin(walk.n0, walk.width(), walk.k0, walk.k1);
        };
        auto load = [&](auto d) {
            constexpr int D = decltype(d)::value;
            if (!walk.valid()) return;
            a.load(va[D]);
            if constexpr (BRING == kThrough) b.load(vb[D]);
            ++asked;
            if (++s == walk.steps) {
                s = 0;
                walk.next();
                begin();
            }
        };
        bool ended = true;
        auto store = [&](auto d) {
            constexpr int D = decltype(d)::value;
            if (step == asked || !ended) return false;
            const int stage = ring.stage;
            ended = barrier_wait(empty + 8 * stage, ring.emptied());
            if (!ended) return false;
            const unsigned to = stages + stage * S::STAGE;
            a.store(to, va[D]);
            if constexpr (BRING == kThrough) b.store(to + S::A_BYTES, vb[D]);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if ((threadIdx.x & 31) == 0) barrier_arrive(full + 8 * stage);      // 256 arrivals at one barrier would queue
            ++step;
            ring.next();
            load(d);
            return true;
        };
        begin();
        load(std::integral_constant<int, 0>());
        if constexpr (DEPTH == 3) {
            load(std::integral_constant<int, 1>());
            load(std::integral_constant<int, 2>());
            while (store(std::integral_constant<int, 0>()) && store(std::integral_constant<int, 1>()) && store(std::integral_constant<int, 2>())) {}
        } else {
            load(std::integral_constant<int, 1>());
            while (store(std::integral_constant<int, 0>()) && store(std::integral_constant<int, 1>())) {}
        }
    }
    __syncwarp();
    barrier_wait(last, 0);      // no matrix instruction is in flight
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == OUT) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(accumulators), "n"(2 * S::SET));
    }
}

// The image of B that kImage copies: for every tile of columns and step of K its values as they lie in shared memory (along K, split).
template <bool B_ALONG_K>
__global__ void __launch_bounds__(256) image_kernel(Operand<float> B, int N, int K, char *image) {
    using S = TileShape<float>;
    using L = SharedLayout<S::KS, true>;
    const int steps = (K + S::KS - 1) / S::KS, n0 = (int)blockIdx.x / steps * S::BN, k0 = (int)blockIdx.x % steps * S::KS;
    char *const to = image + (long long)blockIdx.x * S::B_BYTES;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < S::BN * S::KS / 8; i += gridDim.y * 256) {
        const int row = B_ALONG_K ? i / (S::KS / 8) : i % S::BN, unit = B_ALONG_K ? i % (S::KS / 8) : i / S::BN, n = n0 + row, k = k0 + unit * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = n < N && k + e < K ? B.at[B_ALONG_K ? (long long)n * B.ld + k + e : (long long)(k + e) * B.ld + n] : 0.f;
        unsigned planes[3][4];
        split_values<8>(v, planes);
#pragma unroll
        for (int q = 0; q < S::PLANES; ++q) *reinterpret_cast<uint4 *>(to + q * S::B_PLANE + L::offset(row, unit)) = make_uint4(planes[q][0], planes[q][1], planes[q][2], planes[q][3]);
    }
}

// How many bytes of an operand's rows can be read at once.
template <typename T>
Operand<T> operand(const void *p, long long ld) {
    const unsigned long long bits = reinterpret_cast<uintptr_t>(p) | (unsigned long long)ld * sizeof(T) | 16;
    return {(const T *)p, ld, (int)(bits & (~bits + 1))};
}

// A tensor map of 16-bit values: boxes of 64 values (128 bytes, in the order of the 128-byte swizzle) of `box` rows.
int tile_map(CUtensorMap *map, bool bf16, const void *p, long long width, long long rows, long long ld, int box);

template <typename T, Bring BRING, bool A_ALONG_K, bool B_ALONG_K>
int launch_product_tiles(const Operand<T> &A, const Operand<T> &B, int M, int N, int K, int share, int shares, void *image, const LinearOut<T> &out, int sms,
                         cudaStream_t st) {
    using S = TileShape<T>;
    ProductArgs<T, BRING, A_ALONG_K, B_ALONG_K> p = {};
    p.A = A, p.B = B, p.image = (const char *)image, p.M = M, p.N = N, p.K = K, p.share = share, p.shares = shares, p.out = out;
    if constexpr (BRING == kCopied) {
        constexpr bool bf16 = std::is_same_v<T, __nv_bfloat16>;
        int rc = A_ALONG_K ? tile_map(&p.map_a, bf16, A.at, K, M, A.ld, S::ROWS) : tile_map(&p.map_a, bf16, A.at, M, K, A.ld, S::KS);
        if (!rc) rc = B_ALONG_K ? tile_map(&p.map_b, bf16, B.at, K, N, B.ld, S::BN) : tile_map(&p.map_b, bf16, B.at, N, K, B.ld, S::KS);
        if (rc) return rc;
    } else if constexpr (BRING == kImage) {
        const int blocks = ceil_div(N, S::BN) * ceil_div(K, S::KS);
        image_kernel<B_ALONG_K><<<dim3(blocks, S::BN * S::KS / 8 / 256), 256, 0, st>>>(B, N, K, (char *)image);
        DRONE_LAUNCH_CHECK("image_kernel");
    }
    // Rows that do not start on 16 bytes share lines between neighbouring steps: what two stages leave of an SM's memory is L1 that keeps them.
    // us with two and three, floats with bias and ReLU, calls one after another: 249,169 x 602 x 16 / 128 / 256 204 and 263 / 292 and 320 / 540 and 572; 600,000 x 154 x 16 /
    // 128 144 and 180 / 217 and 240; 600,000 x 115 x 64 151 and 174; 149,850 x 1001 x 64 235 and 274; 600,000 x 47 x 128 147 and 150, but of two steps, 600,000 x
    // 33 x 64, 105 and 98.  On 16 bytes 232,965 x 128 x 602 296 and 260.
    p.stages = BRING == kImage && A.bytes < 16 ? 2 : S::STAGES;
    const int bytes = S::shared(p.stages, kOutWarps<BRING>);
    auto *const kernel = product_tile_kernel<T, BRING, A_ALONG_K, B_ALONG_K>;
    // once a device: the call costs more than the launch's other preparations together
    static std::atomic<unsigned long long> devices{0};
    int device = 0;
    DRONE_CUDA(cudaGetDevice(&device));
    if (device > 63 || !(devices.load(std::memory_order_relaxed) >> device & 1)) {
        DRONE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::shared(S::STAGES, kOutWarps<BRING>)));
        if (device <= 63) devices.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    const long long tiles = (long long)ceil_div(M, S::ROWS) * ceil_div(N, S::BN) * shares;
    kernel<<<(unsigned)std::min<long long>(tiles, sms), kProductThreads<BRING>, bytes, st>>>(p);
    DRONE_LAUNCH_CHECK("product_tile_kernel");
    return DRONE_OK;
}

}  // namespace drone
