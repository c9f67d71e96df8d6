// C[M, N] = A[M, K] B[K, N] on the tensor cores: a block has a tile of 128 rows and BN columns, its accumulators in tensor memory.
//
// Eight warps bring the operands: they read a step of K from global memory into registers, whatever the rows' alignment (features of
// 602 or 47 values start anywhere, which no tensor map takes), and store it in the swizzled order that the matrix instructions read; one
// thread issues these.  The values of A and B lie along K or along the other dimension in shared memory as they do in global memory.
//
// Floats are split into three bfloat16 of 8 bits each, x = h + m + l exactly (but for values below 2^-110), and six of the nine products are added:
// h h' in one accumulator, h m' + m h' + m m' + h l' + l h' in a second one that is 2^-8 of it, so that neither loses bits of the other.
// The rest is below 2^-25 of |x y|.  An output that is not finite (infinities split into NaN, values within 2^-9 of the largest float round
// to infinity) is computed again from the operands.
#pragma once

#include "dense_types.cuh"

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
    bool fours;         // four columns of every operand can be read and written at once
};

// An operand: values `ld` apart along one dimension and side by side along the other; read `bytes` at a time.
template <typename T>
struct Operand {
    const T *at;
    long long ld;
    int bytes;
};

template <typename T> struct TileShape {
    static constexpr int PLANES = sizeof(T) == 4 ? 3 : 1;
    static constexpr int KS = sizeof(T) == 4 ? 32 : 64;          // of K in a step
    static constexpr int STAGES = sizeof(T) == 4 ? 2 : 3;
    static constexpr int ROWS = 128, THREADS = 256 + 32;
    static constexpr int operand_bytes(int rows) { return PLANES * rows * KS * 2; }
    static constexpr int stage_bytes(int bn) { return operand_bytes(ROWS) + operand_bytes(bn); }
    static constexpr int accumulators = sizeof(T) == 4 ? 2 : 1;
    static constexpr int shared_bytes(int bn) { return STAGES * stage_bytes(bn) + 1024; }
};

__device__ __forceinline__ unsigned shared_address(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void barrier_init(unsigned bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count)); }
__device__ __forceinline__ void barrier_arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory"); }
// Waits for a phase of a barrier, two seconds at most: false if it did not end.
__device__ __forceinline__ bool barrier_wait(unsigned bar, unsigned parity) {
    unsigned long long began = 0;
    for (;;) {
        unsigned done;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
        unsigned long long now;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
        if (began == 0) began = now;
        else if (now - began > 2000000000ull) return false;
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

// Eight values side by side, of which `live` exist (the others are 0).
__device__ __forceinline__ void load_eight(const float *p, int live, int bytes, float (&v)[8]) {
    if (live >= 8) {
        if (bytes == 16) {
            const float4 a = __ldg((const float4 *)p), b = __ldg((const float4 *)p + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else if (bytes == 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 a = __ldg((const float2 *)p + i);
                v[2 * i] = a.x, v[2 * i + 1] = a.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __ldg(p + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < live ? __ldg(p + i) : 0.f;
    }
}
// 16-bit values in pairs
template <typename T>
__device__ __forceinline__ void load_eight(const T *p, int live, int bytes, unsigned (&v)[4]) {
    if (live >= 8 && bytes >= 4) {
        if (bytes == 16) {
            const uint4 a = __ldg((const uint4 *)p);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        } else if (bytes == 8) {
            const uint2 a = __ldg((const uint2 *)p), b = __ldg((const uint2 *)p + 1);
            v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __ldg((const unsigned *)p + i);
        }
    } else {
        const unsigned short *q = reinterpret_cast<const unsigned short *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned lo = 2 * i < live ? __ldg(q + 2 * i) : 0, hi = 2 * i + 1 < live ? __ldg(q + 2 * i + 1) : 0;
            v[i] = lo | hi << 16;
        }
    }
}

__device__ __forceinline__ void store_shared(unsigned at, unsigned a, unsigned b, unsigned c, unsigned d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ unsigned bf16_pair(float low, float high) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(low, high);
    return reinterpret_cast<const unsigned &>(p);
}
__device__ __forceinline__ void store_eight(unsigned at, unsigned plane_bytes, const float (&v)[8]) {
    unsigned h[4], m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = v[2 * i], b = v[2 * i + 1];
        h[i] = bf16_pair(a, b);
        a -= __uint_as_float(h[i] << 16), b -= __uint_as_float(h[i] & 0xffff0000u);
        m[i] = bf16_pair(a, b);
        a -= __uint_as_float(m[i] << 16), b -= __uint_as_float(m[i] & 0xffff0000u);
        l[i] = bf16_pair(a, b);
    }
    store_shared(at, h[0], h[1], h[2], h[3]);
    store_shared(at + plane_bytes, m[0], m[1], m[2], m[3]);
    store_shared(at + 2 * plane_bytes, l[0], l[1], l[2], l[3]);
}
__device__ __forceinline__ void store_eight(unsigned at, unsigned, const unsigned (&v)[4]) { store_shared(at, v[0], v[1], v[2], v[3]); }

// What a thread brings of an operand in each step: UNITS times eight values.
template <typename T, int R, bool ALONG_K>
struct Share {
    using S = TileShape<T>;
    using L = SharedLayout<S::KS, ALONG_K>;
    static constexpr int ACROSS = (ALONG_K ? S::KS : R) / 8;                 // units of a row
    static constexpr int UNITS = R * S::KS / 8 / 256, STEP = 256 / ACROSS;   // rows between a thread's units
    static constexpr unsigned PLANE = R * S::KS * 2;
    using Eight = std::conditional_t<sizeof(T) == 4, float[8], unsigned[4]>;
    const T *at;
    long long ld;
    // limit: rows or columns of the tile that exist; needed: that the instructions read; k: of K until the share's end
    int row, unit, bytes, limit, needed, k;

    __device__ Share(const Operand<T> &o, long long start, int size, int read, int k0, int k1) : ld(o.ld), bytes(o.bytes), limit(size), needed(read), k(k1 - k0) {
        row = threadIdx.x / ACROSS, unit = threadIdx.x % ACROSS;
        at = ALONG_K ? o.at + (start + row) * ld + k0 + unit * 8 : o.at + (long long)(k0 + row) * ld + start + unit * 8;
    }
    __device__ void load(Eight (&v)[UNITS]) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int r = row + u * STEP;
            const bool in_row = ALONG_K ? r < limit : r < k;
            load_eight(at + (long long)(u * STEP) * ld, in_row ? (ALONG_K ? k : limit) - unit * 8 : 0, bytes, v[u]);
        }
        k -= S::KS;
        at += ALONG_K ? S::KS : S::KS * ld;
    }
    __device__ void store(unsigned to, const Eight (&v)[UNITS]) const {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int r = row + u * STEP;
            if ((ALONG_K ? r : unit * 8) < needed) store_eight(to + L::offset(r, unit), PLANE, v[u]);
        }
    }
};

__device__ __forceinline__ void mma(unsigned accumulator, unsigned long long a, unsigned long long b, unsigned instruction, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(accumulator), "l"(a), "l"(b),
                 "r"(instruction), "r"((unsigned)add) : "memory");
}
__device__ __forceinline__ void mma_commit(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void load_accumulators(unsigned at, float (&v)[32]) {
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

// One output from the operands, for those that the split does not give.
template <typename T, bool A_ALONG_K, bool B_ALONG_K>
__device__ __noinline__ float plain_product(Operand<T> A, Operand<T> B, long long m, int n, int k0, int k1) {
    float acc = 0;
    for (int k = k0; k < k1; ++k)
        acc = fmaf(to_float(A.at[A_ALONG_K ? m * A.ld + k : k * A.ld + m]), to_float(B.at[B_ALONG_K ? n * B.ld + k : k * B.ld + n]), acc);
    return acc;
}

template <typename T, int BN, bool A_ALONG_K, bool B_ALONG_K>
__global__ void __launch_bounds__(TileShape<T>::THREADS, 2)
product_tile_kernel(Operand<T> A, Operand<T> B, int M, int N, int K, int share, LinearOut<T> out) {
    using S = TileShape<T>;
    using LA = SharedLayout<S::KS, A_ALONG_K>;
    using LB = SharedLayout<S::KS, B_ALONG_K>;
    constexpr int COLUMNS = S::accumulators * BN, A_PLANE = S::ROWS * S::KS * 2, B_PLANE = BN * S::KS * 2, A_BYTES = S::operand_bytes(S::ROWS);
    extern __shared__ char bytes[];
    __shared__ __align__(8) unsigned long long bars[2 * S::STAGES + 1];
    __shared__ unsigned tensor_memory;
    char *const shared = bytes + ((1024 - (shared_address(bytes) & 1023)) & 1023);
    const unsigned stages = shared_address(shared), full = shared_address(bars), empty = full + 8 * S::STAGES, all_done = full + 16 * S::STAGES;
    const int tiles_n = (N + BN - 1) / BN, warp = threadIdx.x >> 5;
    const long long m0 = (long long)(blockIdx.x / tiles_n) * S::ROWS;
    const int n0 = (int)(blockIdx.x % tiles_n) * BN, k0 = (int)blockIdx.y * share, k1 = min(K, k0 + share), steps = (k1 - k0 + S::KS - 1) / S::KS;
    const int columns = min(BN, (N - n0 + 15) / 16 * 16);      // of the tile that the instructions compute

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            barrier_init(full + 8 * s, 256);
            barrier_init(empty + 8 * s, 1);
        }
        barrier_init(all_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(shared_address(&tensor_memory)), "n"(COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned accumulators = tensor_memory;

    bool ended = true;      // no wait was given up
    if (warp < 8) {
        Share<T, S::ROWS, A_ALONG_K> a(A, m0, (int)min((long long)S::ROWS, M - m0), S::ROWS, k0, k1);
        Share<T, BN, B_ALONG_K> b(B, n0, min(BN, N - n0), columns, k0, k1);
        typename decltype(a)::Eight va[decltype(a)::UNITS];
        typename decltype(b)::Eight vb[decltype(b)::UNITS];
        a.load(va);
        b.load(vb);
        for (int s = 0; s < steps && ended; ++s) {
            const int stage = s % S::STAGES;
            if (s >= S::STAGES) ended = barrier_wait(empty + 8 * stage, (s / S::STAGES - 1) & 1);
            const unsigned to = stages + stage * S::stage_bytes(BN);
            a.store(to, va);
            b.store(to + A_BYTES, vb);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            barrier_arrive(full + 8 * stage);
            if (s + 1 < steps) {
                a.load(va);
                b.load(vb);
            }
        }
    } else if (threadIdx.x == 256) {
        // float accumulators, both operands of this type, rows along K (0) or not (1), columns / 8, rows / 16
        constexpr unsigned TYPE = std::is_same_v<T, __half> ? 0 : 1;
        const unsigned instruction = 1u << 4 | TYPE << 7 | TYPE << 10 | (A_ALONG_K ? 0u : 1u) << 15 | (B_ALONG_K ? 0u : 1u) << 16 | (unsigned)(columns / 8) << 17 |
                                     (unsigned)(S::ROWS / 16) << 24;
        for (int s = 0; s < steps && ended; ++s) {
            const int stage = s % S::STAGES;
            ended = barrier_wait(full + 8 * stage, (s / S::STAGES) & 1);
            if (!ended) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned a = stages + stage * S::stage_bytes(BN), b = a + A_BYTES;
#pragma unroll
            for (int k = 0; k < S::KS; k += 16) {
                const bool add = s > 0 || k > 0;
                if (S::PLANES == 1) {
                    mma(accumulators, LA::descriptor(a, k), LB::descriptor(b, k), instruction, add);
                } else {
                    const unsigned long long ah = LA::descriptor(a, k), am = LA::descriptor(a + A_PLANE, k), al = LA::descriptor(a + 2 * A_PLANE, k);
                    const unsigned long long bh = LB::descriptor(b, k), bm = LB::descriptor(b + B_PLANE, k), bl = LB::descriptor(b + 2 * B_PLANE, k);
                    mma(accumulators, ah, bh, instruction, add);
                    mma(accumulators + BN, ah, bl, instruction, add);
                    mma(accumulators + BN, al, bh, instruction, true);
                    mma(accumulators + BN, am, bm, instruction, true);
                    mma(accumulators + BN, ah, bm, instruction, true);
                    mma(accumulators + BN, am, bh, instruction, true);
                }
            }
            mma_commit(empty + 8 * stage);
        }
        mma_commit(all_done);
    }
    __syncwarp();
    ended = barrier_wait(all_done, 0) && ended;
    ended = __syncthreads_and(ended);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");

    // Accumulators to shared memory (a row a lane), from there to the outputs with neighbouring columns in neighbouring lanes.
    constexpr int PITCH = BN + 4;
    static_assert(S::ROWS * PITCH * 4 <= S::STAGES * S::stage_bytes(BN), "the tile fits the stages");
    float *const tile = reinterpret_cast<float *>(shared);
    if (warp < 8) {
        const int row = (warp & 3) * 32 + (threadIdx.x & 31);
        for (int c = (warp >> 2) * 32; c < columns; c += 64) {
            float v[32];
            const unsigned at = accumulators + ((unsigned)((warp & 3) * 32) << 16) + c;
            load_accumulators(at, v);
            if (S::PLANES > 1) {
                float w[32];
                load_accumulators(at + BN, w);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] += w[i];
            }
            if (!ended)      // a wait was given up: nothing plausible comes out
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = NAN;
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4 *>(tile + row * PITCH + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    __syncthreads();
    if (warp == 8) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(accumulators), "n"(COLUMNS));
        return;
    }
    const int rows = (int)min((long long)S::ROWS, M - m0), width = min(BN, N - n0);
    auto mended = [&](float acc, int r, int c) {      // what the split does not give
        if (S::PLANES > 1 && !(fabsf(acc) < INFINITY)) acc = ended ? plain_product<T, A_ALONG_K, B_ALONG_K>(A, B, m0 + r, n0 + c, k0, k1) : NAN;
        return acc;
    };
    if (out.shares) {
        float *const to = out.shares + ((long long)blockIdx.y * M + m0) * N + n0;
        for (int r = warp; r < rows; r += 8)
            for (int c = threadIdx.x & 31; c < width; c += 32) to[(long long)r * N + c] = mended(tile[r * PITCH + c], r, c);
        return;
    }
    with_activation(out.activation, [&](auto act) {
        constexpr int ACTIVATION = decltype(act)::value;
        if (out.fours) {
            constexpr int LANES = BN / 4, AT_ONCE = 256 / LANES;      // of a row; rows
            using Four = Values<T, 4>;
            const int c = (int)(threadIdx.x % LANES) * 4;
            if (c >= width) return;
            float4 b = make_float4(0, 0, 0, 0);
            if (out.bias) b = __ldg((const float4 *)(out.bias + n0 + c));
#pragma unroll 2
            for (int r = threadIdx.x / LANES; r < rows; r += AT_ONCE) {
                const long long row = m0 + r;
                Four x = {}, y;
                if (out.residual) x = *reinterpret_cast<const Four *>(out.residual + row * out.ldr + n0 + c);
                const float4 acc = *reinterpret_cast<const float4 *>(tile + r * PITCH + c);
                float z[4] = {mended(acc.x, r, c) + b.x, mended(acc.y, r, c + 1) + b.y, mended(acc.z, r, c + 2) + b.z, mended(acc.w, r, c + 3) + b.w}, v[4], added[4];
                x.get(added);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = activate<T, ACTIVATION>(z[i]);
                    if (out.residual) v[i] += added[i];
                }
                if (out.pre) {
                    Four p;
                    p.set(z);
                    *reinterpret_cast<Four *>(out.pre + row * out.ldp + n0 + c) = p;
                }
                y.set(v);
                *reinterpret_cast<Four *>(out.y + row * out.ldy + n0 + c) = y;
            }
            return;
        }
        for (int r = warp; r < rows; r += 8)
            for (int c = threadIdx.x & 31; c < width; c += 32) {
                const long long row = m0 + r;
                float acc = mended(tile[r * PITCH + c], r, c);
                if (out.bias) acc += __ldg(out.bias + n0 + c);
                if (out.pre) out.pre[row * out.ldp + n0 + c] = from_float<T>(acc);
                float v = activate<T, ACTIVATION>(acc);
                if (out.residual) v += to_float(out.residual[row * out.ldr + n0 + c]);
                out.y[row * out.ldy + n0 + c] = from_float<T>(v);
            }
    });
}

// How many bytes of an operand's rows can be read at once.
template <typename T>
Operand<T> operand(const void *p, long long ld) {
    const unsigned long long bits = reinterpret_cast<uintptr_t>(p) | (unsigned long long)ld * sizeof(T) | 16;
    return {(const T *)p, ld, (int)(bits & (~bits + 1))};
}

template <typename T, int BN, bool A_ALONG_K, bool B_ALONG_K>
int launch_product_tiles(const Operand<T> &A, const Operand<T> &B, int M, int N, int K, int share, int shares, const LinearOut<T> &out, cudaStream_t st) {
    constexpr int bytes = TileShape<T>::shared_bytes(BN);
    auto *const kernel = product_tile_kernel<T, BN, A_ALONG_K, B_ALONG_K>;
    DRONE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    const long long tiles = (long long)ceil_div(M, 128) * ceil_div(N, BN);
    kernel<<<dim3((unsigned)tiles, shares), TileShape<T>::THREADS, bytes, st>>>(A, B, M, N, K, share, out);
    DRONE_LAUNCH_CHECK("product_tile_kernel");
    return DRONE_OK;
}

}  // namespace drone
