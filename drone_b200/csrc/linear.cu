// Products of a dense layer, Y = activation(X W + bias) + residual, and its backward pass.
#include "product_tile.cuh"
#include "row_shape.cuh"
#include "thin_products.cuh"

#include <algorithm>

namespace drone {

// Shares of a product, added in order.  A block has 256 / WAYS values, its parts every WAYS-th share: all of them for a thread where they are few.
template <typename T, int WAYS>
__global__ void __launch_bounds__(256) add_product_shares_kernel(const float *__restrict__ parts, int shares, int M, int N, T *__restrict__ out, long long ld) {
    constexpr int VALUES = 256 / WAYS;
    __shared__ double of_part[WAYS][VALUES];
    const long long count = (long long)M * N, i = (long long)blockIdx.x * VALUES + threadIdx.x % VALUES;
    const int w = threadIdx.x / VALUES;
    double sum = 0;
    if (i < count) {
#pragma unroll 8
        for (int s = w; s < shares; s += WAYS) sum += __ldg(parts + s * count + i);
    }
    if (WAYS > 1) {
        of_part[w][threadIdx.x % VALUES] = sum;
        __syncthreads();
    }
    if (w == 0 && i < count) {
        for (int o = 1; o < WAYS; ++o) sum += of_part[o][threadIdx.x];
        out[i / N * ld + i % N] = from_float<T>((float)sum);
    }
}

template <typename T>
static int add_product_shares(const float *parts, int shares, int M, int N, T *out, long long ld, cudaStream_t st) {
    const long long values = (long long)M * N;
    if (shares <= 32) add_product_shares_kernel<T, 1><<<ceil_div(values, 256), 256, 0, st>>>(parts, shares, M, N, out, ld);
    else add_product_shares_kernel<T, 8><<<ceil_div(values, 32), 256, 0, st>>>(parts, shares, M, N, out, ld);
    DRONE_LAUNCH_CHECK("add_product_shares_kernel");
    return DRONE_OK;
}

// A few rows: W is read once for up to ROWS of them, by as many warps as there are loads to hide.
//   W [K, N]: a block has 32 columns, a lane one of them, its 32 warps every 32nd k; the warps' sums are added in order.
//   W [N, K]: a warp has a column, its lanes every 32nd k.
constexpr int kFewRows = 8;
// Where that is faster than a few tiles, whose steps of K follow one another however few rows there are.  us here / with tiles: floats 602 x 128
// 256 rows 7.9 / 21.8, 512 rows 14 / 21.8, 1024 rows 26 / 21.8; 256 x 256 256 rows 7.9 / 12.9, 512 rows 14 / 12.9; 2048 x 2048 32 rows 36 / 58, 64
// rows 68 / 58; with a call's image of the weights, 1400 rows 600 x 32 16 / 29, 2048 rows 600 x 8 16 / 23, 4096 rows 164 x 21 15 / 19, 4096 rows 300 x 25 19 / 20, 8192
// rows 100 x 12 15 / 19, 8192 rows 164 x 21 25 / 20, 4096 rows 600 x 32 29 / 23; bfloat16 256 x 256 32 rows 5.1 / 6.8, 256 rows 9.2 / 7.2; 2048 x 2048 1 row 6.6 / 13.9, 4 rows 24 / 13.9.
static bool few_rows(int type, int n, int N, int K) {
    const long long outputs = (long long)n * N;
    if (type == DRONE_F32 && N <= 32 && n <= 8192 && (long long)ceil_div(n, kFewRows) * K <= 1 << 17) return true;
    return n == 1 || (type == DRONE_F32 ? n <= 512 && outputs <= 1 << 16 : outputs <= 1 << 13 && outputs * K <= 1 << 22);
}
template <typename T, bool TRANSPOSED>
__global__ void __launch_bounds__(TRANSPOSED ? 256 : 1024) few_rows_kernel(Operand<T> X, Operand<T> W, int n, int N, int K, LinearOut<T> out) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row0 = blockIdx.y * kFewRows, rows = min(kFewRows, n - row0);
    const T *x = X.at + row0 * X.ld;
    float acc[kFewRows];
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) acc[r] = 0;
    const int c = TRANSPOSED ? (int)blockIdx.x * 8 + warp : (int)blockIdx.x * 32 + lane;
    if (c < N) {
        const T *w = TRANSPOSED ? W.at + c * W.ld : W.at + c;
        const long long along = TRANSPOSED ? 1 : W.ld;
        auto add = [&](auto all) {      // rows that do not exist read the last one
            constexpr int R = decltype(all)::value;
#pragma unroll(R == 1 ? 8 : 4)
            for (int k = TRANSPOSED ? lane : warp; k < K; k += 32) {
                const float v = to_float(w[k * along]);
#pragma unroll
                for (int r = 0; r < R; ++r) acc[r] = fmaf(to_float(x[(R == 1 ? 0 : min(r, rows - 1)) * X.ld + k]), v, acc[r]);
            }
        };
        if (rows == 1) add(std::integral_constant<int, 1>());
        else add(std::integral_constant<int, kFewRows>());
    }
    if constexpr (TRANSPOSED) {
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
        if (c < N && lane < rows) {
            float z = 0;
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) z = lane == r ? acc[r] : z;
            with_activation(out.activation, [&](auto act) { put_value<T, decltype(act)::value>(out, row0 + lane, c, z); });
        }
    } else {
        __shared__ float of_warp[32][kFewRows][32];
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
            if (r < rows) of_warp[warp][r][lane] = acc[r];
        __syncthreads();
        if (warp < rows && c < N) {
            float z = 0;
#pragma unroll 8
            for (int i = 0; i < 32; ++i) z += of_warp[i][warp][lane];
            with_activation(out.activation, [&](auto act) { put_value<T, decltype(act)::value>(out, row0 + warp, c, z); });
        }
    }
}

// Many rows, few products each: a block keeps W and some rows of X in shared memory as floats, a thread an output at a time, so that X and Y go
// over neighbouring lanes whatever their widths and distances.  Bound: two reads of shared memory a product; where one side is of a few values and the other long
// thin_products.cuh is faster.  us here / with tiles: 410,000 x 3 x 20 floats 35 / 60, bfloat16 37 / 57; 3,000 x 16 x 7 18 / 25 and 18 / 24; but 400,000 x 16 x
// 64 158 / 72.
constexpr int kNarrowProducts = 128, kNarrowValues = 8192;
static bool narrow_rows(int K, int N) { return (long long)K * N <= kNarrowProducts; }
template <typename T>
__global__ void __launch_bounds__(256) narrow_rows_kernel(Operand<T> X, Operand<T> W, bool transposed, int n, int N, int K, int rows_at_once, LinearOut<T> out) {
    __shared__ float w[kNarrowProducts], x[kNarrowValues];
    for (int i = threadIdx.x; i < K * N; i += 256) {
        const int k = i / N, c = i % N;
        w[i] = to_float(W.at[transposed ? c * W.ld + k : k * W.ld + c]);
    }
    const int pitch = K | 1;
    with_activation(out.activation, [&](auto act) {
        for (long long row0 = (long long)blockIdx.x * rows_at_once; row0 < n; row0 += (long long)gridDim.x * rows_at_once) {
            const int rows = (int)min((long long)rows_at_once, n - row0);
            __syncthreads();
            for (RowColumn at(threadIdx.x, 256, K); at.row < rows; at.advance()) x[at.row * pitch + at.col] = to_float(X.at[(row0 + at.row) * X.ld + at.col]);
            __syncthreads();
            for (RowColumn at(threadIdx.x, 256, N); at.row < rows; at.advance()) {
                float acc = 0;
#pragma unroll 4
                for (int k = 0; k < K; ++k) acc = fmaf(x[at.row * pitch + k], w[k * N + at.col], acc);
                put_value<T, decltype(act)::value>(out, row0 + at.row, at.col, acc);
            }
        }
    });
}

// Its weight gradient: a thread has a value of dW and every 256 / values-th row of what the block keeps; shares[block].
template <typename T>
__global__ void __launch_bounds__(256) narrow_gradient_kernel(Operand<T> X, Operand<T> Z, int n, int N, int K, bool transposed, int rows_at_once, float *shares) {
    __shared__ float x[kNarrowValues / 2], z[kNarrowValues / 2];
    const int values = K * N, parts = 256 / values, part = (int)threadIdx.x / values, value = (int)threadIdx.x % values;
    const int k = transposed ? value % K : value / N, c = transposed ? value / K : value % N, pitch_x = K | 1, pitch_z = N | 1;
    float acc = 0;
    for (long long row0 = (long long)blockIdx.x * rows_at_once; row0 < n; row0 += (long long)gridDim.x * rows_at_once) {
        const int rows = (int)min((long long)rows_at_once, n - row0);
        __syncthreads();
        for (RowColumn at(threadIdx.x, 256, K); at.row < rows; at.advance()) x[at.row * pitch_x + at.col] = to_float(X.at[(row0 + at.row) * X.ld + at.col]);
        for (RowColumn at(threadIdx.x, 256, N); at.row < rows; at.advance()) z[at.row * pitch_z + at.col] = to_float(Z.at[(row0 + at.row) * Z.ld + at.col]);
        __syncthreads();
        if (part < parts)
            for (int r = part; r < rows; r += parts) acc = fmaf(x[r * pitch_x + k], z[r * pitch_z + c], acc);
    }
    __syncthreads();
    x[threadIdx.x] = acc;
    __syncthreads();
    if ((int)threadIdx.x < values) {
        float sum = 0;
        for (int i = 0; i < parts; ++i) sum += x[i * values + threadIdx.x];
        shares[(long long)blockIdx.x * values + threadIdx.x] = sum;
    }
}
// Rows that a block has at a time, of so many values each; blocks.
static int narrow_rows_at_once(int width, int operands) { return std::min(256, kNarrowValues / operands / (width | 1)); }
static int narrow_blocks(int n, int rows_at_once, int sms) { return (int)std::min<long long>(((long long)n + rows_at_once - 1) / rows_at_once, sms * 3); }

// 16-bit rows to rows that start on 16 bytes: a thread 16 bytes of them.  What lies behind a row's end is never read.
__global__ void __launch_bounds__(256) pad_rows_kernel(const unsigned short *__restrict__ from, long long ld, int n, int width, uint4 *__restrict__ to, int vectors) {
    const bool pairs = (reinterpret_cast<uintptr_t>(from) & 3) == 0 && ld % 2 == 0;
    for (RowColumn at(blockIdx.x * 256LL + threadIdx.x, gridDim.x * 256LL, vectors); at.row < n; at.advance()) {
        const unsigned short *p = from + at.row * ld + at.col * 8;
        const int live = width - at.col * 8;
        unsigned v[4];
        if (pairs && live >= 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __ldg((const unsigned *)p + i);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (2 * i < live ? (unsigned)__ldg(p + 2 * i) : 0u) | (2 * i + 1 < live ? (unsigned)__ldg(p + 2 * i + 1) : 0u) << 16;
        }
        to[(long long)at.row * vectors + at.col] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}
// Floats that the copy of such a matrix takes: none if its rows are on 16 bytes as they are.
static long long padded_floats(const void *p, long long ld, long long rows, int width) {
    return rows_on_16_bytes(p, ld, 2) ? 0 : rows * ((width + 7) / 8) * 4;
}
// The matrix itself, or its copy at *scratch, which moves on.
template <typename T>
static int on_16_bytes(const void *p, long long ld, int rows, int width, float **scratch, int sms, cudaStream_t st, Operand<T> *out) {
    const long long floats = padded_floats(p, ld, rows, width);
    if (floats == 0) {
        *out = operand<T>(p, ld);
        return DRONE_OK;
    }
    const int vectors = (width + 7) / 8;
    pad_rows_kernel<<<(int)std::min<long long>(((long long)rows * vectors + 255) / 256, sms * 16), 256, 0, st>>>((const unsigned short *)p, ld, rows, width, (uint4 *)*scratch,
                                                                                                            vectors);
    DRONE_LAUNCH_CHECK("pad_rows_kernel");
    *out = operand<T>(*scratch, vectors * 8);
    *scratch += floats;
    return DRONE_OK;
}

int tile_map(CUtensorMap *map, bool bf16, const void *p, long long width, long long rows, long long ld, int box) {
    using Encode = decltype(&cuTensorMapEncodeTiled);
    static const Encode encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        return cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) == cudaSuccess ? (Encode)f : nullptr;
    }();
    if (!encode) return set_error(DRONE_E_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t sizes[2] = {(cuuint64_t)width, (cuuint64_t)rows}, stride[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t boxes[2] = {64, (cuuint32_t)box}, steps[2] = {1, 1};
    const CUresult rc = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(p), sizes, stride, boxes, steps,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? DRONE_OK : set_error(DRONE_E_CUDA, "cuTensorMapEncodeTiled failed: %d (%lld x %lld, %lld apart)", (int)rc, rows, width, ld);
}

// dZ = G * activation'(pre) and the sums of its columns, of those from blockIdx.y * width on; sums[blockIdx.x] = those of the block's rows.
// Bound: HBM, two reads and a write: 232,965 rows of 128 floats, ReLU, 57 us (98 % of the copy rate), 100,003 of 512 bfloat16, GELU, 65 (73 %).
template <typename T, int L, int U, bool VEC, int ACTIVATION>
__global__ void __launch_bounds__(256, 4)
activation_gradient_kernel(const T *G, long long ldg, const T *pre, long long ldp, int n, int N, int width, T *dZ, long long ldz, float *sums) {
    using S = RowShape<T, L, U, VEC>;
    const int gl = threadIdx.x % L, c0 = blockIdx.y * width, F = min(width, N - c0);
    float sum[S::PER];
#pragma unroll
    for (int i = 0; i < S::PER; ++i) sum[i] = 0;
    for (long long row = (long long)blockIdx.x * S::GROUPS + threadIdx.x / L; row < n; row += (long long)gridDim.x * S::GROUPS) {
        float d[S::PER];
        S::load(G + row * ldg + c0, F, gl, d);
        if (ACTIVATION != DRONE_ACT_NONE) {
            float z[S::PER];
            S::load(pre + row * ldp + c0, F, gl, z);
#pragma unroll
            for (int i = 0; i < S::PER; ++i) d[i] *= activation_slope<T, ACTIVATION>(z[i]);
            if (dZ) S::store(dZ + row * ldz + c0, F, gl, d);
        } else if (dZ) {
            S::store(dZ + row * ldz + c0, F, gl, d);
        }
#pragma unroll
        for (int i = 0; i < S::PER; ++i) sum[i] += d[i];
    }
    if (sums) S::add_groups(sum, F, gl, sums + (long long)blockIdx.x * N + c0);
}

// A block has 32 of the columns, its 32 warps every 32nd of the sums (with 8 warps 888 blocks' sums of 128 columns took 20 us).
__global__ void __launch_bounds__(1024) fold_columns_kernel(const float *__restrict__ sums, int blocks, int columns, float *a, int split, float *b) {
    __shared__ double of_warp[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
    double sum = 0;
    if (c < columns) {
#pragma unroll 8
        for (int i = w; i < blocks; i += 32) sum += __ldg(sums + (long long)i * columns + c);
    }
    of_warp[threadIdx.x & 31][w] = sum;
    __syncthreads();
    sum = of_warp[w][threadIdx.x & 31];      // a warp a column
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int column = blockIdx.x * 32 + w;
    if ((threadIdx.x & 31) == 0 && column < columns) {
        if (column < split) {
            if (a) a[column] = (float)sum;
        } else if (b) {
            b[column - split] = (float)sum;
        }
    }
}

int fold_columns(const float *sums, int blocks, int columns, float *a, int split, float *b, cudaStream_t st) {
    fold_columns_kernel<<<ceil_div(columns, 32), 1024, 0, st>>>(sums, blocks, columns, a, split, b);
    DRONE_LAUNCH_CHECK("fold_columns_kernel");
    return DRONE_OK;
}

// How the rows of a weight gradient, its K, are cut: a block an SM, but a share of four steps at least.
struct Shares {
    int share, count;
};
template <typename T>
static Shares product_shares(int M, int N, int K, int sms) {
    using S = TileShape<T>;
    const int most = std::max(1, sms / (ceil_div(M, S::ROWS) * ceil_div(N, S::BN)));
    Shares s;
    s.share = std::max(4 * S::KS, ceil_div(ceil_div(K, most), S::KS) * S::KS);
    s.count = std::max(1, ceil_div(K, s.share));
    return s;
}
static Shares product_shares(int type, int M, int N, int K, int sms) {
    return type == DRONE_F32 ? product_shares<float>(M, N, K, sms) : product_shares<__half>(M, N, K, sms);
}

// Blocks of the activations' gradient: as many as the SMs hold, of at most 64 vectors a row.
struct GradientBlocks {
    int width, columns, rows;      // of a block; blocks along the columns and the rows
};
static GradientBlocks gradient_blocks(int type, int n, int N, int sms) {
    const int V = 16 / type_size(type);
    GradientBlocks b;
    b.width = std::min(N, 64 * V);
    b.columns = ceil_div(N, b.width);
    const int groups = ceil_div(b.width, V) <= 16 ? 32 : 8;
    b.rows = (int)std::min<long long>(((long long)n + groups - 1) / groups, std::max(1, 4 * sms / b.columns));
    return b;
}

}  // namespace drone

using namespace drone;

#define DRONE_LINEAR_SIZES(n_rows, K, N) \
    ((n_rows) >= 0 && (n_rows) <= 1 << 30 && (K) >= 1 && (K) <= 1 << 15 && (N) >= 1 && (N) <= 1 << 15)

extern "C" {

int drone_linear_scratch(int type, int n_rows, int K, int N, const void *d_X, int ldx, const void *d_W, int ldw, int transposed, long long *n_floats) {
    DRONE_REQUIRE(DRONE_TYPE_OK(type) && DRONE_LINEAR_SIZES(n_rows, K, N) && (transposed == 0 || transposed == 1) && n_floats,
                  "drone_linear_scratch: type=%d n_rows=%d K=%d N=%d transposed=%d", type, n_rows, K, N, transposed);
    using S = TileShape<float>;
    if (few_rows(type, n_rows, N, K) || narrow_rows(K, N) || few_columns(K, N) || short_rows(type, K, N)) *n_floats = 0;
    else if (type == DRONE_F32) *n_floats = (long long)ceil_div(N, S::BN) * ceil_div(K, S::KS) * (S::B_BYTES / 4);      // the image of the weights
    else *n_floats = padded_floats(d_X, ldx, n_rows, K) + padded_floats(d_W, ldw, transposed ? N : K, transposed ? K : N);
    return DRONE_OK;
}

int drone_linear(int type, int n_rows, int K, int N, const void *d_X, int ldx, const void *d_W, int ldw, int transposed, const float *d_bias,
                 int activation, const void *d_residual, int ldr, void *d_Y, int ldy, void *d_pre, int ldp, float *d_scratch, long long n_scratch, void *stream) {
    DRONE_REQUIRE(DRONE_TYPE_OK(type), "drone_linear: type=%d", type);
    DRONE_REQUIRE(DRONE_LINEAR_SIZES(n_rows, K, N), "drone_linear: n_rows=%d K=%d N=%d", n_rows, K, N);
    DRONE_REQUIRE(activation >= DRONE_ACT_NONE && activation <= DRONE_ACT_SILU, "drone_linear: activation=%d", activation);
    DRONE_REQUIRE((transposed == 0 || transposed == 1) && ldx >= K && ldw >= (transposed ? K : N) && ldy >= N && (!d_residual || ldr >= N) &&
                  (!d_pre || ldp >= N), "drone_linear: ldx=%d ldw=%d transposed=%d ldr=%d ldy=%d ldp=%d", ldx, ldw, transposed, ldr, ldy, ldp);
    if (n_rows == 0) return DRONE_OK;
    DRONE_REQUIRE(d_X && d_W && d_Y, "drone_linear: NULL argument");
    DRONE_REQUIRE(DRONE_ALIGNED(d_X, type) && DRONE_ALIGNED(d_W, type) && DRONE_ALIGNED(d_Y, type) && DRONE_ALIGNED(d_residual, type) &&
                  DRONE_ALIGNED(d_pre, type) && (reinterpret_cast<uintptr_t>(d_bias) & 3) == 0, "drone_linear: an operand is not aligned to its type");
    long long need = 0;
    int sms = 0, rc = drone_linear_scratch(type, n_rows, K, N, d_X, ldx, d_W, ldw, transposed, &need);
    if (rc) return rc;
    DRONE_REQUIRE(need == 0 || (n_scratch >= need && d_scratch && (reinterpret_cast<uintptr_t>(d_scratch) & 15) == 0),
                  "drone_linear: %lld floats of scratch on 16 bytes needed, %lld at %p given", need, n_scratch, (void *)d_scratch);
    rc = device_sms(&sms);
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    return with_type(type, [&](auto tag) {
        using T = typename decltype(tag)::T;
        const auto in_steps_of = [&](int values) {
            const auto fits = [&](const void *p, long long ld) { return !p || ((reinterpret_cast<uintptr_t>(p) & (values * sizeof(T) - 1)) == 0 && ld % values == 0); };
            return N % values == 0 && (reinterpret_cast<uintptr_t>(d_bias) & 15) == 0 && fits(d_Y, ldy) && fits(d_residual, ldr) && fits(d_pre, ldp);
        };
        const int at_once = in_steps_of(kVector<T>) ? kVector<T> : in_steps_of(4) ? 4 : 1;
        const LinearOut<T> out = {d_bias, activation, (const T *)d_residual, ldr, (T *)d_Y, ldy, (T *)d_pre, ldp, nullptr, at_once};
        const Operand<T> x = operand<T>(d_X, ldx), w = operand<T>(d_W, ldw);
        if (few_rows(type, n_rows, N, K)) {
            const int groups = ceil_div(n_rows, kFewRows);
            if (transposed) few_rows_kernel<T, true><<<dim3(ceil_div(N, 8), groups), 256, 0, st>>>(x, w, n_rows, N, K, out);
            else few_rows_kernel<T, false><<<dim3(ceil_div(N, 32), groups), 1024, 0, st>>>(x, w, n_rows, N, K, out);
            DRONE_LAUNCH_CHECK("few_rows_kernel");
            return DRONE_OK;
        }
        if (few_columns(K, N)) return launch_few_columns<T>(x, w, transposed != 0, n_rows, N, K, out, sms, st);
        if constexpr (sizeof(T) == 4) {
            if (short_rows(type, K, N)) return launch_short_rows(x, w, transposed != 0, n_rows, N, K, out, sms, st);
        }
        if (narrow_rows(K, N)) {
            const int rows_at_once = narrow_rows_at_once(K, 1);
            narrow_rows_kernel<T><<<(int)std::min<long long>(((long long)n_rows + rows_at_once - 1) / rows_at_once, sms * 5), 256, 0, st>>>(x, w, transposed != 0, n_rows, N,
                                                                                                                                 K, rows_at_once, out);
            DRONE_LAUNCH_CHECK("narrow_rows_kernel");
            return DRONE_OK;
        }
        if constexpr (sizeof(T) == 2) {
            Operand<T> a, b;
            float *scratch = d_scratch;
            int failed = on_16_bytes(d_X, ldx, n_rows, K, &scratch, sms, st, &a);
            if (!failed) failed = on_16_bytes(d_W, ldw, transposed ? N : K, transposed ? K : N, &scratch, sms, st, &b);
            if (failed) return failed;
            return transposed ? launch_product_tiles<T, kCopied, true, true>(a, b, n_rows, N, K, K, 1, nullptr, out, sms, st)
                              : launch_product_tiles<T, kCopied, true, false>(a, b, n_rows, N, K, K, 1, nullptr, out, sms, st);
        } else {
            return transposed ? launch_product_tiles<T, kImage, true, true>(x, w, n_rows, N, K, K, 1, d_scratch, out, sms, st)
                              : launch_product_tiles<T, kImage, true, false>(x, w, n_rows, N, K, K, 1, d_scratch, out, sms, st);
        }
    });
}

int drone_activation_gradient_scratch(int type, int n_rows, int N, long long *n_floats) {
    DRONE_REQUIRE(DRONE_TYPE_OK(type) && DRONE_LINEAR_SIZES(n_rows, 1, N) && n_floats, "drone_activation_gradient_scratch: type=%d n_rows=%d N=%d", type, n_rows,
                  N);
    int sms = 0;
    const int rc = device_sms(&sms);
    if (rc) return rc;
    *n_floats = (long long)gradient_blocks(type, n_rows, N, sms).rows * N;
    return DRONE_OK;
}

int drone_activation_gradient(int type, int n_rows, int N, const void *d_G, int ldg, const void *d_pre, int ldp, int activation, void *d_dZ, int ldz,
                              float *d_bias_grad, float *d_scratch, long long n_scratch, void *stream) {
    DRONE_REQUIRE(DRONE_TYPE_OK(type), "drone_activation_gradient: type=%d", type);
    DRONE_REQUIRE(DRONE_LINEAR_SIZES(n_rows, 1, N), "drone_activation_gradient: n_rows=%d N=%d", n_rows, N);
    DRONE_REQUIRE(activation >= DRONE_ACT_NONE && activation <= DRONE_ACT_SILU, "drone_activation_gradient: activation=%d", activation);
    const bool reads_pre = activation != DRONE_ACT_NONE;
    DRONE_REQUIRE(ldg >= N && (!reads_pre || ldp >= N) && (!d_dZ || ldz >= N), "drone_activation_gradient: ldg=%d ldp=%d ldz=%d", ldg, ldp, ldz);
    DRONE_REQUIRE(n_rows == 0 || (d_G && (d_pre || !reads_pre)), "drone_activation_gradient: NULL argument");
    DRONE_REQUIRE(DRONE_ALIGNED(d_G, type) && DRONE_ALIGNED(d_pre, type) && DRONE_ALIGNED(d_dZ, type),
                  "drone_activation_gradient: an operand is not aligned to its type");
    cudaStream_t st = (cudaStream_t)stream;
    int sms = 0;
    const int rc = device_sms(&sms);
    if (rc) return rc;
    const GradientBlocks b = gradient_blocks(type, n_rows, N, sms);
    if (d_bias_grad) {
        const long long need = (long long)b.rows * N;
        DRONE_REQUIRE(n_scratch >= need && (need == 0 || d_scratch), "drone_activation_gradient: %lld floats of scratch, %lld needed", n_scratch, need);
    }
    if (n_rows > 0 && (d_dZ || d_bias_grad)) {
        const int launched = with_type(type, [&](auto tag) {
            using T = typename decltype(tag)::T;
            constexpr int V = kVector<T>;
            const bool vec = N % V == 0 && rows_on_16_bytes(d_G, ldg, sizeof(T)) && (!reads_pre || rows_on_16_bytes(d_pre, ldp, sizeof(T))) &&
                             (!d_dZ || rows_on_16_bytes(d_dZ, ldz, sizeof(T)));
            return with_row_shape(ceil_div(b.width, V), [&](auto shape) {
                constexpr int L = decltype(shape)::L, U = decltype(shape)::U;
                if constexpr (L == 8 || L == 32) {
                    with_activation(activation, [&](auto act) {
                        constexpr int A = decltype(act)::value;
                        auto *const kernel = vec ? activation_gradient_kernel<T, L, U, true, A> : activation_gradient_kernel<T, L, U, false, A>;
                        kernel<<<dim3(b.rows, b.columns), 256, 0, st>>>((const T *)d_G, ldg, (const T *)d_pre, ldp, n_rows, N, b.width, (T *)d_dZ, ldz,
                                                                        d_bias_grad ? d_scratch : nullptr);
                    });
                }
                DRONE_LAUNCH_CHECK("activation_gradient_kernel");
                return DRONE_OK;
            });
        });
        if (launched) return launched;
    }
    return d_bias_grad ? fold_columns(d_scratch, b.rows, N, d_bias_grad, N, nullptr, st) : DRONE_OK;
}

int drone_linear_weight_gradient_scratch(int type, int n_rows, int K, int N, const void *d_X, int ldx, const void *d_dZ, int ldz, int transposed,
                                         long long *n_floats) {
    DRONE_REQUIRE(DRONE_TYPE_OK(type) && DRONE_LINEAR_SIZES(n_rows, K, N) && (transposed == 0 || transposed == 1) && n_floats,
                  "drone_linear_weight_gradient_scratch: type=%d n_rows=%d K=%d N=%d transposed=%d", type, n_rows, K, N, transposed);
    int sms = 0;
    const int rc = device_sms(&sms);
    if (rc) return rc;
    const bool thin = thin_gradient(type, K, N), narrow = !thin && narrow_rows(K, N);
    const int shares = thin ? thin_gradient_grid(n_rows, K, N, sms).rows : narrow ? narrow_blocks(n_rows, narrow_rows_at_once(std::max(K, N), 2), sms) : product_shares(type, transposed ? N : K, transposed ? K : N, n_rows, sms).count;
    *n_floats = n_rows == 0 ? 0 : (long long)shares * K * N;
    if (type != DRONE_F32 && !narrow && !thin) *n_floats = (*n_floats + 3) / 4 * 4 + padded_floats(d_X, ldx, n_rows, K) + padded_floats(d_dZ, ldz, n_rows, N);
    return DRONE_OK;
}

int drone_linear_weight_gradient(int type, int n_rows, int K, int N, const void *d_X, int ldx, const void *d_dZ, int ldz, int transposed, void *d_dW,
                                 int ldw, float *d_scratch, long long n_scratch, void *stream) {
    DRONE_REQUIRE(DRONE_TYPE_OK(type), "drone_linear_weight_gradient: type=%d", type);
    DRONE_REQUIRE(DRONE_LINEAR_SIZES(n_rows, K, N), "drone_linear_weight_gradient: n_rows=%d K=%d N=%d", n_rows, K, N);
    DRONE_REQUIRE((transposed == 0 || transposed == 1) && ldx >= K && ldz >= N && ldw >= (transposed ? K : N),
                  "drone_linear_weight_gradient: ldx=%d ldz=%d ldw=%d transposed=%d", ldx, ldz, ldw, transposed);
    DRONE_REQUIRE(d_dW && (n_rows == 0 || (d_X && d_dZ)), "drone_linear_weight_gradient: NULL argument");
    DRONE_REQUIRE(DRONE_ALIGNED(d_X, type) && DRONE_ALIGNED(d_dZ, type) && DRONE_ALIGNED(d_dW, type),
                  "drone_linear_weight_gradient: an operand is not aligned to its type");
    cudaStream_t st = (cudaStream_t)stream;
    int sms = 0;
    const int rc = device_sms(&sms);
    if (rc) return rc;
    const int rows = transposed ? N : K, columns = transposed ? K : N;
    if (n_rows == 0) {
        DRONE_CUDA(cudaMemset2DAsync(d_dW, (size_t)ldw * type_size(type), 0, (size_t)columns * type_size(type), rows, st));
        return DRONE_OK;
    }
    const Shares s = product_shares(type, rows, columns, n_rows, sms);
    long long need = 0;
    const int sized = drone_linear_weight_gradient_scratch(type, n_rows, K, N, d_X, ldx, d_dZ, ldz, transposed, &need);
    if (sized) return sized;
    DRONE_REQUIRE(n_scratch >= need && d_scratch && (reinterpret_cast<uintptr_t>(d_scratch) & 15) == 0,
                  "drone_linear_weight_gradient: %lld floats of scratch on 16 bytes needed, %lld at %p given", need, n_scratch, (void *)d_scratch);
    return with_type(type, [&](auto tag) {
        using T = typename decltype(tag)::T;
        Operand<T> x = operand<T>(d_X, ldx), dz = operand<T>(d_dZ, ldz);
        if constexpr (sizeof(T) == 4) {
            if (thin_gradient(type, K, N)) {
                const int failed = launch_thin_gradient(x, dz, n_rows, N, K, transposed != 0, d_scratch, sms, st);
                return failed ? failed : add_product_shares<T>(d_scratch, thin_gradient_grid(n_rows, K, N, sms).rows, rows, columns, (T *)d_dW, ldw, st);
            }
        }
        if (narrow_rows(K, N)) {
            const int rows_at_once = narrow_rows_at_once(std::max(K, N), 2), blocks = narrow_blocks(n_rows, rows_at_once, sms);
            narrow_gradient_kernel<T><<<blocks, 256, 0, st>>>(x, dz, n_rows, N, K, transposed != 0, rows_at_once, d_scratch);
            DRONE_LAUNCH_CHECK("narrow_gradient_kernel");
            return add_product_shares<T>(d_scratch, blocks, rows, columns, (T *)d_dW, ldw, st);
        }
        if constexpr (sizeof(T) == 2) {
            float *scratch = d_scratch + ((long long)s.count * K * N + 3) / 4 * 4;
            int failed = on_16_bytes(d_X, ldx, n_rows, K, &scratch, sms, st, &x);
            if (!failed) failed = on_16_bytes(d_dZ, ldz, n_rows, N, &scratch, sms, st, &dz);
            if (failed) return failed;
        }
        const Operand<T> a = transposed ? dz : x, b = transposed ? x : dz;
        const LinearOut<T> out = {nullptr, DRONE_ACT_NONE, nullptr, 0, nullptr, 0, nullptr, 0, d_scratch, 1};
        constexpr Bring BRING = sizeof(T) == 2 ? kCopied : kThrough;
        const int launched = launch_product_tiles<T, BRING, false, false>(a, b, rows, columns, n_rows, s.share, s.count, nullptr, out, sms, st);
        if (launched) return launched;
        return add_product_shares<T>(d_scratch, s.count, rows, columns, (T *)d_dW, ldw, st);
    });
}

}  // extern "C"
