// Products whose weights are a few rows or columns, Y = activation(X W + bias) + residual with N or K of at most 4, and their weight gradients: each value
// of the long operand meets a few others, so that nothing is to be gained from tiles, of which most would be empty.
//
//   few columns   a warp has some rows, its lanes every 32nd k; W lies in shared memory as floats, the lanes' sums are added by shuffles
//   short rows    (floats) a warp has some rows and up to 128 columns, W's values of them in its registers
//   gradient      (floats) the same of the wide operand, whose values are added up over a block's rows for each of the thin one's; shares[block]
//
// Bound: HBM, the long operand read or written once: 60 M floats in 45 us where two columns are formed of rows of 256 (83 % of the copy rate), in 59 in the gradient of
// 125,523 x 1 x 477; 100 M written in 97 us from rows of one value to 256 (64 %).
#pragma once

#include "product_tile.cuh"

namespace drone {

constexpr int kThinWeights = 8192, kThinSums = 16;      // floats of W in shared memory, sums of a lane

template <typename T, int ACTIVATION>
__device__ __forceinline__ void put_value(const LinearOut<T> &out, long long row, int c, float z) {
    if (out.bias) z += __ldg(out.bias + c);
    if (out.pre) out.pre[row * out.ldp + c] = from_float<T>(z);
    out.y[row * out.ldy + c] = from_float<T>(activate<T, ACTIVATION>(z, out.residual ? to_float(out.residual[row * out.ldr + c]) : 0.f));
}

// C: N rounded up to a power of two
template <typename T, int C>
__global__ void __launch_bounds__(256, 4) few_columns_kernel(Operand<T> X, Operand<T> W, bool transposed, int n, int N, int K, LinearOut<T> out) {
    constexpr int R = kThinSums / C;      // rows at once
    __shared__ float w[kThinWeights];
    for (int c = 0; c < C; ++c)
        for (int k = threadIdx.x; k < K; k += 256) w[c * K + k] = c < N ? to_float(W.at[transposed ? c * W.ld + k : k * W.ld + c]) : 0.f;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    with_activation(out.activation, [&](auto act) {
        for (long long row0 = (blockIdx.x * 8LL + (threadIdx.x >> 5)) * R; row0 < n; row0 += gridDim.x * 8LL * R) {
            const T *x = X.at + row0 * X.ld;
            const int rows = (int)min((long long)R, n - row0);
            float sum[kThinSums];
#pragma unroll
            for (int i = 0; i < kThinSums; ++i) sum[i] = 0;
            auto add = [&](auto whole) {      // rows that do not exist read the last one
#pragma unroll(R >= 16 ? 1 : R >= 8 ? 2 : 4)
                for (int k = lane; k < K; k += 32) {
                    float v[R];
#pragma unroll
                    for (int r = 0; r < R; ++r) v[r] = to_float(x[(decltype(whole)::value ? r : min(r, rows - 1)) * X.ld + k]);
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        const float of = w[c * K + k];
#pragma unroll
                        for (int r = 0; r < R; ++r) sum[r * C + c] = fmaf(v[r], of, sum[r * C + c]);
                    }
                }
            };
            if (rows == R) add(std::true_type());
            else add(std::false_type());
            // half of the lanes go on with half of the sums, until each has one
#pragma unroll
            for (int o = 16, left = kThinSums; o > 0; o >>= 1, left = left > 1 ? left / 2 : 1) {
                if (left > 1) {
#pragma unroll
                    for (int i = 0; i < left / 2; ++i) {
                        const bool upper = lane & o;
                        const float keep = upper ? sum[i + left / 2] : sum[i], other = upper ? sum[i] : sum[i + left / 2];
                        sum[i] = keep + __shfl_xor_sync(0xffffffffu, other, o);
                    }
                } else {
                    sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], o);
                }
            }
            constexpr int EACH = 32 / kThinSums;      // lanes with the same sum
            const int r = lane / EACH / C, c = lane / EACH % C;
            if (lane % EACH == 0 && r < rows && c < N) put_value<T, decltype(act)::value>(out, row0 + r, c, sum[0]);
        }
    });
}

// A warp has some rows, four at once, and 128 columns at most, its lanes every 32nd of them: what they read of X serves four outputs.
// S: K rounded up to a power of two
template <int S>
__global__ void __launch_bounds__(256) short_rows_kernel(Operand<float> X, Operand<float> W, bool transposed, int n, int N, int K, int width, LinearOut<float> out) {
    constexpr int AT_ONCE = 4, EACH = 4;
    const int c0 = blockIdx.y * width + (threadIdx.x & 31), limit = min(N, ((int)blockIdx.y + 1) * width);
    float w[EACH][S], b[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int c = c0 + i * 32;
#pragma unroll
        for (int k = 0; k < S; ++k) w[i][k] = k < K && c < limit ? W.at[transposed ? c * W.ld + k : k * W.ld + c] : 0.f;
        b[i] = out.bias && c < limit ? __ldg(out.bias + c) : 0.f;
    }
    const long long step = gridDim.x * 8LL;
    with_activation(out.activation, [&](auto act) {
        for (long long row0 = blockIdx.x * 8LL + (threadIdx.x >> 5); row0 < n; row0 += step * AT_ONCE) {
            float x[AT_ONCE][S], added[AT_ONCE][EACH];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const long long row = min(row0 + u * step, n - 1LL);      // a row that does not exist reads the last one
#pragma unroll
                for (int k = 0; k < S; ++k) x[u][k] = k < K ? X.at[row * X.ld + k] : 0.f;
#pragma unroll
                for (int i = 0; i < EACH; ++i) added[u][i] = out.residual && c0 + i * 32 < limit ? out.residual[row * out.ldr + c0 + i * 32] : 0.f;
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const long long row = row0 + u * step;
                if (row >= n) break;
#pragma unroll
                for (int i = 0; i < EACH; ++i) {
                    const int c = c0 + i * 32;
                    if (c >= limit) break;
                    float z = 0;
#pragma unroll
                    for (int k = 0; k < S; ++k) z = fmaf(x[u][k], w[i][k], z);
                    z += b[i];
                    if (out.pre) out.pre[row * out.ldp + c] = z;
                    out.y[row * out.ldy + c] = activate<float, decltype(act)::value>(z, added[u][i]);
                }
            }
        }
    });
}

// thin [n, S] and wide [n, columns]: shares[block][s * apart_s + c * apart_c] = the sums of thin[r, s] wide[r, c] over the block's rows.  A warp has some rows, four at
// once, and 128 columns at most.  S: rounded up to a power of two
template <int S>
__global__ void __launch_bounds__(256) thin_gradient_kernel(Operand<float> thin, Operand<float> wide, int n, int count, int columns, int width, int apart_s, int apart_c, float *shares) {
    constexpr int AT_ONCE = 4, EACH = 4;
    __shared__ float of_warp[8][S][EACH * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = blockIdx.y * width, limit = min(columns - c0, width);
    float sum[S][EACH];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < EACH; ++i) sum[s][i] = 0;
    const long long step = gridDim.x * 8LL;
    for (long long row0 = blockIdx.x * 8LL + warp; row0 < n; row0 += step * AT_ONCE) {
        float a[AT_ONCE][S], b[AT_ONCE][EACH];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const long long row = row0 + u * step;
            const bool live = row < n;
#pragma unroll
            for (int i = 0; i < EACH; ++i) b[u][i] = live && lane + i * 32 < limit ? wide.at[row * wide.ld + c0 + lane + i * 32] : 0.f;
#pragma unroll
            for (int s = 0; s < S; ++s) a[u][s] = live && s < count ? thin.at[row * thin.ld + s] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < EACH; ++i) sum[s][i] = fmaf(a[u][s], b[u][i], sum[s][i]);
    }
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < EACH; ++i) of_warp[warp][s][lane + i * 32] = sum[s][i];
    __syncthreads();
    for (int at = threadIdx.x; at < S * EACH * 32; at += 256) {
        const int s = at / (EACH * 32), c = at % (EACH * 32);
        if (c >= limit || s >= count) continue;
        float all = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) all += of_warp[w][s][c];
        shares[(long long)blockIdx.x * count * columns + (long long)s * apart_s + (long long)(c0 + c) * apart_c] = all;
    }
}

// f(std::integral_constant) of the power of two that this many values, 4 at most, are rounded up to
template <typename F>
void with_thin(int values, const F &f) {
    if (values == 1) f(std::integral_constant<int, 1>());
    else if (values == 2) f(std::integral_constant<int, 2>());
    else f(std::integral_constant<int, 4>());
}

// Where that is faster than tiles, and than the narrow kernels, which read shared memory twice a product: us here / there.
// Few columns, bias and ReLU: floats 461,538 x 130 x 1 49 / 118, 234,375 x 256 x 2 45 / 76, 100,000 x 600 x 3 53 / 100, 14,648 x 4096 x 2 55 / 90, but 7,324 x 8192 x 1 185 / 164 (too few
// warps); 600,000 x 100 x 4 137 / 123, 234,375 x 256 x 5 125 / 78; bfloat16 39 / 185, 37 / 64, 47 / 109, 52 / 45, 145 / 57; 137 / 168, 122 / 80.
// Narrow, floats without an epilogue: 465,116 x 128 x 1 64 / 182, 1.8 M x 32 x 1 71 / 173, 3.5 M x 16 x 1 130 / 177, 1.8 M x 32 x 2 132 / 180, but 6.7 M x 8 x 1 238 / 188, 3.3 M x
// 16 x 2 243 / 179; bfloat16 within 10 of these.
inline bool few_columns(int K, int N) { return N <= 2 ? K >= 16 * N && 2 * K <= kThinWeights : N <= 4 && K >= 128 && 4 * K <= kThinWeights; }
// Short rows, floats without an epilogue, and with bias, GELU and residual: 763,358 x 1 x 131 224 / 376, 319 / 869; 390,625 x 3 x 256 130 / 162, 222 / 331; 2.3 M x 4 x 43
// 290 / 329, 480 / 645; but 1.6 M x 5 x 64 280 / 214, 432 / 367; 16 bits, a column a thread, 458,015 x 1 x 131 with residual 404 / 256.
// Narrow: 465,116 x 1 x 128 60 / 161, 109 / 293; 1.8 M x 1 x 32 144 / 164, 222 / 268; 1.7 M x 3 x 32 178 / 180, 285 / 273; but 3.5 M x 1 x 16 270 / 172.
inline bool short_rows(int type, int K, int N) { return type == DRONE_F32 && K <= 4 && N >= 32; }
// Gradients: floats 125,523 x 1 x 477 59 / 154, 230,769 x 4 x 256 75 / 107, 99,833 x 600 x 1 56 / 129, 99,337 x 600 x 4 74 / 114; bfloat16 142 / 86, 154 / 37, 96 / 45, 152 / 45.
// Narrow: floats 465,116 x 1 x 128 66 / 311, 3.5 M x 1 x 16 215 / 306, 3.2 M x 3 x 16 332 / 324, but 6.7 M x 1 x 8 390 / 313.
inline bool thin_gradient(int type, int K, int N) { return type == DRONE_F32 && (K <= 4 || N <= 4) && (K >= 16 || N >= 16); }

template <typename T>
int launch_few_columns(const Operand<T> &x, const Operand<T> &w, bool transposed, int n, int N, int K, const LinearOut<T> &out, int sms, cudaStream_t st) {
    with_thin(N, [&](auto columns) {
        constexpr int C = decltype(columns)::value, ROWS = 8 * kThinSums / C;
        few_columns_kernel<T, C><<<(int)std::min<long long>(((long long)n + ROWS - 1) / ROWS, sms * 4), 256, 0, st>>>(x, w, transposed, n, N, K, out);
    });
    DRONE_LAUNCH_CHECK("few_columns_kernel");
    return DRONE_OK;
}

// Of the other two: columns of a block, blocks along them, blocks along the rows (of a gradient as many as there are shares), a warp of which has so many at least.
struct ThinGrid {
    int width, columns, rows;
    ThinGrid(int n, int wide, int of_warp, int blocks_per_sm, int sms) : columns(ceil_div(wide, 128)) {
        width = ceil_div(wide, columns);
        rows = (int)std::max<long long>(1, std::min<long long>(((long long)n + 8 * of_warp - 1) / (8 * of_warp), std::max(1, sms * blocks_per_sm / columns)));
    }
};
inline int launch_short_rows(const Operand<float> &x, const Operand<float> &w, bool transposed, int n, int N, int K, const LinearOut<float> &out, int sms, cudaStream_t st) {
    const ThinGrid g(n, N, 1, 8, sms);
    with_thin(K, [&](auto values) { short_rows_kernel<decltype(values)::value><<<dim3(g.rows, g.columns), 256, 0, st>>>(x, w, transposed, n, N, K, g.width, out); });
    DRONE_LAUNCH_CHECK("short_rows_kernel");
    return DRONE_OK;
}
inline ThinGrid thin_gradient_grid(int n, int K, int N, int sms) { return ThinGrid(n, std::max(K, N), 4, 6, sms); }
inline int launch_thin_gradient(const Operand<float> &x, const Operand<float> &dz, int n, int N, int K, bool transposed, float *shares, int sms, cudaStream_t st) {
    const bool short_k = K <= N;      // dW[k, c], or with `transposed` [c, k]
    const Operand<float> &thin = short_k ? x : dz, &wide = short_k ? dz : x;
    const int apart_k = transposed ? 1 : N, apart_n = transposed ? K : 1, apart_s = short_k ? apart_k : apart_n, apart_c = short_k ? apart_n : apart_k;
    const ThinGrid g = thin_gradient_grid(n, K, N, sms);
    const dim3 grid(g.rows, g.columns);
    with_thin(std::min(K, N), [&](auto values) {
        thin_gradient_kernel<decltype(values)::value><<<grid, 256, 0, st>>>(thin, wide, n, std::min(K, N), std::max(K, N), g.width, apart_s, apart_c, shares);
    });
    DRONE_LAUNCH_CHECK("thin_gradient_kernel");
    return DRONE_OK;
}

}  // namespace drone
