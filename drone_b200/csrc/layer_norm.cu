// Layer norm of the rows of a matrix and its backward pass: with mean m and r = 1 / sqrt(variance + eps) of a row,
//     y  = (x - m) r scale + shift                              (and a ReLU of it)
//     dx = r (h - mean(h) - xhat mean(h xhat)),   h = g scale,  xhat = (x - m) r,  g = dy (0 where the ReLU's output is not positive)
//     d_scale = sum over rows of g xhat,  d_shift = sum over rows of g.
//
// Bound: HBM, one read of every operand and one write of y or dx.  A group of L lanes holds a row in registers (16 bytes a load
// where rows allow it), so that mean, variance and the two means of the backward pass cost shuffles and no second read; the
// variance is that of the differences from the mean, in 32 bits.  The sums over rows stay in a thread's registers for all rows it
// takes, are added within the block in shared memory and over the blocks in double, always in the same order.
// us: 2.4 M rows of 256 floats with ReLU 870 (90 % of the copy rate); backward 232,965 rows of 128 floats with ReLU 83 (90 %), 98 without reading a
// row ahead; 65,537 rows of 1024 bfloat16 110 (57 %): a lane's 32 values and their two sums take 255 registers; four warps a row with a
// barrier took 150 to 162.
#include "row_shape.cuh"

#include <algorithm>

namespace drone {

// Sums of two values per lane over the L lanes of a row (L <= 32: within the warp; above: the block is the row).  Calls alternate between two buffers, so that one barrier a call is enough: nobody writes a buffer before everybody has passed the
// barrier behind its last reads.
template <int L>
__device__ __forceinline__ float2 sum_over_row(float2 v, int buffer) {
#pragma unroll
    for (int o = (L < 32 ? L : 32) / 2; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if constexpr (L > 32) {
        __shared__ float2 of_warp[2][L / 32];
        if ((threadIdx.x & 31) == 0) of_warp[buffer][threadIdx.x >> 5] = v;
        __syncthreads();
        v = of_warp[buffer][0];
#pragma unroll
        for (int w = 1; w < L / 32; ++w) {
            v.x += of_warp[buffer][w].x;
            v.y += of_warp[buffer][w].y;
        }
    }
    return v;
}

template <typename T, int L, int U, bool VEC>
__global__ void __launch_bounds__(L > 32 ? L : 256)
layer_norm_kernel(const T *x, long long ldx, const float *__restrict__ scale, const float *__restrict__ shift, int n, int F, float eps, bool relu,
                  T *y, long long ldy, float *__restrict__ mean, float *__restrict__ rstd) {
    using S = RowShape<T, L, U, VEC>;
    const int gl = threadIdx.x % L;
    float a[S::PER], b[S::PER];
    S::load_vector(scale, F, gl, a);
    S::load_vector(shift, F, gl, b);
    // whole warps stay for the shuffles: a group without a row repeats the last one and writes nothing
    const long long first = (long long)blockIdx.x * S::GROUPS, group = threadIdx.x / L, step = (long long)gridDim.x * S::GROUPS;
    for (long long row0 = first; row0 < n; row0 += step) {
        const bool live = row0 + group < n;
        const long long row = live ? row0 + group : n - 1;
        float v[S::PER];
        S::load(x + row * ldx, F, gl, v);
        float2 s = make_float2(0, 0);
#pragma unroll
        for (int i = 0; i < S::PER; ++i) s.x += v[i];
        const float m = sum_over_row<L>(s, 0).x / F;
        s.x = 0;
#pragma unroll
        for (int i = 0; i < S::PER; ++i) {
            v[i] -= m;
            if (S::column(gl, i) < F) s.x += v[i] * v[i];
        }
        const float r = 1.f / sqrtf(sum_over_row<L>(s, 1).x / F + eps);
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < S::PER; ++i) {
            v[i] = v[i] * r * a[i] + b[i];
            if (relu && v[i] < 0.f) v[i] = 0.f;
        }
        S::store(y + row * ldy, F, gl, v);
        if (gl == 0) {
            if (mean) mean[row] = m;
            if (rstd) rstd[row] = r;
        }
    }
}

// Rows too wide for the registers of a block: a block a row, read once more for each step (out of L2).
constexpr int kWideThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kWideThreads)
layer_norm_wide_kernel(const T *x, long long ldx, const float *__restrict__ scale, const float *__restrict__ shift, int n, int F, float eps, bool relu,
                       T *y, long long ldy, float *__restrict__ mean, float *__restrict__ rstd) {
    for (long long row = blockIdx.x; row < n; row += gridDim.x) {
        const T *in = x + row * ldx;
        T *out = y + row * ldy;
        float2 s = make_float2(0, 0);
        for (int c = threadIdx.x; c < F; c += kWideThreads) s.x += to_float(in[c]);
        const float m = sum_over_row<kWideThreads>(s, 0).x / F;
        s.x = 0;
        for (int c = threadIdx.x; c < F; c += kWideThreads) {
            const float d = to_float(in[c]) - m;
            s.x += d * d;
        }
        const float r = 1.f / sqrtf(sum_over_row<kWideThreads>(s, 1).x / F + eps);
        for (int c = threadIdx.x; c < F; c += kWideThreads) {
            const float z = (to_float(in[c]) - m) * r * __ldg(scale + c) + __ldg(shift + c);
            out[c] = from_float<T>(relu && z < 0.f ? 0.f : z);
        }
        if (threadIdx.x == 0) {
            if (mean) mean[row] = m;
            if (rstd) rstd[row] = r;
        }
    }
}

// What both forms of the backward pass read and write; sums[block] = {d_scale[F], d_shift[F]} of the block's rows.
template <typename T>
struct NormBackward {
    const T *g, *x, *out;
    long long ldg, ldx, ldo;
    const float *scale, *mean, *rstd;
    const int *mirror2worker;      // rows with an entry other than -1 are left out of the sums
    T *dx;
    long long ld;
    float *sums;
    int n, F;
};

template <typename T, int L, int U, bool VEC>
__global__ void __launch_bounds__(L > 32 ? L : 256) layer_norm_backward_kernel(NormBackward<T> p) {
    using S = RowShape<T, L, U, VEC>;
    const int gl = threadIdx.x % L, F = p.F;
    float a[S::PER], d_scale[S::PER], d_shift[S::PER];
    S::load_vector(p.scale, F, gl, a);
#pragma unroll
    for (int i = 0; i < S::PER; ++i) d_scale[i] = d_shift[i] = 0;
    const long long first = (long long)blockIdx.x * S::GROUPS, group = threadIdx.x / L, step = (long long)gridDim.x * S::GROUPS;
    // what a row reads, one row ahead where the registers allow it
    constexpr bool AHEAD = S::PER <= 8;
    struct Row {
        float g[S::PER], x[S::PER], o[AHEAD ? S::PER : 1], m, r;
        bool counts;
    };
    auto read = [&](Row &to, long long row0) {
        const long long row = row0 + group < p.n ? row0 + group : p.n - 1;      // whole warps stay for the shuffles
        S::load(p.g + row * p.ldg, F, gl, to.g);
        S::load(p.x + row * p.ldx, F, gl, to.x);
        if (p.out) {
            if constexpr (AHEAD) {
                S::load(p.out + row * p.ldo, F, gl, to.o);
            } else {
                float o[S::PER];
                S::load(p.out + row * p.ldo, F, gl, o);
#pragma unroll
                for (int i = 0; i < S::PER; ++i) to.g[i] = o[i] > 0.f ? to.g[i] : 0.f;
            }
        }
        to.m = __ldg(p.mean + row);
        to.r = __ldg(p.rstd + row);
        to.counts = row0 + group < p.n && (!p.mirror2worker || __ldg(p.mirror2worker + row) == -1);
    };
    Row next;
    if (AHEAD && first < p.n) read(next, first);
    int buffer = 0;
    for (long long row0 = first; row0 < p.n; row0 += step, buffer ^= 1) {
        const bool live = row0 + group < p.n;
        Row now;
        if (AHEAD) {
            now = next;
            if (row0 + step < p.n) read(next, row0 + step);
        } else {
            read(now, row0);
        }
        float2 s = make_float2(0, 0);
#pragma unroll
        for (int i = 0; i < S::PER; ++i) {
            float g = now.g[i];
            if (AHEAD && p.out) g = now.o[AHEAD ? i : 0] > 0.f ? g : 0.f;
            const float hat = S::column(gl, i) < F ? (now.x[i] - now.m) * now.r : 0.f;
            if (now.counts) {
                d_scale[i] += g * hat;
                d_shift[i] += g;
            }
            now.x[i] = hat;
            now.g[i] = g * a[i];
            s.x += now.g[i];
            s.y += now.g[i] * hat;
        }
        s = sum_over_row<L>(s, buffer);
        s.x /= F;
        s.y /= F;
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < S::PER; ++i) now.g[i] = now.r * (now.g[i] - s.x - now.x[i] * s.y);
        S::store(p.dx + (row0 + group) * p.ld, F, gl, now.g);
    }
    float *of_block = p.sums + (long long)blockIdx.x * 2 * F;
    S::add_groups(d_scale, F, gl, of_block);
    S::add_groups(d_shift, F, gl, of_block + F);
}

template <typename T>
__global__ void __launch_bounds__(kWideThreads) layer_norm_backward_wide_kernel(NormBackward<T> p) {
    const int F = p.F;
    float *d_scale = p.sums + (long long)blockIdx.x * 2 * F, *d_shift = d_scale + F;      // a thread always has the same columns
    for (int c = threadIdx.x; c < F; c += kWideThreads) d_scale[c] = d_shift[c] = 0;
    int buffer = 0;
    for (long long row = blockIdx.x; row < p.n; row += gridDim.x, buffer ^= 1) {
        const T *in = p.x + row * p.ldx, *dy = p.g + row * p.ldg, *out = p.out ? p.out + row * p.ldo : nullptr;
        const float m = __ldg(p.mean + row), r = __ldg(p.rstd + row);
        const bool counts = !p.mirror2worker || __ldg(p.mirror2worker + row) == -1;
        float2 s = make_float2(0, 0);
        for (int c = threadIdx.x; c < F; c += kWideThreads) {
            const float g = out && !(to_float(out[c]) > 0.f) ? 0.f : to_float(dy[c]), h = (to_float(in[c]) - m) * r;
            if (counts) {
                d_scale[c] += g * h;
                d_shift[c] += g;
            }
            s.x += g * __ldg(p.scale + c);
            s.y += g * __ldg(p.scale + c) * h;
        }
        s = sum_over_row<kWideThreads>(s, buffer);
        for (int c = threadIdx.x; c < F; c += kWideThreads) {
            const float g = out && !(to_float(out[c]) > 0.f) ? 0.f : to_float(dy[c]), h = (to_float(in[c]) - m) * r;
            p.dx[row * p.ld + c] = from_float<T>(r * (g * __ldg(p.scale + c) - s.x / F - h * (s.y / F)));
        }
    }
}

struct NormGrid {
    int groups, blocks;      // rows a block takes at once; blocks
};
static NormGrid norm_grid(int type, int n, int F, int sms, int threads_per_sm) {
    const int V = type == DRONE_F32 ? 4 : 8, vectors = ceil_div(F, V);
    NormGrid g;
    g.groups = vectors <= 16 ? 32 : vectors <= 128 ? 8 : 1;
    const int threads = vectors <= 128 ? 256 : vectors <= 256 ? 128 : vectors <= 1024 ? 256 : 512;
    g.blocks = (int)std::min<long long>(((long long)n + g.groups - 1) / g.groups, (long long)sms * (threads_per_sm / threads));
    return g;
}
// of the blocks: all that the registers hold at the shapes of most rows
constexpr int kForwardThreadsPerSm = 2048, kBackwardThreadsPerSm = 1024;

}  // namespace drone

using namespace drone;

extern "C" {

int drone_layer_norm(int type, int n_rows, int F, const void *d_X, int ldx, const float *d_scale, const float *d_shift, float eps, int relu, void *d_Y,
                     int ldy, float *d_mean, float *d_rstd, void *stream) {
    DRONE_REQUIRE(DRONE_TYPE_OK(type), "drone_layer_norm: type=%d", type);
    DRONE_REQUIRE(n_rows >= 0 && F >= 1 && F <= DRONE_NORM_MAX_WIDTH && ldx >= F && ldy >= F && eps > 0 && (relu == 0 || relu == 1),
                  "drone_layer_norm: n_rows=%d F=%d ldx=%d ldy=%d eps=%g relu=%d", n_rows, F, ldx, ldy, eps, relu);
    if (n_rows == 0) return DRONE_OK;
    DRONE_REQUIRE(d_X && d_scale && d_shift && d_Y, "drone_layer_norm: NULL argument");
    DRONE_REQUIRE(DRONE_ALIGNED(d_X, type) && DRONE_ALIGNED(d_Y, type), "drone_layer_norm: an operand is not aligned to its type");
    cudaStream_t st = (cudaStream_t)stream;
    int sms = 0, rc = device_sms(&sms);
    if (rc) return rc;
    const int blocks = norm_grid(type, n_rows, F, sms, kForwardThreadsPerSm).blocks;
    return with_type(type, [&](auto tag) {
        using T = typename decltype(tag)::T;
        constexpr int V = kVector<T>;
        const bool vec = F % V == 0 && rows_on_16_bytes(d_X, ldx, sizeof(T)) && rows_on_16_bytes(d_Y, ldy, sizeof(T));
        return with_row_shape(ceil_div(F, V), [&](auto shape) {
            constexpr int L = decltype(shape)::L, U = decltype(shape)::U;
            auto launch = [&](auto kernel, int threads) {
                kernel<<<blocks, threads, 0, st>>>((const T *)d_X, ldx, d_scale, d_shift, n_rows, F, eps, relu != 0, (T *)d_Y, ldy, d_mean, d_rstd);
            };
            if constexpr (L == 0) launch(layer_norm_wide_kernel<T>, kWideThreads);
            else if (vec) launch(layer_norm_kernel<T, L, U, true>, L > 32 ? L : 256);
            else launch(layer_norm_kernel<T, L, U, false>, L > 32 ? L : 256);
            DRONE_LAUNCH_CHECK("layer_norm_kernel");
            return DRONE_OK;
        });
    });
}

int drone_layer_norm_backward_scratch(int type, int n_rows, int F, long long *n_floats) {
    DRONE_REQUIRE(DRONE_TYPE_OK(type) && n_rows >= 0 && F >= 1 && F <= DRONE_NORM_MAX_WIDTH && n_floats,
                  "drone_layer_norm_backward_scratch: type=%d n_rows=%d F=%d", type, n_rows, F);
    int sms = 0;
    const int rc = device_sms(&sms);
    if (rc) return rc;
    *n_floats = 2LL * F * norm_grid(type, n_rows, F, sms, kBackwardThreadsPerSm).blocks;
    return DRONE_OK;
}

int drone_layer_norm_backward(int type, int n_rows, int F, const void *d_G, int ldg, const void *d_X, int ldx, const float *d_scale,
                              const float *d_mean, const float *d_rstd, const void *d_out, int ldo, const int *d_mirror2worker, void *d_dX, int ld,
                              float *d_scale_grad, float *d_shift_grad, float *d_scratch, long long n_scratch, void *stream) {
    DRONE_REQUIRE(DRONE_TYPE_OK(type), "drone_layer_norm_backward: type=%d", type);
    DRONE_REQUIRE(n_rows >= 0 && F >= 1 && F <= DRONE_NORM_MAX_WIDTH && ldg >= F && ldx >= F && ld >= F && (!d_out || ldo >= F),
                  "drone_layer_norm_backward: n_rows=%d F=%d ldg=%d ldx=%d ldo=%d ld=%d", n_rows, F, ldg, ldx, ldo, ld);
    DRONE_REQUIRE(n_rows == 0 || (d_G && d_X && d_scale && d_mean && d_rstd && d_dX), "drone_layer_norm_backward: NULL argument");
    DRONE_REQUIRE(DRONE_ALIGNED(d_G, type) && DRONE_ALIGNED(d_X, type) && DRONE_ALIGNED(d_out, type) && DRONE_ALIGNED(d_dX, type),
                  "drone_layer_norm_backward: an operand is not aligned to its type");
    cudaStream_t st = (cudaStream_t)stream;
    int sms = 0, rc = device_sms(&sms);
    if (rc) return rc;
    const int blocks = norm_grid(type, n_rows, F, sms, kBackwardThreadsPerSm).blocks;
    const long long need = 2LL * F * blocks;
    DRONE_REQUIRE(n_scratch >= need && (need == 0 || d_scratch), "drone_layer_norm_backward: %lld floats of scratch, %lld needed", n_scratch, need);
    if (n_rows > 0) {
        rc = with_type(type, [&](auto tag) {
            using T = typename decltype(tag)::T;
            constexpr int V = kVector<T>;
            const bool vec = F % V == 0 && rows_on_16_bytes(d_G, ldg, sizeof(T)) && rows_on_16_bytes(d_X, ldx, sizeof(T)) &&
                             rows_on_16_bytes(d_dX, ld, sizeof(T)) && (!d_out || rows_on_16_bytes(d_out, ldo, sizeof(T)));
            const NormBackward<T> p = {(const T *)d_G, (const T *)d_X, (const T *)d_out, ldg, ldx, ldo, d_scale, d_mean, d_rstd, d_mirror2worker,
                                       (T *)d_dX, ld, d_scratch, n_rows, F};
            return with_row_shape(ceil_div(F, V), [&](auto shape) {
                constexpr int L = decltype(shape)::L, U = decltype(shape)::U;
                if constexpr (L == 0) layer_norm_backward_wide_kernel<T><<<blocks, kWideThreads, 0, st>>>(p);
                else if (vec) layer_norm_backward_kernel<T, L, U, true><<<blocks, L > 32 ? L : 256, 0, st>>>(p);
                else layer_norm_backward_kernel<T, L, U, false><<<blocks, L > 32 ? L : 256, 0, st>>>(p);
                DRONE_LAUNCH_CHECK("layer_norm_backward_kernel");
                return DRONE_OK;
            });
        });
        if (rc) return rc;
    }
    if (!d_scale_grad && !d_shift_grad) return DRONE_OK;
    return fold_columns(d_scratch, blocks, 2 * F, d_scale_grad, F, d_shift_grad, st);
}

}  // extern "C"
