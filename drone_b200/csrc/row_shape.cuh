// Rows of a matrix in the registers of groups of lanes, and sums over rows: shared by the layer norm and the activations' gradients.
#pragma once

#include "dense_types.cuh"

namespace drone {

// How a row lies in the registers of its lanes: U vectors of V values a lane, or (rows that are not on 16 bytes) U * V single
// values a lane, L apart.
template <typename T, int L, int U, bool VEC>
struct RowShape {
    static constexpr int V = kVector<T>, PER = U * V, THREADS = L > 32 ? L : 256, GROUPS = THREADS / L;
    __device__ static int column(int gl, int i) { return VEC ? (gl + i / V * L) * V + i % V : gl + i * L; }
    // values beyond the row are 0
    __device__ static void load(const T *row, int F, int gl, float (&v)[PER]) {
        if (VEC) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                Values<T, V> x = {};
                if (column(gl, u * V) < F) x = *reinterpret_cast<const Values<T, V> *>(row + column(gl, u * V));
                x.get(v + u * V);
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) v[i] = column(gl, i) < F ? to_float(row[column(gl, i)]) : 0.f;
        }
    }
    __device__ static void store_vector(T *row, int F, int gl, int u, const float *v) {
        if constexpr (VEC) {
            Values<T, V> x;
            x.set(v);
            if (column(gl, u * V) < F) *reinterpret_cast<Values<T, V> *>(row + column(gl, u * V)) = x;
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (column(gl, u * V + e) < F) row[column(gl, u * V + e)] = from_float<T>(v[e]);
        }
    }
    __device__ static void store(T *row, int F, int gl, const float (&v)[PER]) {
#pragma unroll
        for (int u = 0; u < U; ++u) store_vector(row, F, gl, u, v + u * V);
    }
    __device__ static void load_vector(const float *p, int F, int gl, float (&v)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = column(gl, i) < F ? __ldg(p + column(gl, i)) : 0.f;
    }
    // The sums of a block's groups, added in order, to out[0, F).
    __device__ static void add_groups(const float (&v)[PER], int F, int gl, float *out) {
        if constexpr (GROUPS == 1) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (column(gl, i) < F) out[column(gl, i)] = v[i];
        } else {
            __shared__ float of_group[THREADS * PER];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PER; ++i) of_group[(threadIdx.x / L * PER + i) * L + gl] = v[i];
            __syncthreads();
            for (int at = threadIdx.x; at < L * PER; at += THREADS) {
                const int c = column(at % L, at / L);
                if (c >= F) continue;
                float sum = 0;
                for (int w = 0; w < GROUPS; ++w) sum += of_group[w * PER * L + at];
                out[c] = sum;
            }
        }
    }
};

// f(shape) for the lanes of a row of so many vectors: shape.L lanes with shape.U vectors each; L = 0: too wide for a block's registers.
template <int LANES, int VECTORS> struct LanesOfRow { static constexpr int L = LANES, U = VECTORS; };
template <typename F>
int with_row_shape(int vectors, const F &f) {
    if (vectors <= 8) return f(LanesOfRow<8, 1>());
    if (vectors <= 16) return f(LanesOfRow<8, 2>());
    if (vectors <= 32) return f(LanesOfRow<32, 1>());
    if (vectors <= 64) return f(LanesOfRow<32, 2>());
    if (vectors <= 128) return f(LanesOfRow<32, 4>());
    if (vectors <= 256) return f(LanesOfRow<128, 2>());
    if (vectors <= 512) return f(LanesOfRow<256, 2>());
    if (vectors <= 1024) return f(LanesOfRow<256, 4>());
    if (vectors <= 2048) return f(LanesOfRow<512, 4>());
    return f(LanesOfRow<0, 0>());
}

// Column sums from those of `blocks` blocks, sums[blocks][columns], added in order in double: the first `split` to a, the others to b
// (either may be NULL).
int fold_columns(const float *sums, int blocks, int columns, float *a, int split, float *b, cudaStream_t st);

}  // namespace drone
