// Loss and gradient of logits against a teacher's top logits, and of the labels where there are some.  With the temperature t, the
// teacher's entries (v_j, c_j) of a row and p(s) = softmax of the row's logits z over s:
//     q_j  = softmax of v_j / t over the row's entries,   soft = t^2 sum_j q_j (log q_j - log p(t)_{c_j}),   d soft / d z = t (p(t) - q)
//     hard = -log p(1)_truth,                             d hard / d z = p(1) - one-hot
// and the gradient written is  soft_weight * d soft + hard_weight * d hard.  Entries with a negative class or a value of minus infinity
// are none; a row without any has no soft part, a row that is not labelled no hard part.
//
// Bound: HBM, one read of the logits and one write of the gradient.  Both softmaxes share the row's maximum, so that a row is read
// once: a group of lanes, or for many classes a block, keeps it in registers.
#include "dense_types.cuh"

#include <algorithm>

namespace drone {

constexpr int kMaxTop = DRONE_DISTILLATION_MAX_TOP;
constexpr int kRowBlocks = DRONE_DISTILLATION_SCRATCH / 4;

// The sums of a block's rows: soft losses, rows that have one, hard losses, rows that have one.
struct LossSums {
    double soft, soft_rows, hard, hard_rows;
};

template <typename T>
struct Distillation {
    const T *logits;
    long long ld;
    const void *teacher;
    long long ldt;
    int teacher_type;
    const long long *classes_of;
    long long ldc;
    int top;
    const long long *truth;
    const unsigned char *labelled;
    float temperature, soft, hard;
    T *grad;
    long long ldg;
    LossSums *sums;
    int n, classes;
};

__device__ __forceinline__ float load_as(const void *p, long long i, int type) {
    return type == DRONE_F32 ? __ldg((const float *)p + i) : type == DRONE_BF16 ? to_float(((const __nv_bfloat16 *)p)[i]) : to_float(((const __half *)p)[i]);
}

// Entry j of a row: class (-1: none) and value over the temperature.  A class that does not exist makes the value NaN, and with it the row.
template <typename T>
__device__ __forceinline__ int teacher_entry(const Distillation<T> &p, long long row, int j, float *value) {
    const long long c = __ldg(p.classes_of + row * p.ldc + j);
    const float v = load_as(p.teacher, row * p.ldt + j, p.teacher_type);
    *value = c >= p.classes ? NAN : v / p.temperature;
    if (c < 0 || v == -INFINITY) return -1;
    return c >= p.classes ? 0 : (int)c;
}

template <int L>
__device__ __forceinline__ float max_of_lanes(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <int L, typename V>
__device__ __forceinline__ V sum_of_lanes(V v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A block's sums over its threads, in a fixed order, to sums[blockIdx.x].
template <int THREADS>
__device__ __forceinline__ void write_sums(LossSums s, LossSums *sums) {
    __shared__ LossSums of_warp[THREADS / 32];
    s.soft = sum_of_lanes<32>(s.soft);
    s.soft_rows = sum_of_lanes<32>(s.soft_rows);
    s.hard = sum_of_lanes<32>(s.hard);
    s.hard_rows = sum_of_lanes<32>(s.hard_rows);
    if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < THREADS / 32; ++w) {
            s.soft += of_warp[w].soft;
            s.soft_rows += of_warp[w].soft_rows;
            s.hard += of_warp[w].hard;
            s.hard_rows += of_warp[w].hard_rows;
        }
        sums[blockIdx.x] = s;
    }
}

// Rows of at most L * PER classes, L lanes a row.
template <typename T, int L, int PER, bool HARD>
__global__ void __launch_bounds__(256) distillation_rows_kernel(Distillation<T> p) {
    const int gl = threadIdx.x & (L - 1), classes = p.classes;
    const float t = p.temperature;
    LossSums sums = {0, 0, 0, 0};
    const long long step = (long long)gridDim.x * (256 / L), in_block = threadIdx.x / L;
    for (long long row0 = (long long)blockIdx.x * (256 / L); row0 < p.n; row0 += step) {
        const bool live = row0 + in_block < p.n;      // whole warps stay for the shuffles
        const long long row = live ? row0 + in_block : p.n - 1;
        const T *x = p.logits + row * p.ld;
        float v[PER], m = -INFINITY;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            v[u] = gl + u * L < classes ? to_float(x[gl + u * L]) : -INFINITY;
            m = fmaxf(m, v[u]);
        }
        m = max_of_lanes<L>(m);
        float s = 0, s1 = 0;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            if (gl + u * L < classes) {
                s += expf((v[u] - m) / t);
                if (HARD) s1 += expf(v[u] - m);
            }
        }
        s = sum_of_lanes<L>(s);
        // the teacher's softmax
        float tm = -INFINITY, ts = 0, value;
        int entries = 0;
        for (int j = gl; j < p.top; j += L)
            if (teacher_entry(p, row, j, &value) >= 0) {
                tm = fmaxf(tm, value);
                ++entries;
            }
        tm = max_of_lanes<L>(tm);
        entries = sum_of_lanes<L>(entries);
        for (int j = gl; j < p.top; j += L)
            if (teacher_entry(p, row, j, &value) >= 0) ts += expf(value - tm);
        ts = sum_of_lanes<L>(ts);
        const float log_s = logf(s), log_ts = logf(ts);
        float target[PER], soft = 0;
#pragma unroll
        for (int u = 0; u < PER; ++u) target[u] = 0;
        for (int j0 = 0; j0 < p.top; j0 += L) {
            int c = -1;
            float q = 0;
            if (j0 + gl < p.top) {
                c = teacher_entry(p, row, j0 + gl, &value);
                if (c >= 0) {
                    q = expf(value - tm) / ts;
                    if (q != 0.f) soft += q * ((value - tm - log_ts) - ((to_float(x[c]) - m) / t - log_s));
                }
            }
#pragma unroll
            for (int from = 0; from < L; ++from) {
                if (j0 + from >= p.top) break;
                const int c_j = __shfl_sync(0xffffffffu, c, from, L);
                const float q_j = __shfl_sync(0xffffffffu, q, from, L);
#pragma unroll
                for (int u = 0; u < PER; ++u)
                    if (c_j == gl + u * L) target[u] += q_j;
            }
        }
        soft = sum_of_lanes<L>(soft);
        float at_truth = 0, label = 0;
        long long truth = 0;
        if (HARD) {
            s1 = sum_of_lanes<L>(s1);
            truth = __ldg(p.truth + row);
            label = truth < 0 || truth >= classes ? NAN : __ldg(p.labelled + row) ? 1.f : 0.f;
            at_truth = truth < 0 || truth >= classes ? 0.f : to_float(x[truth]) - m;
        }
        __syncwarp();      // the gradient may lie on the logits, and other lanes have read this lane's
        if (!live) continue;
        T *g = p.grad + row * p.ldg;
        const float soft_weight = p.soft * t * (isnan(ts) ? NAN : 1.f);
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int c = gl + u * L;
            if (c >= classes) continue;
            float d = entries ? soft_weight * (expf((v[u] - m) / t) / s - target[u]) : 0.f;
            if (HARD && label != 0.f) d += p.hard * label * (expf(v[u] - m) / s1 - (c == truth ? 1.f : 0.f));
            g[c] = from_float<T>(d);
        }
        if (gl == 0) {
            if (entries) {
                sums.soft += (double)(t * t * soft);
                sums.soft_rows += 1;
            }
            if (HARD && label != 0.f) {
                sums.hard += (double)((logf(s1) - at_truth) * label);
                sums.hard_rows += label;
            }
        }
    }
    write_sums<256>(sums, p.sums);
}

// Maximum or sums of a block, the same in every thread.
constexpr int kBlock = 512;
__device__ __forceinline__ float block_max(float v, float *of_warp) {
    v = max_of_lanes<32>(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = v;
    __syncthreads();
    return max_of_lanes<32>(of_warp[threadIdx.x & (kBlock / 32 - 1)]);
}
__device__ __forceinline__ float block_sum(float v, float *of_warp) {
    v = sum_of_lanes<32>(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = v;
    __syncthreads();
    return sum_of_lanes<kBlock / 32>(of_warp[threadIdx.x & (kBlock / 32 - 1)]);
}

// Rows of any number of classes, a block a row.
template <typename T, bool HARD>
__global__ void __launch_bounds__(kBlock) distillation_block_kernel(Distillation<T> p) {
    __shared__ float of_warp[kBlock / 32], entry_q[kMaxTop];
    __shared__ int entry_class[kMaxTop];
    static_assert(kMaxTop <= kBlock, "an entry a thread");
    const int tid = threadIdx.x, classes = p.classes;
    const float t = p.temperature;
    LossSums sums = {0, 0, 0, 0};
    for (long long row = blockIdx.x; row < p.n; row += gridDim.x) {
        const T *x = p.logits + row * p.ld;
        T *g = p.grad + row * p.ldg;
        float m = -INFINITY;
        for (int c = tid; c < classes; c += kBlock) m = fmaxf(m, to_float(x[c]));
        m = block_max(m, of_warp);
        float s = 0, s1 = 0;
        for (int c = tid; c < classes; c += kBlock) {
            const float z = to_float(x[c]) - m;
            s += expf(z / t);
            if (HARD) s1 += expf(z);
        }
        s = block_sum(s, of_warp);
        if (HARD) s1 = block_sum(s1, of_warp);
        float value = -INFINITY, q = 0, soft = 0, z_c = 0;
        const int c_mine = tid < p.top ? teacher_entry(p, row, tid, &value) : -1;
        const float tm = block_max(c_mine >= 0 ? value : -INFINITY, of_warp);
        const float e = c_mine >= 0 ? expf(value - tm) : 0.f, ts = block_sum(e, of_warp);
        const bool any = __syncthreads_or(c_mine >= 0);
        if (c_mine >= 0) {
            q = e / ts;
            z_c = to_float(x[c_mine]) - m;
            if (q != 0.f) soft = q * ((value - tm - logf(ts)) - (z_c / t - logf(s)));
        }
        soft = block_sum(soft, of_warp);
        if (tid < p.top) {
            entry_class[tid] = c_mine;
            entry_q[tid] = q;
        }
        float label = 0, at_truth = 0;
        long long truth = -1;
        if (HARD) {
            truth = __ldg(p.truth + row);
            label = truth < 0 || truth >= classes ? NAN : __ldg(p.labelled + row) ? 1.f : 0.f;
            at_truth = truth < 0 || truth >= classes ? 0.f : to_float(x[truth]) - m;
        }
        const float soft_weight = p.soft * t * (isnan(ts) ? NAN : 1.f);
        // the gradient of a class whose logit is m + z and whose share of the teacher is q
        auto gradient = [&](float z, float q_c, bool is_truth) {
            float d = any ? soft_weight * (expf(z / t) / s - q_c) : 0.f;
            if (HARD && label != 0.f) d += p.hard * label * (expf(z) / s1 - (is_truth ? 1.f : 0.f));
            return from_float<T>(d);
        };
        // the entries of a class that is there more than once are added by the first; before the gradient, which may lie on the logits
        __syncthreads();
        bool first = c_mine >= 0;
        float q_class = 0;
        if (first)
            for (int j = 0; j < p.top; ++j)
                if (entry_class[j] == c_mine) {
                    if (j < tid) first = false;
                    q_class += entry_q[j];
                }
        for (int c = tid; c < classes; c += kBlock) g[c] = gradient(to_float(x[c]) - m, 0.f, c == truth);
        __syncthreads();
        if (first) g[c_mine] = gradient(z_c, q_class, c_mine == truth);
        if (tid == 0) {
            if (any) {
                sums.soft += (double)(t * t * soft);
                sums.soft_rows += 1;
            }
            if (HARD && label != 0.f) {
                sums.hard += (double)((logf(s1) - at_truth) * label);
                sums.hard_rows += label;
            }
        }
    }
    write_sums<kBlock>(sums, p.sums);
}

// loss[0], loss[1] = the means of the soft and of the hard losses over the rows that have one (0 where there are none)
__global__ void __launch_bounds__(256) fold_distillation_kernel(const LossSums *sums, int blocks, float *loss) {
    __shared__ LossSums total;
    LossSums s = {0, 0, 0, 0};
    for (int i = threadIdx.x; i < blocks; i += 256) {
        s.soft += sums[i].soft;
        s.soft_rows += sums[i].soft_rows;
        s.hard += sums[i].hard;
        s.hard_rows += sums[i].hard_rows;
    }
    write_sums<256>(s, &total);
    if (threadIdx.x == 0) {
        // a NaN among the numbers of rows (a label that does not exist) stays one
        loss[0] = (float)(total.soft / (total.soft_rows == 0 ? 1.0 : total.soft_rows));
        loss[1] = (float)(total.hard / (total.hard_rows == 0 ? 1.0 : total.hard_rows));
    }
}

template <typename T, bool HARD>
static int launch_distillation(const Distillation<T> &p, float *loss, cudaStream_t st) {
    const int lanes = p.classes <= 64 ? 8 : p.classes <= 256 ? 32 : 0, rows = lanes ? 256 / lanes : 1;
    const int blocks = (int)std::min<long long>(kRowBlocks, ((long long)p.n + rows - 1) / rows);
    if (p.n > 0) {
        if (p.classes <= 8) distillation_rows_kernel<T, 8, 1, HARD><<<blocks, 256, 0, st>>>(p);
        else if (p.classes <= 16) distillation_rows_kernel<T, 8, 2, HARD><<<blocks, 256, 0, st>>>(p);
        else if (p.classes <= 32) distillation_rows_kernel<T, 8, 4, HARD><<<blocks, 256, 0, st>>>(p);
        else if (p.classes <= 64) distillation_rows_kernel<T, 8, 8, HARD><<<blocks, 256, 0, st>>>(p);
        else if (p.classes <= 256) distillation_rows_kernel<T, 32, 8, HARD><<<blocks, 256, 0, st>>>(p);
        else distillation_block_kernel<T, HARD><<<blocks, kBlock, 0, st>>>(p);
        DRONE_LAUNCH_CHECK("distillation_kernel");
    }
    fold_distillation_kernel<<<1, 256, 0, st>>>(p.sums, p.n > 0 ? blocks : 0, loss);
    DRONE_LAUNCH_CHECK("fold_distillation_kernel");
    return DRONE_OK;
}

}  // namespace drone

using namespace drone;

extern "C" {

int drone_distillation_loss(int type, int n_rows, int classes, const void *d_logits, int ld, int teacher_type, int top, const void *d_teacher, int ldt,
                            const long long *d_classes, int ldc, float temperature, const long long *d_truth, const unsigned char *d_labelled,
                            float soft, float hard, void *d_grad, int ld_grad, float *d_loss, double *d_scratch, void *stream) {
    DRONE_REQUIRE(DRONE_TYPE_OK(type) && DRONE_TYPE_OK(teacher_type), "drone_distillation_loss: type=%d teacher_type=%d", type, teacher_type);
    DRONE_REQUIRE(n_rows >= 0 && classes >= 1 && ld >= classes && ld_grad >= classes, "drone_distillation_loss: n_rows=%d classes=%d ld=%d ld_grad=%d",
                  n_rows, classes, ld, ld_grad);
    DRONE_REQUIRE(top >= 1 && top <= kMaxTop && ldt >= top && ldc >= top, "drone_distillation_loss: top=%d (1..%d) ldt=%d ldc=%d", top, kMaxTop, ldt, ldc);
    DRONE_REQUIRE(temperature > 0 && temperature <= 1e30f, "drone_distillation_loss: temperature=%g", temperature);
    DRONE_REQUIRE(d_loss && d_scratch && (n_rows == 0 || (d_logits && d_teacher && d_classes && d_grad)), "drone_distillation_loss: NULL argument");
    DRONE_REQUIRE((d_truth == nullptr) == (d_labelled == nullptr), "drone_distillation_loss: d_truth and d_labelled come together");
    DRONE_REQUIRE(DRONE_ALIGNED(d_logits, type) && DRONE_ALIGNED(d_grad, type) && DRONE_ALIGNED(d_teacher, teacher_type),
                  "drone_distillation_loss: an operand is not aligned to its type");
    DRONE_REQUIRE((reinterpret_cast<uintptr_t>(d_scratch) & 7) == 0, "drone_distillation_loss: d_scratch is not 8-byte aligned");
    cudaStream_t st = (cudaStream_t)stream;
    return with_type(type, [&](auto tag) {
        using T = typename decltype(tag)::T;
        const Distillation<T> p = {(const T *)d_logits, ld, d_teacher, ldt, teacher_type, d_classes, ldc, top, d_truth, d_labelled, temperature, soft,
                                   hard, (T *)d_grad, ld_grad, (LossSums *)d_scratch, n_rows, classes};
        return d_truth ? launch_distillation<T, true>(p, d_loss, st) : launch_distillation<T, false>(p, d_loss, st);
    });
}

}  // extern "C"
