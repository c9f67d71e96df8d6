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
constexpr int kRowBlocks = DRONE_DISTILLATION_SCRATCH / 4;      // eight for each of 148 SMs; the results are right for any number

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

// Entry j of a row: class (-1: none) and value.  (Over the temperature only as a difference from the largest: the quotient of a value at either end of its
// type need not be a float.)  A class that does not exist makes the value NaN, and with it the row.
template <typename T>
__device__ __forceinline__ int teacher_entry(const Distillation<T> &p, long long row, int j, float *value) {
    const long long c = __ldg(p.classes_of + row * p.ldc + j);
    const float v = load_as(p.teacher, row * p.ldt + j, p.teacher_type);
    *value = c >= p.classes ? NAN : v;
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

// Exponentials are exp2_fast of (z - the row's maximum) log2(e) / t, whose rounding is off by as much.  (The difference comes first: a row whose
// logits are all the type's lowest value is a row of equal ones, and what all of them have in common leaves no rounding behind.  One multiply-add on
// the maximum times log2(e) / t would leave 2^-24 of that product in the exponent: 2.7e-5 of a share at logits around 1000.)
constexpr float kLog2e = 1.44269504f;
__device__ __forceinline__ float log_fast(float x) {      // off by 2^-22 and 2^-22 of the value
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y * 0.693147181f;
}

// A sum of floats with what its additions cut off.
struct LongSum {
    float sum = 0, lost = 0;
    __device__ __forceinline__ void add(float x) {
        x -= lost;
        const float now = sum + x;
        lost = fabsf(now) < INFINITY ? (now - sum) - x : 0.f;
        sum = now;
    }
};

// Rows of (PER - 1) * L + 1 to PER * L classes, L lanes a row: logits and exponentials stay in registers, the teacher's shares are added up in
// shared memory, where the lane of an entry finds its class.
// 2.4 M rows of 47 classes, 8 entries, labels: 1.18 GB in 344 us (53 % of the copy rate; instructions, and the round trips of a row's
// reductions); with 74 registers instead of 64 421; as exponentials by division and expf, computed twice, and every entry shown to every
// lane 1171 us.
template <typename T, int L, int PER, bool HARD>
__global__ void __launch_bounds__(256, 4) distillation_rows_kernel(Distillation<T> p) {
    constexpr int ROWS = 32 / L;      // of a warp
    __shared__ float shares[8][ROWS][L * PER];
    const int gl = threadIdx.x & (L - 1), classes = p.classes, lane = threadIdx.x & 31;
    const unsigned group = (L < 32 ? (1u << L) - 1 : 0xffffffffu) << (lane & ~(L - 1));
    float *const target = shares[threadIdx.x >> 5][lane / L];
#pragma unroll
    for (int u = 0; u < PER; ++u) target[gl + u * L] = 0;
    __syncwarp();
    const float t = p.temperature, scale = kLog2e / t;
    LongSum soft_sum, hard_sum;
    float soft_rows = 0, hard_rows = 0;      // of this group: fewer than 2^24
    auto inside = [&](int u) { return u < PER - 1 || gl + u * L < classes; };
    const long long step = (long long)gridDim.x * (256 / L), in_block = threadIdx.x / L;
    // logits, label and the first L entries of a row, read while the row before is worked on
    float next[PER], next_value = 0;
    int next_class = -1, next_truth = 0;
    bool next_labelled = false;
    auto read = [&](long long row0) {
        const long long row = row0 + in_block < p.n ? row0 + in_block : p.n - 1;      // whole warps stay for the shuffles
        next_class = gl < p.top ? teacher_entry(p, row, gl, &next_value) : -1;
        if (HARD) {
            const long long c = __ldg(p.truth + row);
            next_truth = c >= 0 && c < classes ? (int)c : -1;
            next_labelled = __ldg(p.labelled + row) != 0;
        }
#pragma unroll
        for (int u = 0; u < PER; ++u) next[u] = inside(u) ? to_float(p.logits[row * p.ld + gl + u * L]) : -INFINITY;
    };
    if ((long long)blockIdx.x * (256 / L) < p.n) read((long long)blockIdx.x * (256 / L));
    for (long long row0 = (long long)blockIdx.x * (256 / L); row0 < p.n; row0 += step) {
        const bool live = row0 + in_block < p.n, labelled = next_labelled;
        const long long row = live ? row0 + in_block : p.n - 1;
        const T *x = p.logits + row * p.ld;
        const int c0 = next_class, truth = next_truth;      // of the first L entries
        const float value0 = next_value;
        float v[PER], e[PER], m = -INFINITY, value;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            v[u] = next[u];
            m = fmaxf(m, v[u]);
        }
        if (row0 + step < p.n) read(row0 + step);
        bool some = c0 >= 0;
        float tm = some ? value0 : -INFINITY;
        for (int j = L + gl; j < p.top; j += L)
            if (teacher_entry(p, row, j, &value) >= 0) {
                tm = fmaxf(tm, value);
                some = true;
            }
        some = (__ballot_sync(0xffffffffu, some) & group) != 0;
        m = max_of_lanes<L>(m);
        tm = max_of_lanes<L>(tm);
        float s = 0, s1 = 0, ts = 0, apart = 0;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const float z = v[u] - m;
            e[u] = inside(u) ? exp2_fast(z * scale) : 0.f;
            s += e[u];
            if (HARD) {
                v[u] = inside(u) ? exp2_fast(z * kLog2e) : 0.f;      // from here on
                s1 += v[u];
            }
        }
        // the weight of an entry in the teacher's softmax, and its part of the distance, times the temperature
        auto weigh = [&](int c, float of) {
            if (c < 0) return 0.f;
            const float w = exp2_fast((of - tm) * scale);
            ts += w;
            if (w != 0.f) apart += w * ((of - tm) - (to_float(x[c]) - m));
            return w;
        };
        const float weight0 = weigh(c0, value0);
        for (int j = L + gl; j < p.top; j += L) {
            const int c = teacher_entry(p, row, j, &value);
            weigh(c, value);
        }
        s = sum_of_lanes<L>(s);
        ts = sum_of_lanes<L>(ts);
        apart = sum_of_lanes<L>(apart);
        float at_truth = 0, label = 0, per_s1 = 0;
        if (HARD) {
            s1 = sum_of_lanes<L>(s1);
            per_s1 = reciprocal_fast(s1);
            label = !labelled ? 0.f : truth < 0 ? NAN : 1.f;
            at_truth = truth < 0 ? 0.f : to_float(x[truth]) - m;
        }
        const float per_ts = reciprocal_fast(ts), soft_weight = some ? p.soft * t * (isnan(ts) ? NAN : 1.f) : 0.f, hard_weight = label != 0.f ? p.hard * label : 0.f;
        // What the gradient loses at the classes of entries, and of the label.  A lane puts its entry's share at its class, where its number says
        // first whether another lane has the same class: then each adds up the shares of all of them.
        auto share = [&](int c, float w) {
            float q = soft_weight * (w * per_ts);
            const float before = c >= 0 ? target[c] : 0.f;
            __syncwarp();
            if (c >= 0) target[c] = __int_as_float(lane);
            __syncwarp();
            if (__any_sync(0xffffffffu, c >= 0 && __float_as_int(target[c]) != lane)) {
                float sum = 0;
#pragma unroll 1
                for (int from = 0; from < L; ++from) {
                    const int other_c = __shfl_sync(0xffffffffu, c, from, L);
                    const float other_q = __shfl_sync(0xffffffffu, q, from, L);
                    if (other_c == c) sum += other_q;
                }
                q = sum;
            }
            __syncwarp();
            if (c >= 0) target[c] = before + q;
            __syncwarp();
        };
        share(c0, weight0);
        for (int j0 = L; j0 < p.top; j0 += L) {
            const int c = j0 + gl < p.top ? teacher_entry(p, row, j0 + gl, &value) : -1;
            share(c, c >= 0 ? exp2_fast((value - tm) * scale) : 0.f);
        }
        if (HARD && gl == 0 && truth >= 0) target[truth] += hard_weight;
        __syncwarp();      // and from here on the gradient may lie on the logits
        T *g = p.grad + row * p.ldg;
        const float of_e = some ? soft_weight * reciprocal_fast(s) : 0.f, of_v = hard_weight * per_s1;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            float d = fmaf(e[u], of_e, -target[gl + u * L]);
            if (HARD) d = fmaf(v[u], of_v, d);
            if (!some && label == 0.f) d = 0.f;      // counts for nothing, also where 0 times its exponentials is not 0 (a branch around the row costs 4 % more)
            if (inside(u) && live) g[gl + u * L] = from_float<T>(d);
        }
        __syncwarp();
        if (c0 >= 0) target[c0] = 0;
        for (int j = L + gl; j < p.top; j += L) {
            const int c = teacher_entry(p, row, j, &value);
            if (c >= 0) target[c] = 0;
        }
        if (HARD && gl == 0 && truth >= 0) target[truth] = 0;
        __syncwarp();
        if (live) {      // the same in every lane of the row
            if (some) {
                soft_sum.add(t * (apart * per_ts) + t * t * (log_fast(s) - log_fast(ts)));
                soft_rows += 1;
            }
            if (HARD && label != 0.f) {
                hard_sum.add((log_fast(s1) - at_truth) * label);
                hard_rows += label;
            }
        }
    }
    LossSums sums = {0, 0, 0, 0};
    if (gl == 0) sums = {(double)soft_sum.sum, (double)soft_rows, (double)hard_sum.sum, (double)hard_rows};
    write_sums<256>(sums, p.sums);
}

// Rows of any number of classes, a block a row: one pass for maximum and sums (every thread its own maximum, so that the sums are scaled when
// it grows), one for the gradient that finds the row in L2.  16 bytes at a time behind the first values up to a multiple of 16, where logits
// and gradient lie alike; VEC = false: single values.
// 8,192 rows of 32,000 bfloat16 classes, 64 entries: 1.05 GB in 249 us (65 % of the copy rate; two exponentials a value); in three passes of single values
// 845 us, with blocks of 512 threads 316.
template <typename T, int THREADS, bool HARD, bool VEC>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) distillation_block_kernel(Distillation<T> p) {
    constexpr int V = VEC ? kVector<T> : 1, WARPS = THREADS / 32, AT_ONCE = VEC ? 4 : 8;      // vectors in flight a thread
    using Vector = Values<T, V>;
    __shared__ float2 max_of_warp[WARPS];
    __shared__ float4 sums_of_warp[WARPS];
    __shared__ float entry_weight[kMaxTop];
    __shared__ int entry_class[kMaxTop];
    static_assert(kMaxTop <= THREADS, "an entry a thread");
    const int tid = threadIdx.x, classes = p.classes;
    const float t = p.temperature, scale = kLog2e / t;
    LossSums sums = {0, 0, 0, 0};
    for (long long row = blockIdx.x; row < p.n; row += gridDim.x) {
        const T *x = p.logits + row * p.ld;
        T *g = p.grad + row * p.ldg;
        float value = -INFINITY;
        const int c_mine = tid < p.top ? teacher_entry(p, row, tid, &value) : -1;
        if (tid < p.top) entry_class[tid] = c_mine;
        const int head = VEC ? min(classes, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T))) : 0, vectors = (classes - head) / V,
                  tail = head + vectors * V;
        float m = -INFINITY, s = 0, s1 = 0;
        // adds values of which `to` is the largest
        auto add = [&](const float *z, int count, float to) {
            if (to > m) {
                s *= exp2_fast((m - to) * scale);
                if (HARD) s1 *= exp2_fast((m - to) * kLog2e);
                m = to;
            }
            const float from = m == -INFINITY ? 0.f : m;      // minus infinity adds 0, also where the thread has seen nothing else
#pragma unroll
            for (int k = 0; k < count; ++k) {
                s += exp2_fast((z[k] - from) * scale);
                if (HARD) s1 += exp2_fast((z[k] - from) * kLog2e);
            }
        };
        int i = tid;
        for (; i + (AT_ONCE - 1) * THREADS < vectors; i += THREADS * AT_ONCE) {
            Vector w[AT_ONCE];
            float z[AT_ONCE * V], most = -INFINITY;
#pragma unroll
            for (int b = 0; b < AT_ONCE; ++b) w[b] = *reinterpret_cast<const Vector *>(x + head + (long long)(i + b * THREADS) * V);
#pragma unroll
            for (int b = 0; b < AT_ONCE; ++b) w[b].get(z + b * V);
#pragma unroll
            for (int k = 0; k < AT_ONCE * V; ++k) most = fmaxf(most, z[k]);
            add(z, AT_ONCE * V, most);
        }
        for (; i < vectors; i += THREADS) {
            const Vector w = *reinterpret_cast<const Vector *>(x + head + (long long)i * V);
            float z[V], most = -INFINITY;
            w.get(z);
#pragma unroll
            for (int k = 0; k < V; ++k) most = fmaxf(most, z[k]);
            add(z, V, most);
        }
        if (VEC) {      // fewer than 16 bytes at either end
            const int c = tid < head ? tid : tail + tid - head;
            if (tid < head || (tid >= head && c < classes)) {
                const float z = to_float(x[c]);
                add(&z, 1, isnan(z) ? -INFINITY : z);
            }
        }
        const float2 most = make_float2(max_of_lanes<32>(m), max_of_lanes<32>(c_mine >= 0 ? value : -INFINITY));
        if ((tid & 31) == 0) max_of_warp[tid >> 5] = most;
        const bool any = __syncthreads_or(c_mine >= 0);
        float2 of_warp = max_of_warp[(tid & 31) % WARPS];
        const float row_max = max_of_lanes<32>(of_warp.x), tm = max_of_lanes<32>(of_warp.y);
        // sums of the row (those of a thread that has seen nothing but minus infinity are 0), and the teacher's
        float weight = 0, z_mine = 0;
        float4 sum = make_float4(m == -INFINITY ? s : s * exp2_fast((m - row_max) * scale), m == -INFINITY ? s1 : s1 * exp2_fast((m - row_max) * kLog2e), 0, 0);
        bool first = c_mine >= 0, again = false;
        if (c_mine >= 0) {
            weight = expf((value - tm) / t);
            z_mine = to_float(x[c_mine]);
            sum.z = weight;
            if (weight != 0.f) sum.w = weight * ((value - tm) - (z_mine - row_max));
            entry_weight[tid] = weight;
#pragma unroll 4
            for (int j = 0; j < p.top; ++j) {
                const bool same = j != tid && entry_class[j] == c_mine;
                again = again || same;
                first = first && !(same && j < tid);
            }
        }
        sum.x = sum_of_lanes<32>(sum.x);
        if (HARD) sum.y = sum_of_lanes<32>(sum.y);
        sum.z = sum_of_lanes<32>(sum.z);
        sum.w = sum_of_lanes<32>(sum.w);
        if ((tid & 31) == 0) sums_of_warp[tid >> 5] = sum;
        float label = 0, at_truth = 0;
        int truth = -1;
        if (HARD) {
            const long long wanted = __ldg(p.truth + row);
            const bool exists = wanted >= 0 && wanted < classes;
            label = !__ldg(p.labelled + row) ? 0.f : exists ? 1.f : NAN;
            truth = exists ? (int)wanted : -1;
            at_truth = exists ? to_float(x[truth]) : 0.f;
        }
        __syncthreads();      // and from here on the gradient may lie on the logits
        sum = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float4 o = sums_of_warp[w];
            sum.x += o.x, sum.y += o.y, sum.z += o.z, sum.w += o.w;
        }
        const float per_ts = 1.f / sum.z, soft_weight = any ? p.soft * t * (isnan(sum.z) ? NAN : 1.f) : 0.f, per_s = soft_weight / sum.x;
        const float hard_weight = label != 0.f ? p.hard * label : 0.f, per_s1 = hard_weight / sum.y;
        // the gradient of a class whose logit is z, without the teacher's share and the label
        auto gradient = [&](float z) {
            float d = exp2_fast((z - row_max) * scale) * per_s;
            if (HARD) d = fmaf(exp2_fast((z - row_max) * kLog2e), per_s1, d);
            return d;
        };
        auto write = [&] {
            int i = tid;
            for (; i + (AT_ONCE - 1) * THREADS < vectors; i += THREADS * AT_ONCE) {
                Vector w[AT_ONCE];
#pragma unroll
                for (int b = 0; b < AT_ONCE; ++b) w[b] = *reinterpret_cast<const Vector *>(x + head + (long long)(i + b * THREADS) * V);
#pragma unroll
                for (int b = 0; b < AT_ONCE; ++b) {
                    float z[V];
                    w[b].get(z);
#pragma unroll
                    for (int k = 0; k < V; ++k) z[k] = gradient(z[k]);
                    w[b].set(z);
                    *reinterpret_cast<Vector *>(g + head + (long long)(i + b * THREADS) * V) = w[b];
                }
            }
            for (; i < vectors; i += THREADS) {
                Vector w = *reinterpret_cast<const Vector *>(x + head + (long long)i * V);
                float z[V];
                w.get(z);
#pragma unroll
                for (int k = 0; k < V; ++k) z[k] = gradient(z[k]);
                w.set(z);
                *reinterpret_cast<Vector *>(g + head + (long long)i * V) = w;
            }
            if (VEC) {
                const int c = tid < head ? tid : tail + tid - head;
                if (tid < head || (tid >= head && c < classes)) g[c] = from_float<T>(gradient(to_float(x[c])));
            }
        };
        if (!any && label == 0.f) {
            for (int c = tid; c < classes; c += THREADS) g[c] = from_float<T>(0.f);
        } else {
            write();
        }
        __syncthreads();
        if (first) {      // the first entry of a class has the share of all of them
            float all = weight;
            if (again)
                for (int j = tid + 1; j < p.top; ++j)
                    if (entry_class[j] == c_mine) all += entry_weight[j];
            float d = gradient(z_mine) - soft_weight * (all * per_ts);
            if (HARD && c_mine == truth) d -= hard_weight;
            g[c_mine] = from_float<T>(d);
        }
        if (HARD) {      // a labelled class that is no entry
            bool entry = false;
            if (tid < p.top) entry = c_mine == truth;
            entry = __syncthreads_or(entry);
            if (!entry && tid == 0 && truth >= 0 && label != 0.f) g[truth] = from_float<T>(gradient(at_truth) - hard_weight);
        }
        if (tid == 0) {
            if (any) {
                sums.soft += (double)(t * (sum.w * per_ts) + t * t * (logf(sum.x) - logf(sum.z)));
                sums.soft_rows += 1;
            }
            if (HARD && label != 0.f) {
                sums.hard += (double)((logf(sum.y) - (at_truth - row_max)) * label);
                sums.hard_rows += label;
            }
        }
        __syncthreads();      // the entries have been read
    }
    write_sums<THREADS>(sums, p.sums);
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
        const bool alike = ((reinterpret_cast<uintptr_t>(p.logits) ^ reinterpret_cast<uintptr_t>(p.grad)) & 15) == 0 && (p.ld - p.ldg) * (long long)sizeof(T) % 16 == 0;
        const int per = lanes ? (p.classes + lanes - 1) / lanes : 0;
        switch (lanes + per) {
#define DRONE_ROWS(L, PER) case L + PER: distillation_rows_kernel<T, L, PER, HARD><<<blocks, 256, 0, st>>>(p); break
            DRONE_ROWS(8, 1); DRONE_ROWS(8, 2); DRONE_ROWS(8, 3); DRONE_ROWS(8, 4); DRONE_ROWS(8, 5); DRONE_ROWS(8, 6); DRONE_ROWS(8, 7); DRONE_ROWS(8, 8);
            DRONE_ROWS(32, 3); DRONE_ROWS(32, 4); DRONE_ROWS(32, 5); DRONE_ROWS(32, 6); DRONE_ROWS(32, 7); DRONE_ROWS(32, 8);
#undef DRONE_ROWS
            default:
                alike ? distillation_block_kernel<T, 256, HARD, true><<<blocks, 256, 0, st>>>(p)
                      : distillation_block_kernel<T, 256, HARD, false><<<blocks, 256, 0, st>>>(p);
        }
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
    DRONE_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, "drone_distillation_loss: temperature=%g", temperature);
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
