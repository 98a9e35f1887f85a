// The readout's operators on logits: the rules of a generation step, the draw of a category, and the distillation loss with
// its gradient.  One row = one sequence (or chain) of up to 2^30 categories; sums, softmax statistics and scores are held in
// f32 or f64, and each output is rounded once to its own type.
#include "device_math.cuh"
#include "readout.cuh"

using namespace thrml;
using namespace thrml::readout;

namespace {

constexpr int64_t MAX_COLS = 1 << 30;  // indices inside a row stay in 32 bits
constexpr int TOP_MAX = 1024;          // listed teacher entries held in shared memory
constexpr uint32_t TAG_DRAW = 0x44524157u;

// ---------------------------------------------------------------------------------------------------------
// Rules on logits.
// ---------------------------------------------------------------------------------------------------------
constexpr int ADJUST_THREADS = 256, ADJUST_SLICE = 8192;
constexpr uint32_t IN_PROMPT = 0x80000000u;

struct AdjustArgs {
    const void* logits;
    void* out;
    int64_t pitch, out_pitch;
    int32_t cols, slices;
    thrml_logit_rules rules;
};

// A CTA takes one slice of one row.  The history's tokens that fall into the slice are counted in shared memory (integer
// atomics: the counts do not depend on their order), the biases are summed there, and one pass over the slice reads, adjusts
// and writes the logits.
template <class T>
__global__ void __launch_bounds__(ADJUST_THREADS) k_adjust(const AdjustArgs g) {
    extern __shared__ uint32_t adjust_smem[];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / g.slices;
    const int32_t k0 = static_cast<int32_t>(blockIdx.x % g.slices) * ADJUST_SLICE, n = min(ADJUST_SLICE, g.cols - k0);
    const thrml_logit_rules& ru = g.rules;
    uint32_t* count = adjust_smem;
    float* bias = reinterpret_cast<float*>(adjust_smem + (ru.history ? ADJUST_SLICE : 0));

    const int64_t h0 = ru.history ? ru.history_ptr[row] : 0, h1 = ru.history ? ru.history_ptr[row + 1] : 0;
    const int64_t b0 = ru.bias_ids ? ru.bias_ptr[row] : 0, b1 = ru.bias_ids ? ru.bias_ptr[row + 1] : 0;
    const bool has_history = h1 > h0, has_bias = b1 > b0;
    if (has_history)
        for (int i = tid; i < n; i += ADJUST_THREADS) count[i] = 0;
    if (has_bias)
        for (int i = tid; i < n; i += ADJUST_THREADS) bias[i] = 0.0f;
    __syncthreads();
    if (has_history) {
        const int64_t prompt_end = h0 + (ru.n_prompt ? max(ru.n_prompt[row], 0) : 0);
        for (int64_t i = h0 + tid; i < h1; i += ADJUST_THREADS) {
            const int64_t at = load_as_int(ru.history, ru.history_type, i) - k0;
            if (at >= 0 && at < n) {
                if (i < prompt_end) atomicOr(count + at, IN_PROMPT);
                else atomicAdd(count + at, 1u);
            }
        }
    }
    if (has_bias) {
        // the first entry of a run of equal ids adds the run up in its order
        for (int64_t i = b0 + tid; i < b1; i += ADJUST_THREADS) {
            const int32_t id = ru.bias_ids[i], at = id - k0;
            if (id < 0 || at < 0 || at >= n || (i > b0 && ru.bias_ids[i - 1] == id)) continue;
            float sum = ru.bias_values[i];
            for (int64_t j = i + 1; j < b1 && ru.bias_ids[j] == id; ++j) sum += ru.bias_values[j];
            atomicAdd(bias + at, sum);  // one addend unless the ids are not in order
        }
    }
    __syncthreads();

    const float repetition = ru.repetition ? ru.repetition[row] : 1.0f, frequency = ru.frequency ? ru.frequency[row] : 0.0f,
                presence = ru.presence ? ru.presence[row] : 0.0f;
    const int64_t m = !ru.mask ? -1 : ru.mask_rows ? ru.mask_rows[row] : row;
    const uint32_t* mask = ru.mask && m >= 0 && m < ru.n_masks ? ru.mask + m * ru.mask_pitch : nullptr;
    const T* in = static_cast<const T*>(g.logits) + row * g.pitch + k0;
    T* out = static_cast<T*>(g.out) + row * g.out_pitch + k0;
    for_row<T>(in, n, tid, ADJUST_THREADS, [&](int32_t i, const float* v, auto cnt) {
        constexpr int N = decltype(cnt)::value;
        float x[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            x[j] = v[j];
            const uint32_t c = has_history ? count[i + j] : 0u;
            if (c) {
                x[j] = x[j] > 0.0f ? __fdiv_rn(x[j], repetition) : x[j] * repetition;
                const uint32_t told = c & ~IN_PROMPT;
                if (told) x[j] = x[j] - frequency * static_cast<float>(told) - presence;
            }
            if (has_bias) x[j] += bias[i + j];
            if (mask && !((mask[(k0 + i + j) >> 5] >> ((k0 + i + j) & 31)) & 1u)) x[j] = -INFINITY;
        }
        store_n<T>(out + i, x, cnt);
    });
}

// ---------------------------------------------------------------------------------------------------------
// The draw of a category.
// ---------------------------------------------------------------------------------------------------------
constexpr int DRAW_THREADS = 512;

struct DrawArgs {
    const void* logits;
    const float* beta;
    const float* noise;
    int64_t* out;
    int64_t pitch, noise_pitch;
    int32_t cols;
    uint32_t row_offset;
    PhiloxRoundKeys rk;
};

// (score, category) of the larger score, the lower category among equal ones; category -1 = none yet.
struct Best {
    double score;
    int32_t k;
    __device__ __forceinline__ void take(double s, int32_t i) {
        if (i >= 0 && s > -INFINITY && (k < 0 || s > score || (s == score && i < k))) {
            score = s;
            k = i;
        }
    }
};

// One CTA per row; every score in f64.
template <class T>
__global__ void __launch_bounds__(DRAW_THREADS) k_draw(const DrawArgs g) {
    __shared__ double sh_score[DRAW_THREADS / 32];
    __shared__ int32_t sh_k[DRAW_THREADS / 32];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const float beta = g.beta ? g.beta[row] : 1.0f;
    const bool greedy = beta == INFINITY;
    const T* logits = static_cast<const T*>(g.logits) + row * g.pitch;
    const float* noise = g.noise ? g.noise + row * g.noise_pitch : nullptr;
    Best best{0.0, -1};
    if (beta >= 0.0f) {
        for (int32_t k = 4 * tid; k < g.cols; k += 4 * DRAW_THREADS) {
            U4 words{};
            if (!noise && !greedy) words = philox4x32_10_rk(g.row_offset + static_cast<uint32_t>(row), 0u, static_cast<uint32_t>(k) >> 2, TAG_DRAW, g.rk);
            for (int j = 0; j < 4 && k + j < g.cols; ++j) {
                const float l = to_float(logits[k + j]);
                if (!(l > -INFINITY)) continue;  // masked, or not a number
                double score = l;
                if (!greedy) {
                    const double u = noise ? noise[k + j] : u23_open(pick(words, j));
                    score = __dsub_rn(__dmul_rn(beta, l), log(-log(u)));
                }
                best.take(score, k + j);
            }
        }
    }
    for (int d = 16; d; d >>= 1) {
        const double s = __shfl_xor_sync(0xffffffffu, best.score, d);
        const int32_t k = __shfl_xor_sync(0xffffffffu, best.k, d);
        best.take(s, k);
    }
    if ((tid & 31) == 0) {
        sh_score[tid >> 5] = best.score;
        sh_k[tid >> 5] = best.k;
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < DRAW_THREADS / 32; ++w) best.take(sh_score[w], sh_k[w]);
        g.out[row] = best.k;
    }
}

// ---------------------------------------------------------------------------------------------------------
// Distillation.
// ---------------------------------------------------------------------------------------------------------
constexpr int DISTILL_THREADS = 512;
enum Distill { LOSS, GRAD, STEP };

struct DistillArgs {
    const void* logits;
    const void* ids;
    const void* teacher;
    const float* weight;
    const float* lse_in;
    float* loss;
    float* lse_out;
    void* grad;
    int64_t pitch, ids_pitch, teacher_pitch, grad_pitch;
    int32_t cols, top, ids_type, teacher_type;
    float beta;
};

// The teacher's side of one row, in shared memory.
struct Listed {
    int32_t id[TOP_MAX];   // -1 = not listed
    float p[TOP_MAX];      // softmax over the listed entries
    float z[TOP_MAX];      // beta times the student's logit there
    float scratch[32];
    int any;
};

// Fills `L` (all threads of the block).
template <class T>
__device__ __forceinline__ void list_teacher(Listed& L, const DistillArgs& g, int64_t row, const T* logits) {
    if (threadIdx.x == 0) L.any = 0;
    float most = -INFINITY;
    bool some = false;
    __syncthreads();
    for (int j = threadIdx.x; j < g.top; j += blockDim.x) {
        const int64_t id = load_as_int(g.ids, g.ids_type, row * g.ids_pitch + j);
        const float t = g.beta * load_as_float(g.teacher, g.teacher_type, row * g.teacher_pitch + j);
        const bool listed = id >= 0 && id < g.cols && !(t == -INFINITY);
        L.id[j] = listed ? static_cast<int32_t>(id) : -1;
        L.p[j] = t;
        L.z[j] = listed ? g.beta * to_float(logits[id]) : 0.0f;
        if (listed) {
            most = fmaxf(most, t);
            some = true;
        }
    }
    if (some) L.any = 1;
    most = block_reduce<MaxOp>(most, L.scratch);
    float total = 0.0f;
    for (int j = threadIdx.x; j < g.top; j += blockDim.x) {
        L.p[j] = L.id[j] >= 0 ? expf(L.p[j] - most) : 0.0f;
        total += L.p[j];
    }
    total = block_reduce<SumOp>(total, L.scratch);
    for (int j = threadIdx.x; j < g.top; j += blockDim.x) L.p[j] = L.p[j] / total;
    __syncthreads();
}

// One CTA per row.  LOSS: maximum and sum of the softmax in one pass, then the loss over the listed entries.  GRAD: one pass
// that writes weight * beta * q, then the listed entries once more with p subtracted.  STEP: both.
template <class T, int MODE>
__global__ void __launch_bounds__(DISTILL_THREADS) k_distill(const DistillArgs g) {
    __shared__ Listed L;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const float weight = g.weight ? g.weight[row] : 1.0f;
    const T* logits = static_cast<const T*>(g.logits) + row * g.pitch;
    T* grad = MODE == LOSS ? nullptr : static_cast<T*>(g.grad) + row * g.grad_pitch;
    bool live = weight != 0.0f;
    if (live) {
        list_teacher<T>(L, g, row, logits);
        live = L.any != 0;
    }
    if (!live) {  // padding: nothing of the row is read
        if (MODE != LOSS) for (int32_t k = tid; k < g.cols; k += DISTILL_THREADS) grad[k] = from_float<T>(0.0f);
        if (tid == 0 && MODE != GRAD) g.loss[row] = 0.0f;
        if (tid == 0 && MODE == LOSS) g.lse_out[row] = 0.0f;
        return;
    }
    float lse;
    if (MODE == GRAD) {
        lse = g.lse_in[row];
    } else {
        float most = -INFINITY;
        for_row<T>(logits, g.cols, tid, DISTILL_THREADS, [&](int32_t, const float* v, auto cnt) {
#pragma unroll
            for (int j = 0; j < decltype(cnt)::value; ++j) most = v[j] > most || v[j] != v[j] ? v[j] : most;  // a NaN stays
        });
        most = most != most ? INFINITY : most;
        most = g.beta * block_reduce<MaxOp>(most, L.scratch);
        float total = 0.0f;
        for_row<T>(logits, g.cols, tid, DISTILL_THREADS, [&](int32_t, const float* v, auto cnt) {
#pragma unroll
            for (int j = 0; j < decltype(cnt)::value; ++j) total += most == -INFINITY ? 0.0f : expf(g.beta * v[j] - most);
        });
        total = block_reduce<SumOp>(total, L.scratch);
        lse = most == -INFINITY ? -INFINITY : most + logf(total);
        float loss = 0.0f;
        for (int j = tid; j < g.top; j += DISTILL_THREADS)
            if (L.p[j] > 0.0f || L.p[j] != L.p[j]) loss += lse == -INFINITY ? INFINITY : L.p[j] * (logf(L.p[j]) - (L.z[j] - lse));
        loss = block_reduce<SumOp>(loss, L.scratch);
        if (tid == 0) g.loss[row] = loss;
        if (tid == 0 && MODE == LOSS) g.lse_out[row] = lse;
    }
    if (MODE != LOSS) {
        const float scale = weight * g.beta;
        for_row<T>(logits, g.cols, tid, DISTILL_THREADS, [&](int32_t i, const float* v, auto cnt) {
            constexpr int N = decltype(cnt)::value;
            float x[N];
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = lse == -INFINITY ? 0.0f : scale * expf(g.beta * v[j] - lse);
            store_n<T>(grad + i, x, cnt);
        });
        __syncthreads();  // the listed entries are written once more
        for (int j = tid; j < g.top; j += DISTILL_THREADS) {
            if (L.id[j] < 0) continue;
            float p = 0.0f;
            bool first = true;
            for (int i = 0; i < g.top; ++i) {
                if (L.id[i] != L.id[j]) continue;
                if (i < j) first = false;
                p += L.p[i];
            }
            if (first) grad[L.id[j]] = from_float<T>(scale * ((lse == -INFINITY ? 0.0f : expf(L.z[j] - lse)) - p));
        }
    }
}

int32_t check_rows(const char* what, int64_t rows, int64_t cols, const void* p, int32_t type, int64_t pitch) {
    const std::string name(what);
    if (rows < 0 || rows > INT32_MAX) return fail(THRML_ERR_INVALID_ARG, name + ": the number of rows is out of range");
    if (cols < 1 || cols > MAX_COLS) return fail(THRML_ERR_INVALID_ARG, name + ": rows hold 1 to 2^30 elements");
    if (!is_float_type(type)) return fail(THRML_ERR_INVALID_ARG, name + ": the element type is not a float type");
    if (pitch < cols) return fail(THRML_ERR_INVALID_ARG, name + ": the pitch is smaller than a row");
    if (rows && !p) return fail(THRML_ERR_INVALID_ARG, name + ": null pointer");
    if (!aligned_to(p, type_size(type))) return fail(THRML_ERR_INVALID_ARG, name + ": the pointer is not aligned to the element");
    return THRML_OK;
}

int32_t distill(thrml_ctx* ctx, void* stream, int mode, int64_t rows, int32_t type, const DistillArgs& g) {
    if (int32_t rc = check_rows("logits", rows, g.cols, g.logits, type, g.pitch)) return rc;
    if (mode != LOSS) {
        if (int32_t rc = check_rows("grad", rows, g.cols, g.grad, type, g.grad_pitch)) return rc;
        if (g.grad == g.logits && g.grad_pitch != g.pitch) return fail(THRML_ERR_INVALID_ARG, "grad over the logits needs their pitch");
    }
    if (g.top < 0 || g.top > TOP_MAX) return fail(THRML_ERR_INVALID_ARG, "top is not within 0 and 1024");
    if (!is_index_type(g.ids_type)) return fail(THRML_ERR_INVALID_ARG, "ids: the element type is not an index type");
    if (!is_float_type(g.teacher_type)) return fail(THRML_ERR_INVALID_ARG, "teacher: the element type is not a float type");
    if (g.ids_pitch < g.top || g.teacher_pitch < g.top) return fail(THRML_ERR_INVALID_ARG, "ids, teacher: the pitch is smaller than top");
    if (!(g.beta > 0.0f) || g.beta == INFINITY) return fail(THRML_ERR_INVALID_ARG, "beta has to be positive and finite");
    if (rows == 0) return THRML_OK;
    if (g.top && (!g.ids || !g.teacher)) return fail(THRML_ERR_INVALID_ARG, "ids, teacher: null pointer");
    if ((mode != GRAD && !g.loss) || (mode == LOSS && !g.lse_out) || (mode == GRAD && !g.lse_in)) return fail(THRML_ERR_INVALID_ARG, "loss, lse: null pointer");
    return for_type(type, [&](auto e) {
        using T = decltype(e);
        const auto kernel = mode == LOSS ? k_distill<T, LOSS> : mode == GRAD ? k_distill<T, GRAD> : k_distill<T, STEP>;
        kernel<<<static_cast<unsigned>(rows), DISTILL_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(g);
        CU_TRY(cudaGetLastError());
        return THRML_OK;
    });
}

DistillArgs distill_args(const void* logits, int64_t pitch, int64_t cols, int64_t top, const void* ids, int32_t ids_type, int64_t ids_pitch, const void* teacher,
                         int32_t teacher_type, int64_t teacher_pitch, float beta, const float* weight) {
    DistillArgs g{};
    g.logits = logits;
    g.pitch = pitch;
    g.cols = cols >= 1 && cols <= MAX_COLS ? static_cast<int32_t>(cols) : 0;  // 0 is refused
    g.top = top >= 0 && top <= TOP_MAX ? static_cast<int32_t>(top) : -1;      // -1 is refused
    g.ids = ids;
    g.ids_type = ids_type;
    g.ids_pitch = ids_pitch;
    g.teacher = teacher;
    g.teacher_type = teacher_type;
    g.teacher_pitch = teacher_pitch;
    g.beta = beta;
    g.weight = weight;
    return g;
}

}  // namespace

extern "C" {

int32_t thrml_adjust_logits(thrml_ctx* ctx, void* stream, int64_t rows, int64_t cols, const void* logits, int32_t type, int64_t pitch, void* out, int64_t out_pitch,
                            const thrml_logit_rules* rules) {
    return guarded(ctx, [&]() -> int32_t {
        if (!rules) return fail(THRML_ERR_INVALID_ARG, "null rules");
        if (int32_t rc = check_rows("logits", rows, cols, logits, type, pitch)) return rc;
        if (int32_t rc = check_rows("out", rows, cols, out, type, out_pitch)) return rc;
        if (out == logits && out_pitch != pitch) return fail(THRML_ERR_INVALID_ARG, "out over the logits needs their pitch");
        if (rules->history && !is_index_type(rules->history_type)) return fail(THRML_ERR_INVALID_ARG, "history: the element type is not an index type");
        if (rules->history && !rules->history_ptr) return fail(THRML_ERR_INVALID_ARG, "history without history_ptr");
        if (rules->bias_ids && (!rules->bias_ptr || !rules->bias_values)) return fail(THRML_ERR_INVALID_ARG, "bias_ids without bias_ptr and bias_values");
        if (rules->mask && (rules->n_masks < 1 || rules->mask_pitch < (cols + 31) / 32)) return fail(THRML_ERR_INVALID_ARG, "mask: no masks, or a pitch smaller than a row's bits");
        if (rows == 0) return THRML_OK;
        AdjustArgs g{logits, out, pitch, out_pitch, static_cast<int32_t>(cols), static_cast<int32_t>((cols + ADJUST_SLICE - 1) / ADJUST_SLICE), *rules};
        if (rows * g.slices > INT32_MAX) return fail(THRML_ERR_INVALID_ARG, "too many rows of this length in one call");
        const size_t smem = sizeof(uint32_t) * ADJUST_SLICE * ((rules->history ? 1 : 0) + (rules->bias_ids ? 1 : 0));
        return for_type(type, [&](auto e) {
            using T = decltype(e);
            CU_TRY(cudaFuncSetAttribute(k_adjust<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * sizeof(uint32_t) * ADJUST_SLICE));
            k_adjust<T><<<static_cast<unsigned>(rows * g.slices), ADJUST_THREADS, smem, static_cast<cudaStream_t>(stream)>>>(g);
            CU_TRY(cudaGetLastError());
            return THRML_OK;
        });
    });
}

int32_t thrml_draw_categories(thrml_ctx* ctx, void* stream, int64_t rows, int64_t cols, const void* logits, int32_t type, int64_t pitch, const float* beta, uint64_t key,
                              int64_t row_offset, const float* noise, int64_t noise_pitch, int64_t* out) {
    return guarded(ctx, [&]() -> int32_t {
        if (int32_t rc = check_rows("logits", rows, cols, logits, type, pitch)) return rc;
        if (noise)
            if (int32_t rc = check_rows("noise", rows, cols, noise, THRML_F32, noise_pitch)) return rc;
        if (row_offset < 0 || row_offset > (int64_t{1} << 32) - rows) return fail(THRML_ERR_INVALID_ARG, "row_offset is out of range");
        if (rows == 0) return THRML_OK;
        if (!out) return fail(THRML_ERR_INVALID_ARG, "out: null pointer");
        const DrawArgs g{logits, beta, noise, out, pitch, noise_pitch, static_cast<int32_t>(cols), static_cast<uint32_t>(row_offset), make_round_keys(key)};
        return for_type(type, [&](auto e) {
            k_draw<decltype(e)><<<static_cast<unsigned>(rows), DRAW_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(g);
            CU_TRY(cudaGetLastError());
            return THRML_OK;
        });
    });
}

int32_t thrml_distill_loss(thrml_ctx* ctx, void* stream, int64_t rows, int64_t cols, const void* logits, int32_t type, int64_t pitch, int64_t top, const void* ids,
                           int32_t ids_type, int64_t ids_pitch, const void* teacher, int32_t teacher_type, int64_t teacher_pitch, float beta, const float* weight,
                           float* loss, float* lse) {
    return guarded(ctx, [&] {
        DistillArgs g = distill_args(logits, pitch, cols, top, ids, ids_type, ids_pitch, teacher, teacher_type, teacher_pitch, beta, weight);
        g.loss = loss;
        g.lse_out = lse;
        return distill(ctx, stream, LOSS, rows, type, g);
    });
}

int32_t thrml_distill_grad(thrml_ctx* ctx, void* stream, int64_t rows, int64_t cols, const void* logits, int32_t type, int64_t pitch, int64_t top, const void* ids,
                           int32_t ids_type, int64_t ids_pitch, const void* teacher, int32_t teacher_type, int64_t teacher_pitch, float beta, const float* weight,
                           const float* lse, void* grad, int64_t grad_pitch) {
    return guarded(ctx, [&] {
        DistillArgs g = distill_args(logits, pitch, cols, top, ids, ids_type, ids_pitch, teacher, teacher_type, teacher_pitch, beta, weight);
        g.lse_in = lse;
        g.grad = grad;
        g.grad_pitch = grad_pitch;
        return distill(ctx, stream, GRAD, rows, type, g);
    });
}

int32_t thrml_distill_step(thrml_ctx* ctx, void* stream, int64_t rows, int64_t cols, const void* logits, int32_t type, int64_t pitch, int64_t top, const void* ids,
                           int32_t ids_type, int64_t ids_pitch, const void* teacher, int32_t teacher_type, int64_t teacher_pitch, float beta, const float* weight,
                           float* loss, void* grad, int64_t grad_pitch) {
    return guarded(ctx, [&] {
        DistillArgs g = distill_args(logits, pitch, cols, top, ids, ids_type, ids_pitch, teacher, teacher_type, teacher_pitch, beta, weight);
        g.loss = loss;
        g.grad = grad;
        g.grad_pitch = grad_pitch;
        return distill(ctx, stream, STEP, rows, type, g);
    });
}

}  // extern "C"
