// The readout's operators on logits: the rules of a generation step, the draw of a category, and the distillation loss with
// its gradient.  One row = one sequence (or chain) of up to 2^30 categories; sums, softmax statistics and scores are held in
// f32 or f64, and each output is rounded once to its own type.
#include <algorithm>
#include <cstddef>

#include "device_math.cuh"
#include "readout.cuh"
#include "tensor_core.cuh"

using namespace thrml;
using namespace thrml::readout;

namespace {

constexpr int64_t MAX_COLS = 1 << 30;  // indices inside a row stay in 32 bits
constexpr int TOP_MAX = 1024;          // listed teacher entries held in shared memory
constexpr uint32_t TAG_DRAW = 0x44524157u;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Floats as integers in the same order, for integer maxima.
__device__ __forceinline__ int32_t ordered(float x) {
    const int32_t b = __float_as_int(x);
    return b < 0 ? b ^ 0x7fffffff : b;
}
__device__ __forceinline__ float from_ordered(int32_t b) { return __int_as_float(b < 0 ? b ^ 0x7fffffff : b); }

// 16 bytes of -infinity.
template <class T>
__device__ __forceinline__ uint4 nothing_16() {
    constexpr uint32_t w = std::is_same<T, float>::value ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    return make_uint4(w, w, w, w);
}

// ---------------------------------------------------------------------------------------------------------
// Rules on logits.
//
// Every logit is read and written once.  A CTA copies a share of a row into shared memory, ADJUST_PIECES 16-byte pieces a thread,
// in flight together; meanwhile it counts there those of the row's tokens that fall into the share (integer atomics, so the counts
// do not depend on their order).  A count has 16 bits, and 32 in rows of 2^15 tokens or more (and where the repetition penalty has no reciprocal in f32), which are done half a share at a time.
// Every CTA of a row reads the whole history, from L2 after the first.  256 x 131072 bf16 with 4096 tokens, biases and masks 56 us =
// 2.4 TB/s: issue slots are busy for 69 % of it (39 M warp instructions, 35 us at full issue), shared memory and barriers hold the rest;
// without any rule 23, by memory.
// Categories with a bias are finished by a thread of their own, before the pass over the share, which leaves out what a bitmap
// marks.  Measured and dropped for 256 rows of 131072 bf16 with 3000 tokens each: the few named categories in a kernel of
// their own behind a plain copy, 77 us (their scattered 2-byte writes cost more than they are); for 16 rows with 60000
// tokens, the history read once per row with atomics into the shared memory of the CTA that holds the category, 137 us, since
// few categories take most of the tokens.
// ---------------------------------------------------------------------------------------------------------
constexpr int ADJUST_THREADS = 512, ADJUST_PIECES = 4;
template <class T>
constexpr int ADJUST_SHARE = ADJUST_THREADS * ADJUST_PIECES * VEC<T>;  // most positions of a CTA

struct AdjustArgs {
    const void* logits;
    void* out;
    int64_t pitch, out_pitch;
    int32_t cols, share, per_row, count_words;  // positions of a row per CTA, CTAs per row, words of counts
    thrml_logit_rules rules;
};

// -infinity where the bit is 0.
template <class T>
__device__ __forceinline__ uint4 close_16(const uint4& raw, uint32_t open) {
    const uint4 none = nothing_16<T>();
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (sizeof(T) == 4) x[i] = (open >> i) & 1u ? w[i] : none.x;
        else {
            const uint32_t keep = (((open >> (2 * i)) & 1u) | ((open >> (2 * i) & 2u) << 15)) * 0xffffu;  // bits 0 and 16 to all of their halves
            x[i] = (w[i] & keep) | (none.x & ~keep);
        }
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// What the penalties make of a logit that was seen, `told` times behind the prompt.
struct Penalties {
    float repetition, per_repetition, frequency, presence;
    // One division a row instead of one a category (1.5 steps of f32 at most; 256 x 131072 bf16 56 us, with divisions 60), where the
    // reciprocal is a normal number.
    __device__ __forceinline__ bool has_reciprocal() const { return repetition >= 0x1p-126f && repetition <= 0x1p126f; }
    template <bool DIVIDE>
    __device__ __forceinline__ float of(float x, uint32_t told) const {
        if (DIVIDE) x = x > 0.0f ? __fdiv_rn(x, repetition) : x * repetition;
        else x *= x > 0.0f ? per_repetition : repetition;
        return told ? x - fmaf(frequency, static_cast<float>(told), presence) : x;
    }
};

// Counts of BITS bits, packed in words, the highest for "in the prompt".
template <int BITS>
struct Counts {
    static constexpr int PER_WORD = 32 / BITS;
    static constexpr uint32_t IN_PROMPT = 1u << (BITS - 1), ALL = BITS == 32 ? 0xffffffffu : (1u << BITS) - 1u;
    uint32_t* words;
    __device__ __forceinline__ static int shift(uint32_t i) { return BITS * (i % PER_WORD); }
    __device__ __forceinline__ void prompt(uint32_t i) const { atomicOr(words + i / PER_WORD, IN_PROMPT << shift(i)); }
    __device__ __forceinline__ void told(uint32_t i) const { atomicAdd(words + i / PER_WORD, 1u << shift(i)); }
    __device__ __forceinline__ uint32_t at(uint32_t i) const { return (words[i / PER_WORD] >> shift(i)) & ALL; }
};

// f(place) for each token that lies in [low, low + n).
template <class I, class F>
__device__ __forceinline__ void each_token(const I* history, int64_t h0, int64_t h1, int32_t low, uint32_t n, F f) {
    using U = typename std::make_unsigned<I>::type;
    constexpr int AT_ONCE = 4;
    while (h0 < h1) {
        const int32_t len = static_cast<int32_t>(min(h1 - h0, int64_t{1} << 30));
        const I* h = history + h0;
#pragma unroll 1
        for (int32_t i = threadIdx.x; i < len; i += AT_ONCE * ADJUST_THREADS) {
            U at[AT_ONCE];
#pragma unroll
            for (int t = 0; t < AT_ONCE; ++t) at[t] = i + t * ADJUST_THREADS < len ? static_cast<U>(h[i + t * ADJUST_THREADS]) - static_cast<U>(I{low}) : n;
#pragma unroll
            for (int t = 0; t < AT_ONCE; ++t)
                if (at[t] < n) f(static_cast<uint32_t>(at[t]));  // a token below low has wrapped to beyond n
        }
        h0 += len;
    }
}

template <class T>
__global__ void __launch_bounds__(ADJUST_THREADS, 3) k_adjust(const __grid_constant__ AdjustArgs g) {
    constexpr int V = VEC<T>;
    extern __shared__ uint4 adjust_smem[];
    __shared__ uint32_t mask_words[ADJUST_SHARE<T> / 32 + 2];
    const int tid = threadIdx.x;
    const thrml_logit_rules& ru = g.rules;
    const int64_t row = g.per_row == 1 ? blockIdx.x : blockIdx.x / g.per_row;
    const T* logits = static_cast<const T*>(g.logits) + row * g.pitch;
    T* out = static_cast<T*>(g.out) + row * g.out_pitch;
    const Pieces<T> pieces(logits, g.cols);
    const int32_t ahead = pieces.ahead;
    const int32_t from = static_cast<int32_t>(blockIdx.x - row * g.per_row) * g.share, to = min(pieces.end, from + g.share);
    if (from >= to) return;
    uint4* tile = adjust_smem;  // a thread's piece s at s * ADJUST_THREADS + tid
    uint4* counts = tile + ADJUST_PIECES * ADJUST_THREADS;                                                                       // [share] of 16 bits, when there are histories
    uint32_t* biased = reinterpret_cast<uint32_t*>(counts) + (ru.history ? g.count_words : 0);  // [share] bits, when there are biases

    const int64_t h0 = ru.history ? ru.history_ptr[row] : 0, h1 = ru.history ? ru.history_ptr[row + 1] : 0;
    const int64_t b0 = ru.bias_ids ? ru.bias_ptr[row] : 0, b1 = ru.bias_ids ? ru.bias_ptr[row + 1] : 0;
    auto place = [&](int s) { return from + (s * ADJUST_THREADS + tid) * V; };
    for (int s = 0; s < ADJUST_PIECES; ++s)
        if (place(s) < to) pieces.fetch(tile + s * ADJUST_THREADS + tid, place(s));
    commit_copies();
    const int32_t n_bias = static_cast<int32_t>(b1 - b0);
    const bool has_history = h1 > h0, has_bias = n_bias > 0;
    const int32_t* ids = ru.bias_ids + b0;
    const int64_t split = has_history && ru.n_prompt ? min(h1, h0 + max(ru.n_prompt[row], 0)) : h0;
    const float repetition = ru.repetition ? ru.repetition[row] : 1.0f;
    const Penalties penalties{repetition, __fdiv_rn(1.0f, repetition), ru.frequency ? ru.frequency[row] : 0.0f, ru.presence ? ru.presence[row] : 0.0f};
    const int64_t m = !ru.mask ? -1 : ru.mask_rows ? ru.mask_rows[row] : row;
    const uint32_t* mask = ru.mask && m >= 0 && m < ru.n_masks ? ru.mask + m * ru.mask_pitch : nullptr;
    const bool wide = pieces.same_phase(out);
    float logit = 0.0f;  // of the first bias entry that this thread finishes, read early
    if (has_history)
        for (int i = tid; i < g.count_words / 4; i += ADJUST_THREADS) counts[i] = make_uint4(0u, 0u, 0u, 0u);
    const int32_t first_word = max(from - ahead, 0) >> 5;  // of the mask, which the share needs up to the word of its last category
    if (mask)
        for (int32_t i = first_word + tid; i <= (to - 1 - ahead) >> 5; i += ADJUST_THREADS) mask_words[i - first_word] = mask[i];
    if (has_bias) {
        for (int i = tid; i < g.share / 32; i += ADJUST_THREADS) biased[i] = 0u;
        __syncthreads();
        for (int32_t e = tid; e < n_bias; e += ADJUST_THREADS) {
            const uint32_t at = ids[e] - (from - ahead);
            if (ids[e] < 0 || at >= static_cast<uint32_t>(to - from)) continue;
            atomicOr(biased + (at >> 5), 1u << (at & 31));
            if (e == tid) logit = to_float(logits[ids[e]]);
        }
    }

    // Pieces s0 .. s1 of each thread, the positions [begin, stop), with counts of BITS bits.
    auto pass = [&](auto bits, int s0, int s1, int32_t begin, int32_t stop) {
        constexpr int BITS = decltype(bits)::value;
        auto penalise = [&](float x, uint32_t told) { return penalties.of<BITS == 32>(x, told); };
        const Counts<BITS> count{reinterpret_cast<uint32_t*>(counts)};
        if (has_history) {
            if (s0 > 0)  // the second half's; the first begin at 0
                for (int i = tid; i < g.count_words / 4; i += ADJUST_THREADS) counts[i] = make_uint4(0u, 0u, 0u, 0u);
            if (s0 > 0 || !has_bias) __syncthreads();
            // `low` is the category at `begin`; below 0 (the first CTA's, when ahead > 0) lie no categories
            const int32_t low = max(begin - ahead, 0);
            const uint32_t first = low + ahead - begin, n = static_cast<uint32_t>(stop - ahead - low);
            auto each = [&](auto* history) {
                each_token(history, h0, split, low, n, [&](uint32_t i) { count.prompt(first + i); });
                each_token(history, split, h1, low, n, [&](uint32_t i) { count.told(first + i); });
            };
            if (ru.history_type == THRML_I64) each(static_cast<const int64_t*>(ru.history));
            else each(static_cast<const int32_t*>(ru.history));
        }
        wait_copies<0>();  // before any write, which may be in place
        __syncthreads();
        if (has_bias) {
            // the first of a category's entries finishes it for all of them
            for (int32_t e = tid; e < n_bias; e += ADJUST_THREADS) {
                const int32_t id = ids[e];
                const uint32_t at = id - (begin - ahead);
                if (id < 0 || at >= static_cast<uint32_t>(stop - begin) || (e > 0 && ids[e - 1] == id)) continue;
                float sum = ru.bias_values[b0 + e];
                for (int32_t i = e + 1; i < n_bias && ids[i] == id; ++i) sum += ru.bias_values[b0 + i];
                float x = e == tid ? logit : to_float(logits[id]);
                if (has_history) {
                    const uint32_t c = count.at(at);
                    if (c) x = penalise(x, c & ~Counts<BITS>::IN_PROMPT);
                }
                x += sum;
                if (mask && !((mask[id >> 5] >> (id & 31)) & 1u)) x = -INFINITY;
                out[id] = from_float<T>(x);
            }
        }
#pragma unroll 1
        for (int s = s0; s < s1; ++s) {
            const int32_t at = place(s), k = at - ahead;
            if (at >= stop) break;
            uint4& raw = tile[s * ADJUST_THREADS + tid];
            if (has_history) {
                constexpr int WORDS = V * BITS / 32;  // of a piece's counts: 2, 4 or 8
                const uint32_t* w = reinterpret_cast<const uint32_t*>(counts) + (at - begin) / Counts<BITS>::PER_WORD;
                uint32_t some = 0u;  // a bit per word
#pragma unroll
                for (int j = 0; j < WORDS; j += 2) {
                    const uint2 q = *reinterpret_cast<const uint2*>(w + j);
                    some |= (q.x ? 1u << j : 0u) | (q.y ? 2u << j : 0u);
                }
                // A logit is rounded to its type once: what is penalised and not biased is final; what is biased is not written below.
                while (some) {
                    const int word = __ffs(some) - 1;
                    some &= some - 1u;
#pragma unroll
                    for (int h = 0; h < Counts<BITS>::PER_WORD; ++h) {
                        const int j = word * Counts<BITS>::PER_WORD + h;
                        const uint32_t c = (w[word] >> Counts<BITS>::shift(h)) & Counts<BITS>::ALL;
                        T& x = reinterpret_cast<T*>(&raw)[j];
                        if (c) x = from_float<T>(penalise(to_float(x), c & ~Counts<BITS>::IN_PROMPT));
                    }
                }
            }
            uint4 bits = raw;
            if (mask) {
                const int32_t k0 = max(k, 0);  // the first piece of a row may begin before it
                const uint32_t* w = mask_words + (k0 >> 5) - first_word;
                uint32_t open = w[0] >> (k0 & 31);
                if ((k0 & 31) + V > 32) open |= w[1] << (32 - (k0 & 31));  // behind the row's last word: bits that are not used
                bits = close_16<T>(bits, open << (k0 - k));
            }
            const uint32_t done = has_bias ? biased[(at - from) >> 5] >> ((at - from) & 31) & ((1u << V) - 1u) : 0u;  // V positions lie in one word
            pieces.store(out, at, bits, wide, done);
        }
    };
    if (h1 - h0 < 1 << 15 && penalties.has_reciprocal()) {
        pass(Count<16>{}, 0, ADJUST_PIECES, from, to);
    } else {
        const int32_t half = from + ADJUST_PIECES / 2 * ADJUST_THREADS * V;
        pass(Count<32>{}, 0, ADJUST_PIECES / 2, from, min(to, half));
        if (half < to) {
            __syncthreads();  // the counts are read
            pass(Count<32>{}, ADJUST_PIECES / 2, ADJUST_PIECES, half, to);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// The draw of a category.
//
// score = beta l - log(-log u) exceeds a bound B exactly when -ln u < exp(beta l - B), and -ln u >= 1 - u: so a category whose
// 1 - u lies above exp(beta l - B) cannot be the largest once B is a score that some category reaches.  That test costs one
// hardware exponential and no logarithm, and nearly every category fails it.  The ones that pass get their score in f64
// (where two scores that f32 cannot tell apart have an order), which decides.  B starts from approximate scores of each
// thread's first categories, lowered by more than their error, and rises with the scores found, shared in the CTA.
// Ten dependent rounds of the generator serve four categories: half of 23 M warp instructions for 256 x 131072 bf16, 20 us at full
// issue, of which they reach 49 % (waits for memory, for the rounds' results and at barriers hold the rest): 52 us with two CTAs a
// row, 60 with four and 75 with eight, whose starts and first, loose bounds cost more than they spread.  Four CTAs of 128
// threads, which spread evenly over the SMs: 56; 512 x 32000 38 instead of 33, though 2048 x 5003 34 instead of 40.
// ---------------------------------------------------------------------------------------------------------
constexpr int DRAW_THREADS = 256, DRAW_GROUP = 8;  // categories that share two generator calls
constexpr int DRAW_AT_ONCE = 2;                     // groups of a thread whose logits are in flight together

struct DrawArgs {
    const void* logits;
    const float* beta;
    const float* noise;
    int64_t* out;
    int64_t pitch, noise_pitch;
    int32_t cols, share, per_row;  // categories per CTA, CTAs (= a cluster) per row
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

// -log(-log u) to well within 1e-3, for u in (0, 1); near 1 the inner logarithm is a series in 1 - u.
__device__ __forceinline__ float gumbel_fast(float u) {
    const float rest = 1.0f - u, t = rest < 0.125f ? rest * fmaf(rest, fmaf(rest, 0.33333333f, 0.5f), 1.0f) : -__logf(u);
    return -__logf(t);
}

// The scores in f64 of those of DRAW_GROUP categories that reach the bound, out of line: few turns have any.
template <class T>
__device__ __noinline__ void weigh(Best& best, int32_t* bound, const DrawArgs& g, const T* logits, const float* noise, float beta, int64_t row, int32_t k, int32_t to) {
    for (int h = 0; h < DRAW_GROUP && k + h < to; h += 4) {
        U4 w{};
        if (!noise && beta != INFINITY) w = philox4x32_10_rk(g.row_offset + static_cast<uint32_t>(row), 0u, static_cast<uint32_t>(k + h) >> 2, TAG_DRAW, g.rk);
        for (int j = h; j < h + 4 && k + j < to; ++j) {
            const float l = to_float(logits[k + j]);
            if (!(l > -INFINITY)) continue;  // masked, or not a number
            double score = l;
            if (beta != INFINITY) {
                const float u = noise ? noise[k + j] : u23_open(pick(w, j - h));
                const float b = from_ordered(*static_cast<volatile int32_t*>(bound));
                if (beta * l + gumbel_fast(u) + (1e-2f + 1e-5f * fabsf(beta * l)) < b) continue;
                score = __dsub_rn(__dmul_rn(beta, l), log(-log(static_cast<double>(u))));
            }
            best.take(score, k + j);
            if (score > -INFINITY) atomicMax(bound, ordered(__double2float_rd(score)));
        }
    }
}

template <class T, bool GIVEN>
__global__ void __launch_bounds__(DRAW_THREADS, 4) k_draw(const __grid_constant__ DrawArgs g) {
    __shared__ Best warps[DRAW_THREADS / 32], ctas[8];
    __shared__ int32_t bound;
    const int tid = threadIdx.x, lane = tid & 31;
    const int64_t row = g.per_row == 1 ? blockIdx.x : blockIdx.x / g.per_row;
    const int32_t part = static_cast<int32_t>(blockIdx.x - row * g.per_row), from = part * g.share, to = min(g.cols, from + g.share);
    if (g.per_row > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const float beta = g.beta ? g.beta[row] : 1.0f;
    const bool greedy = beta == INFINITY;
    const T* logits = static_cast<const T*>(g.logits) + row * g.pitch;
    const float* noise = GIVEN ? g.noise + row * g.noise_pitch : nullptr;
    const bool wide = on_16(logits + from);  // shares are multiples of DRAW_GROUP
    const float b2 = beta * LOG2E;

    constexpr int PIECES = DRAW_GROUP / VEC<T>;
    struct Group {
        uint4 raw[PIECES];
    };
    // The logits of a group as they lie in memory; what lies behind the share is masked.
    auto load = [&](int32_t k) {
        Group q;
        if (wide && k + DRAW_GROUP <= to) {
#pragma unroll
            for (int h = 0; h < PIECES; ++h) q.raw[h] = *reinterpret_cast<const uint4*>(logits + k + h * VEC<T>);
        } else {
#pragma unroll
            for (int h = 0; h < PIECES; ++h) {
                q.raw[h] = nothing_16<T>();
#pragma unroll
                for (int j = 0; j < VEC<T>; ++j)
                    if (k + h * VEC<T> + j < to) reinterpret_cast<T*>(&q.raw[h])[j] = logits[k + h * VEC<T> + j];
            }
        }
        return q;
    };
    // Four uniforms.  From the key: 1 + n 2^-23, where u = (n + 1/2) 2^-23; given: u.
    auto draw = [&](int32_t k, float (&f)[4]) {
        if (GIVEN) {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = k + j < to ? noise[k + j] : 0.0f;
        } else {
            const U4 w = philox4x32_10_rk(g.row_offset + static_cast<uint32_t>(row), 0u, static_cast<uint32_t>(k) >> 2, TAG_DRAW, g.rk);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(__funnelshift_r(pick(w, j), 0x7fu, 9));  // the exponent of 1, then n
        }
    };
    // Whether any of a group can exceed the bound `b`.
    auto reaches = [&](const Group& q, int32_t k, float b) {
        bool some = false;
        // c = the bound in base 2, lowered by the roundings of c and of beta l log2(e), 2^-22 of their sizes (a category 60 or
        // more below c is out of reach of them), and by the exponential's error
        const float c = b * LOG2E, low = b == INFINITY ? b : c - (fabsf(c) + 60.0f) * 0x1p-21f - 1e-5f;
        float l[DRAW_GROUP];
#pragma unroll
        for (int h = 0; h < PIECES; ++h) {
            float v[VEC<T>];
            unpack_16<T>(q.raw[h], v);
#pragma unroll
            for (int j = 0; j < VEC<T>; ++j) l[h * VEC<T> + j] = v[j];
        }
        if (greedy) {
#pragma unroll
            for (int j = 0; j < DRAW_GROUP; ++j) some |= l[j] >= b;
            return some;
        }
        if (b2 == INFINITY) return true;  // a beta near the largest f32: base 2 cannot hold it, and weigh() decides
#pragma unroll
        for (int h = 0; h < DRAW_GROUP; h += 4) {
            float f[4];
            draw(k + h, f);
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                const float2 a = fma_2(make_float2(l[h + j], l[h + j + 1]), both(b2), both(-low)), e = make_float2(exp2_fast(a.x), exp2_fast(a.y));
                // 1 - u = 2 - f - 2^-24 for the key's; the rounding of 2 - 2^-22 - e is covered.  What is no number passes here.
                if (GIVEN) {
                    some |= !(1.0f - f[j] > e.x) | !(1.0f - f[j + 1] > e.y);
                } else {
                    const float2 least = fma_2(e, both(-1.0f), both(2.0f - 0x1p-22f));
                    some |= !(f[j] < least.x) | !(f[j + 1] < least.y);
                }
            }
        }
        return some;
    };

    Best best{0.0, -1};
    if (beta >= 0.0f) {
        // A first bound, from each thread's first group.
        float first = -INFINITY;
        const int32_t k0 = from + tid * DRAW_GROUP, step = DRAW_THREADS * DRAW_GROUP;
        if (k0 < to) {
            const Group q = load(k0);
#pragma unroll
            for (int h = 0; h < DRAW_GROUP; h += 4) {
                float f[4];
                if (!greedy) draw(k0 + h, f);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float l = to_float(reinterpret_cast<const T*>(q.raw)[h + j]);
                    float s = l;
                    if (!greedy) {
                        const float z = beta * l;
                        s = z + gumbel_fast(GIVEN ? f[j] : (f[j] - 1.0f) + 0x1p-24f) - (1e-2f + 1e-5f * fabsf(z));
                    }
                    if (l > -INFINITY && s < INFINITY) first = fmaxf(first, s);
                }
            }
        }
        const int32_t highest = __reduce_max_sync(0xffffffffu, ordered(first));
        if (tid == 0) bound = ordered(-INFINITY);
        __syncthreads();
        if (lane == 0) atomicMax(&bound, highest);
        __syncthreads();
        for (int32_t k = k0; k < to; k += DRAW_AT_ONCE * step) {
            Group q[DRAW_AT_ONCE];
#pragma unroll
            for (int t = 0; t < DRAW_AT_ONCE; ++t)
                if (k + t * step < to) q[t] = load(k + t * step);
#pragma unroll
            for (int t = 0; t < DRAW_AT_ONCE; ++t)
                if (k + t * step < to && reaches(q[t], k + t * step, from_ordered(*static_cast<volatile int32_t*>(&bound))))
                    weigh<T>(best, &bound, g, logits, noise, beta, row, k + t * step, to);
        }
    }
    for (int d = 16; d; d >>= 1) {
        const double s = __shfl_xor_sync(0xffffffffu, best.score, d);
        const int32_t k = __shfl_xor_sync(0xffffffffu, best.k, d);
        best.take(s, k);
    }
    if (lane == 0) warps[tid >> 5] = best;
    __syncthreads();
    if (tid < 32) {
        best = warps[tid % (DRAW_THREADS / 32)];
        for (int d = 16; d; d >>= 1) {
            const double s = __shfl_xor_sync(0xffffffffu, best.score, d);
            const int32_t k = __shfl_xor_sync(0xffffffffu, best.k, d);
            best.take(s, k);
        }
    }
    if (g.per_row > 1) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // the row's first CTA has started
        if (tid == 0) {
            const uint32_t at = dense::peer_addr(dense::smem_u32(&ctas[part]), 0);
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(best.score) : "memory");
            asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at + static_cast<uint32_t>(offsetof(Best, k))), "r"(best.k) : "memory");
        }
        dense::cluster_sync_all();
        for (int c = 1; c < g.per_row; ++c) best.take(ctas[c].score, ctas[c].k);
    }
    if (part == 0 && tid == 0) g.out[row] = best.k;
}

// ---------------------------------------------------------------------------------------------------------
// Distillation.
//
// With z = beta * logits, the row's softmax q = exp(z - lse) and the teacher's p over the listed entries:
//     loss = sum_j p_j (log p_j - z_id(j) + lse),   d loss / d logits = beta (q - p).
// Two kernels (one where rows are few).  k_softmax streams the rows: lse (loss), weight * beta * q from a given lse (grad), or both (step), where the
// second pass finds the row in L2 (a CTA, or each of a cluster of up to eight, has 64 KB of it).  2048 x 131072 bf16: gradient
// 152 us = 6.3 TB/s, the rate of a copy.  4096 x 32768 bf16: step 90 us = 5.3 TB/s.  k_listed then has one warp, or
// four, for each row's list: the loss, and the few gradients that p changes.  What was measured and dropped (4096 x 32768 bf16,
// 64 listed, a step): rows held in registers or in shared memory, once per CTA or in rings of two and three rows, the
// list inside the same kernel: 125 to 200 us, since the list's chain of small loads, each as slow as a full memory system
// makes it, held up the rows.
// Per element a difference, a product or multiply-add and one hardware exponential a pass, in base 2, two elements an instruction where there is
// one; probabilities below 2^-126 count as 0.
// ---------------------------------------------------------------------------------------------------------
constexpr int SOFTMAX_THREADS = 256;
constexpr int64_t SOFTMAX_BYTES = 64 << 10;  // of a row per CTA
constexpr int LIST_WARPS = 4;
constexpr int64_t APART_CTAS = 64, APART_BYTES = int64_t{16} << 30;  // see launch_distill
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
    int64_t rows, pitch, ids_pitch, teacher_pitch, grad_pitch;
    int32_t cols, top, ids_type, teacher_type;
    float beta, per_beta;
    int32_t share, per_row;  // positions of a row per CTA, CTAs per row
    bool joined;
};

// beta's range: a finite difference of two logits that f32 cannot hold is then weight 0, and base 2 does not overflow.
constexpr float BETA_MIN = 0x1p-100f, BETA_MAX = 0x1p100f;
// The largest |lse| that a gradient takes as it is: its rounding is a relative error of q of up to 2^-17 there and grows with it, so
// the sums of a row beyond (a mask's fill that leaves nothing, mostly) are formed again, which costs another reading of the row.
constexpr float LSE_KEPT = 256.0f;

// A part of a softmax's sum: 2^(b2 (l - ref)) over its logits l.  ref is one of them, -infinity while there is nothing.  The
// difference comes first: it is exact next to ref, however large both are, where rounded products would lie apart.
struct Partial {
    float ref, sum;
    __device__ __forceinline__ void join(Partial o, float b2) {
        const float top = fmaxf(ref, o.ref);
        // a part at -infinity adds nothing; its sum is 0, or NaN when it has met one
        const float a = ref == top || ref == -INFINITY ? 1.0f : exp2_fast((ref - top) * b2);
        const float b = o.ref == top || o.ref == -INFINITY ? 1.0f : exp2_fast((o.ref - top) * b2);
        sum = fmaf(sum, a, o.sum * b);
        ref = top;
    }
};

// The larger of the even and of the odd elements of 16 bytes.  A bf16 in the upper half of a word is compared with the lower half
// as further fraction bits, which do not change which is the largest; upper() drops them.  What is no number, or is made one by
// those bits, gives way (an infinity that is missed so shows in the sum).
template <class T>
__device__ __forceinline__ void larger_16(float& a, float& b, const uint4& raw) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            a = fmaxf(a, __uint_as_float(w[i]));
            b = fmaxf(b, __uint_as_float(w[i] << 16));
        } else if constexpr (std::is_same<T, float>::value) {
            if (i & 1) b = fmaxf(b, __uint_as_float(w[i]));
            else a = fmaxf(a, __uint_as_float(w[i]));
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            a = fmaxf(a, f.x), b = fmaxf(b, f.y);
        }
    }
}
template <class T>
__device__ __forceinline__ float upper(float a) {
    return std::is_same<T, __nv_bfloat16>::value ? __uint_as_float(__float_as_uint(a) & 0xffff0000u) : a;
}
__device__ __forceinline__ float warp_max(float x) { return from_ordered(__reduce_max_sync(0xffffffffu, ordered(x))); }
__device__ __forceinline__ float warp_total(float x) {
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}

// A warp's part of the share's sum, the share being dealt to THREADS threads: with the maximum of its logits first.
template <class T, int THREADS>
__device__ __noinline__ Partial sum_carefully(const Share<T>& s, float b2, int tid) {
    float high = -INFINITY, other = -INFINITY;
    for (int32_t i = tid; i < s.pieces; i += THREADS) larger_16<T>(high, other, s.piece(i));
    high = fmaxf(upper<T>(high), other);
    if (s.head + tid < s.first) high = fmaxf(high, to_float(s.row[s.head + tid]));
    if (s.tail + tid < s.stop) high = fmaxf(high, to_float(s.row[s.tail + tid]));
    high = warp_max(high);
    const float low = high == -INFINITY ? 0.0f : high;
    auto weight = [&](float l) { return exp2_fast((l - low) * b2); };
    float sum = 0.0f;
    for (int32_t i = tid; i < s.pieces; i += THREADS) {
        float v[VEC<T>];
        unpack_16<T>(s.piece(i), v);
#pragma unroll
        for (int j = 0; j < VEC<T>; ++j) sum += weight(v[j]);
    }
    if (s.head + tid < s.first) sum += weight(to_float(s.row[s.head + tid]));
    if (s.tail + tid < s.stop) sum += weight(to_float(s.row[s.tail + tid]));
    return Partial{high, warp_total(sum)};
}
template <class T, int THREADS>
__device__ __forceinline__ Partial sum_of(const Share<T>& s, float b2, int tid) {
    constexpr int V = VEC<T>, AT_ONCE = 4;
    // The reference is the largest of the warp's first pieces, which spares a pass for the maximum: sums are good as long as they
    // stay below 2^100, and what does not is done over with the maximum.
    float2 sums = both(0.0f), more = both(0.0f);
    float ref = -INFINITY, other = -INFINITY;
    if (tid < s.pieces) larger_16<T>(ref, other, s.piece(tid));
    ref = warp_max(fmaxf(upper<T>(ref), other));
    const float2 scale = both(b2), back = both(-ref);
    auto add = [&](const uint4& raw) {
        float v[V];
        unpack_16<T>(raw, v);
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const float2 a = mul_2(add_2(make_float2(v[j], v[j + 1]), back), scale), b = mul_2(add_2(make_float2(v[j + 2], v[j + 3]), back), scale);
            sums = add_2(sums, make_float2(exp2_fast(a.x), exp2_fast(a.y)));
            more = add_2(more, make_float2(exp2_fast(b.x), exp2_fast(b.y)));
        }
    };
    int32_t i = tid;
    for (; i + (AT_ONCE - 1) * THREADS < s.pieces; i += AT_ONCE * THREADS) {
        uint4 raw[AT_ONCE];
#pragma unroll
        for (int t = 0; t < AT_ONCE; ++t) raw[t] = s.piece(i + t * THREADS);
#pragma unroll
        for (int t = 0; t < AT_ONCE; ++t) add(raw[t]);
    }
    for (; i < s.pieces; i += THREADS) add(s.piece(i));
    float sum = (sums.x + sums.y) + (more.x + more.y);
    if (s.head + tid < s.first) sum += exp2_fast((to_float(s.row[s.head + tid]) - ref) * b2);
    if (s.tail + tid < s.stop) sum += exp2_fast((to_float(s.row[s.tail + tid]) - ref) * b2);
    sum = warp_total(sum);
    if (!(sum < 0x1p100f)) return sum_carefully<T, THREADS>(s, b2, tid);  // an infinite reference among them
    return Partial{ref, sum};
}
// A share's sum by a CTA of THREADS threads (or a warp), of whose warps it joins the parts.
template <class T, int THREADS>
__device__ __forceinline__ Partial sum_of_cta(const Share<T>& s, float b2, int tid, Partial* warps) {
    Partial p = sum_of<T, THREADS>(s, b2, tid);
    if (THREADS > 32) {
        if ((tid & 31) == 0) warps[tid >> 5] = p;
        __syncthreads();
        p = warps[tid & (THREADS / 32 - 1)];
        for (int d = THREADS / 64; d; d >>= 1) p.join(Partial{__shfl_xor_sync(0xffffffffu, p.ref, d), __shfl_xor_sync(0xffffffffu, p.sum, d)}, b2);
        p = Partial{__shfl_sync(0xffffffffu, p.ref, 0), __shfl_sync(0xffffffffu, p.sum, 0)};
    }
    return p;
}
// The sum of a row from those of its cluster's CTAs, which have all arrived once at the cluster's barrier.
__device__ __forceinline__ Partial sum_of_cluster(Partial p, float b2, int tid, int32_t part, int32_t per_row, Partial* ctas) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every CTA of the row has started
    if (tid < per_row) {
        const uint32_t to = dense::peer_addr(dense::smem_u32(&ctas[part]), tid);
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(p.ref), "f"(p.sum) : "memory");
    }
    dense::cluster_sync_all();
    p = ctas[0];
    for (int c = 1; c < per_row; ++c) p.join(ctas[c], b2);
    return p;
}
// The sums of a row whose lse a gradient does not take as it is, out of line: by the CTA (or warp) alone, which reads all of the row.
template <class T, int THREADS>
__device__ __noinline__ Partial sum_again(const T* logits, int32_t cols, float b2, int tid, Partial* warps) {
    return sum_of_cta<T, THREADS>(Share<T>(logits, cols, 0, cols + VEC<T>), b2, tid, warps);
}
// And by the row's cluster, of which the CTA reads its share.
template <class T>
__device__ __noinline__ Partial sum_again_together(const T* logits, int32_t cols, int32_t share, float b2, int tid, int32_t part, int32_t per_row, Partial* warps, Partial* ctas) {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const Partial p = sum_of_cta<T, SOFTMAX_THREADS>(Share<T>(logits, cols, part * share, share), b2, tid, warps);
    return sum_of_cluster(p, b2, tid, part, per_row, ctas);
}

// q of a row, from the joined parts of its sum or from its lse: 2^(b2 (l - ref) - sum2).
struct Softmax {
    float ref, sum2;  // a logit, or a number near one, and log2 of the sum relative to it
    bool empty;
    __device__ __forceinline__ static Softmax of(Partial p) { return of(p.ref, p.sum == INFINITY || (p.ref == -INFINITY && p.sum != 0.0f) ? NAN : log2f(p.sum)); }
    __device__ __forceinline__ static Softmax of(float ref, float sum2) { return Softmax{ref, sum2, ref == -INFINITY && sum2 == -INFINITY}; }
    // lse as beta ref + a rest (ref is near lse / beta, whatever per_beta's rounding), so that here too the difference comes first.
    __device__ __forceinline__ static Softmax of_lse(float lse, float beta, float per_beta) {
        const float ref = lse * per_beta;
        return Softmax{ref, LOG2E * fmaf(-beta, ref, lse), false};
    }
    // What is taken from a logit, and from the exponent: a row with nothing has q = 0.
    __device__ __forceinline__ float back() const { return empty ? 0.0f : ref; }
    __device__ __forceinline__ float less() const { return empty ? INFINITY : sum2; }
    __device__ __forceinline__ float q(float l, float b2) const { return exp2_fast(fmaf(l - back(), b2, -less())); }
};

// Slots of a list's table, a power of two: at most half of them are taken.
__host__ __device__ inline int32_t list_slots(int32_t top) {
    int32_t slots = 32;
    while (slots < 2 * top) slots *= 2;
    return slots;
}

// Shared memory of a row's list: ids, p, z and, for a gradient, the table and a bit per entry.
__host__ __device__ inline int32_t list_words(int32_t top, int mode) { return 3 * top + (mode == LOSS ? 0 : list_slots(top) + (top + 31) / 32); }

// A row's list, by a team of threads (`members`, whole warps, this thread number `me`; meet() is their barrier), whose arrays lie in
// shared memory: the loss, and the gradient's listed entries among [low, high) once more, with p subtracted before the rounding.
// sums() waits for the row's sums and gradient and gives its Softmax.  Categories that are listed more than once are found with a
// table by open addressing (a step of 256 rows of 1024 entries 84 us; comparing all pairs 980).  The entry that got the slot
// writes for all of them; which one that was changes nothing, as their sum is taken over the list in one order.
template <class T, int MODE, class Meet, class Sums>
__device__ __forceinline__ void finish_list(const DistillArgs& g, int64_t row, float weight, int32_t* id, int me, int members, bool tells, int32_t low, int32_t high, Meet meet, Sums sums) {
    const int lane = threadIdx.x & 31;
    float* p = reinterpret_cast<float*>(id + g.top);  // the teacher's logits, then their softmax over the listed (differences first, as in Partial); id: -1 = not listed
    float* z = p + g.top;                             // the student's logits there
    int32_t* table = reinterpret_cast<int32_t*>(z + g.top);  // numbers of entries, -1 = free
    const int32_t slots = list_slots(g.top);
    uint32_t* more = reinterpret_cast<uint32_t*>(table + slots);  // bit j: entry j is not the only one of its category
    uint32_t writes = 0;                                          // bit n: this thread's entry n writes for its category (32 at most)
    const T* logits = static_cast<const T*>(g.logits) + row * g.pitch;
    const float b2 = g.beta * LOG2E;
    bool some = false;
    float most = -INFINITY, total = 0.0f;
    if (weight != 0.0f) {
        if (MODE != LOSS)
            for (int i = me; i < slots + (g.top + 31) / 32; i += members) table[i] = i < slots ? -1 : 0;
#pragma unroll 4
        for (int j = me; j < g.top; j += members) {
            const int64_t k = load_as_int(g.ids, g.ids_type, row * g.ids_pitch + j);
            const float t = load_as_float(g.teacher, g.teacher_type, row * g.teacher_pitch + j);
            const bool listed = k >= 0 && k < g.cols && !(t == -INFINITY);
            id[j] = listed ? static_cast<int32_t>(k) : -1;
            p[j] = t;
            if (listed) z[j] = to_float(logits[k]);
        }
    }
    meet();
    if (weight != 0.0f) {
        if (MODE != LOSS)
            for (int j = me, n = 0; j < g.top; j += members, ++n) {
                const int32_t k = id[j];
                if (k < low || k >= high) continue;  // -1 among them
                for (uint32_t at = static_cast<uint32_t>(k) * 2654435761u >> 16, tries = 0; tries < static_cast<uint32_t>(slots); ++at, ++tries) {
                    const int32_t held = atomicCAS(table + (at & (slots - 1)), -1, j);
                    if (held == -1) writes |= 1u << n;
                    else if (id[held] == k) atomicOr(more + (held >> 5), 1u << (held & 31));
                    else continue;
                    break;
                }
            }
        for (int j = lane; j < g.top; j += 32)
            if (id[j] >= 0) {
                most = fmaxf(most, p[j]);
                some = true;
            }
        some = __any_sync(0xffffffffu, some);
        most = warp_max(most);
        for (int j = lane; j < g.top; j += 32) total += id[j] >= 0 ? expf(g.beta * (p[j] - most)) : 0.0f;  // each warp of a team the same sum
        total = warp_total(total);
    }
    meet();
    if (weight != 0.0f)
        for (int j = me; j < g.top; j += members) p[j] = id[j] >= 0 ? expf(g.beta * (p[j] - most)) / total : 0.0f;
    meet();
    const Softmax soft = sums();
    T* grad = MODE == LOSS ? nullptr : static_cast<T*>(g.grad) + row * g.grad_pitch;
    if (weight == 0.0f || !some) {
        if (MODE != GRAD && tells && me == 0) g.loss[row] = 0.0f, g.lse_out[row] = 0.0f;
        if (MODE != LOSS && weight != 0.0f)
            for (int32_t k = low + me; k < high; k += members) grad[k] = from_float<T>(0.0f);
        return;
    }
    if (MODE != GRAD) {
        meet();  // every thread has the row's sum, which may lie where the loss goes
        if (tells && me < 32) {
            const float log_sum = soft.sum2 * LN2;
            float loss = 0.0f;
            for (int j = lane; j < g.top; j += 32)
                if (id[j] >= 0 && !(p[j] == 0.0f)) {
                    const float gap = fmaf(-0.5f, soft.ref, 0.5f * z[j]);  // half of the difference, which f32 may not hold
                    loss += soft.empty ? INFINITY : p[j] * (logf(p[j]) + log_sum) + (gap == -INFINITY ? INFINITY : -2.0f * p[j] * g.beta * gap);
                }
            loss = warp_total(loss);
            if (lane == 0) g.loss[row] = loss;
            if (lane == 0) g.lse_out[row] = soft.empty ? -INFINITY : fmaf(g.beta, soft.ref, log_sum);
        }
    }
    if (MODE != LOSS)
        for (int j = me, n = 0; j - lane < g.top; j += members, ++n) {  // whole warps
            const bool mine = writes >> n & 1;
            float share = mine ? p[j] : 0.0f;
            for (unsigned several = __ballot_sync(0xffffffffu, mine && (more[j >> 5] >> (j & 31) & 1)); several; several &= several - 1) {
                const int from = __ffs(several) - 1;
                const int32_t k = id[j - lane + from];
                float sum = 0.0f;
                for (int t = lane; t < g.top; t += 32) sum += id[t] == k ? p[t] : 0.0f;
                sum = warp_total(sum);
                if (lane == from) share = sum;
            }
            if (mine) grad[id[j]] = from_float<T>(weight * g.beta * (soft.q(z[j], b2) - share));
        }
}

// The rows' sums (reference into loss, log2 of the sum into lse_out, from where k_listed takes them), and weight * beta * q into
// grad.  WHOLE: with few rows the list too, each CTA its own share's (a launch less: a step of 33 x 5003, 20 listed, 17.7 -> 14.6 us as
// the host sees it, which the choice is made for, though 6.4 -> 7.0 on the GPU, as in a replayed graph; 33 x 131072, 1024 listed, a gradient 42 -> 12 us).
template <class T, int MODE, bool WHOLE>
__global__ void __launch_bounds__(SOFTMAX_THREADS, 4) k_softmax(const __grid_constant__ DistillArgs g) {
    constexpr int V = VEC<T>, AT_ONCE = 4;
    __shared__ Partial warps[SOFTMAX_THREADS / 32], ctas[8];
    const int tid = threadIdx.x, lane = tid & 31;
    const int64_t row = g.per_row == 1 ? blockIdx.x : blockIdx.x / g.per_row;
    const int32_t part = static_cast<int32_t>(blockIdx.x - row * g.per_row);
    const bool joined = g.joined;  // the CTAs of a row form a cluster
    if (!WHOLE) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (MODE != GRAD && joined) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const float weight = g.weight ? g.weight[row] : 1.0f;  // 0: padding, nothing of the row is read
    const T* logits = static_cast<const T*>(g.logits) + row * g.pitch;
    const Share<T> s(logits, g.cols, part * g.share, g.share);
    const float b2 = g.beta * LOG2E;
    Softmax soft{};
    if (MODE == GRAD) {
        if (weight != 0.0f) {
            const float lse = g.lse_in[row];
            if (!(fabsf(lse) > LSE_KEPT)) soft = Softmax::of_lse(lse, g.beta, g.per_beta);
            else if (joined) soft = Softmax::of(sum_again_together<T>(logits, g.cols, g.share, b2, tid, part, g.per_row, warps, ctas));
            else soft = Softmax::of(sum_again<T, SOFTMAX_THREADS>(logits, g.cols, b2, tid, warps));
        }
    } else {
        Partial p{-INFINITY, 0.0f};
        if (weight != 0.0f) p = sum_of_cta<T, SOFTMAX_THREADS>(s, b2, tid, warps);  // weight is the row's
        if (joined) p = sum_of_cluster(p, b2, tid, part, g.per_row, ctas);
        soft = Softmax::of(p);
        if (!WHOLE && part == 0 && tid == 0) g.loss[row] = soft.ref, g.lse_out[row] = soft.sum2;
    }
    auto write = [&] {
        T* grad = static_cast<T*>(g.grad) + row * g.grad_pitch;
        const float scale = weight * g.beta;
        const bool zeros = weight == 0.0f;
        auto value = [&](float l) { return scale * soft.q(l, b2); };
        if (tid < s.first - s.head) grad[s.head + tid] = from_float<T>(zeros ? 0.0f : value(to_float(logits[s.head + tid])));
        if (tid < s.stop - s.tail) grad[s.tail + tid] = from_float<T>(zeros ? 0.0f : value(to_float(logits[s.tail + tid])));
        if ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(logits)) & 15u) {
            for (int32_t k = s.first + tid; k < s.tail; k += SOFTMAX_THREADS) grad[k] = from_float<T>(zeros ? 0.0f : value(to_float(logits[k])));
            return;
        }
        uint4* out = reinterpret_cast<uint4*>(grad + s.first);
        if (zeros) {
            for (int32_t i = tid; i < s.pieces; i += SOFTMAX_THREADS) __stcs(out + i, make_uint4(0u, 0u, 0u, 0u));
            return;
        }
        const float2 back = both(-soft.back()), less = both(-soft.less());
        auto gradient = [&](const uint4& raw) {
            float x[V];
            unpack_16<T>(raw, x);
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float2 a = fma_2(add_2(make_float2(x[j], x[j + 1]), back), both(b2), less);
                const float2 y = mul_2(make_float2(exp2_fast(a.x), exp2_fast(a.y)), both(scale));
                x[j] = y.x, x[j + 1] = y.y;
            }
            return pack_16<T>(x);
        };
        int32_t i = tid;
        for (; i + (AT_ONCE - 1) * SOFTMAX_THREADS < s.pieces; i += AT_ONCE * SOFTMAX_THREADS) {
            uint4 raw[AT_ONCE];
#pragma unroll
            for (int t = 0; t < AT_ONCE; ++t) raw[t] = s.piece(i + t * SOFTMAX_THREADS);
#pragma unroll
            for (int t = 0; t < AT_ONCE; ++t) __stcs(out + i + t * SOFTMAX_THREADS, gradient(raw[t]));
        }
        for (; i < s.pieces; i += SOFTMAX_THREADS) __stcs(out + i, gradient(s.piece(i)));
    };
    if (MODE != LOSS) write();
    if (WHOLE) {
        extern __shared__ int32_t listed_smem[];
        __syncthreads();  // the share is written
        finish_list<T, MODE>(g, row, weight, listed_smem, tid, SOFTMAX_THREADS, part == 0, s.head, s.stop, [] { __syncthreads(); }, [&] { return soft; });
    }
}

// The lists: a team of one warp per row, or of all LIST_WARPS where lists are long.  Everything up to the rows' sums is done while
// k_softmax is still at work.
template <class T, int MODE>
__global__ void __launch_bounds__(32 * LIST_WARPS) k_listed(const __grid_constant__ DistillArgs g, int32_t teams) {
    extern __shared__ int32_t listed_smem[];
    __shared__ Partial warps[LIST_WARPS];
    const int warp = threadIdx.x >> 5;
    const int team = teams == 1 ? 0 : warp, members = teams == 1 ? blockDim.x : 32, me = teams == 1 ? threadIdx.x : threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * teams + team;
    if (row >= g.rows) return;  // a warp of its own
    auto meet = [&] {
        if (teams == 1) __syncthreads();
        else __syncwarp();
    };
    const float weight = g.weight ? g.weight[row] : 1.0f;
    auto sums = [&] {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if (weight == 0.0f) return Softmax{};
        if (MODE != GRAD) return Softmax::of(g.loss[row], g.lse_out[row]);
        const float lse = g.lse_in[row], b2 = g.beta * LOG2E;
        if (!(fabsf(lse) > LSE_KEPT)) return Softmax::of_lse(lse, g.beta, g.per_beta);
        const T* logits = static_cast<const T*>(g.logits) + row * g.pitch;
        return Softmax::of(teams == 1 ? sum_again<T, 32 * LIST_WARPS>(logits, g.cols, b2, me, warps) : sum_again<T, 32>(logits, g.cols, b2, me, warps));
    };
    int32_t* arrays = listed_smem + list_words(g.top, MODE) * team;
    finish_list<T, MODE>(g, row, weight, arrays, me, members, true, 0, g.cols, meet, sums);
}

// Positions of a row, counted from the last 16-byte boundary at or before it (the most that any row has).
template <class T>
int64_t positions(const void* p, int64_t pitch, int64_t cols) {
    return aligned_to(p, 16) && pitch % VEC<T> == 0 ? cols : cols + VEC<T> - 1;
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

template <class T, int MODE>
int32_t launch_distill(thrml_ctx* ctx, cudaStream_t stream, DistillArgs g) {
    // CTAs per row: one for each 64 KB (256 KB where it is read once: 2048 rows of 131072 bf16 89 us, with 64 KB 111), eight at
    // most that have to join; with few rows more, so that the GPU is covered.
    const int64_t span = positions<T>(g.logits, g.pitch, g.cols), held = (MODE == LOSS ? 4 : 1) * SOFTMAX_BYTES / sizeof(T);
    int64_t per_row = (span + held - 1) / held;
    // A gradient's CTAs work apart, and each forms the sums of a row whose lse it does not take by itself.  Where that would be more than
    // APART_BYTES (6 ms) of reading for rows of more than APART_CTAS, they share the sums as in the other modes, by eight CTAs a row at
    // most.  f32, us a gradient, lse taken / not taken: a row of 8 million, apart, 15 / 5600; ten of them, shared, 228 / 380 (apart 106 / 56000).
    const bool whole_long = MODE == GRAD && per_row > APART_CTAS && g.rows * per_row > APART_BYTES / (span * static_cast<int64_t>(sizeof(T)));
    if (MODE != GRAD || whole_long) per_row = std::min<int64_t>(per_row, 8);
    while (per_row <= 4 && g.rows * per_row < 2 * ctx->sm_count && span / (2 * per_row) >= SOFTMAX_THREADS * VEC<T>) per_row *= 2;
    if (g.rows * per_row > INT32_MAX) return fail(THRML_ERR_INVALID_ARG, "too many rows of this length in one call");
    g.per_row = static_cast<int32_t>(per_row);
    g.share = static_cast<int32_t>(((span + per_row - 1) / per_row + VEC<T> - 1) / VEC<T> * VEC<T>);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    cfg.gridDim = dim3(static_cast<unsigned>(g.rows * per_row));
    cfg.blockDim = dim3(SOFTMAX_THREADS);
    cfg.stream = stream;
    cfg.attrs = &attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {static_cast<unsigned>(per_row), 1, 1};
    g.joined = (MODE != GRAD || whole_long) && per_row > 1;
    cfg.numAttrs = g.joined ? 1 : 0;
    const size_t list_bytes = 4 * static_cast<size_t>(list_words(g.top, MODE));
    if (g.rows * per_row <= 2 * ctx->sm_count || whole_long) {
        cfg.dynamicSmemBytes = list_bytes;
        CU_TRY(cudaLaunchKernelEx(&cfg, k_softmax<T, MODE, true>, g));
        return THRML_OK;
    }
    CU_TRY(cudaLaunchKernelEx(&cfg, k_softmax<T, MODE, false>, g));
    // The lists start while the last rows are still at work; what they need of those they wait for.
    const int32_t teams = g.top <= 64 ? LIST_WARPS : 1;  // a warp for 64 entries; four for 128 save 7 us of 188 (gradient, 2048 x 131072)
    cfg.gridDim = dim3(static_cast<unsigned>((g.rows + teams - 1) / teams));
    cfg.blockDim = dim3(32 * LIST_WARPS);
    cfg.dynamicSmemBytes = list_bytes * teams;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    CU_TRY(cudaLaunchKernelEx(&cfg, k_listed<T, MODE>, g, teams));
    return THRML_OK;
}

int32_t distill(thrml_ctx* ctx, void* stream, int mode, int64_t rows, int32_t type, DistillArgs g) {
    if (int32_t rc = check_rows("logits", rows, g.cols, g.logits, type, g.pitch)) return rc;
    if (mode != LOSS) {
        if (int32_t rc = check_rows("grad", rows, g.cols, g.grad, type, g.grad_pitch)) return rc;
        if (rows && g.grad == g.logits) return fail(THRML_ERR_INVALID_ARG, "grad must not be the logits themselves");
        if (overlap(Area(g.grad, type_size(type), rows, g.cols, g.grad_pitch), Area(g.logits, type_size(type), rows, g.cols, g.pitch))) return fail(THRML_ERR_INVALID_ARG, "grad overlaps the logits");
    }
    if (g.top < 0 || g.top > TOP_MAX) return fail(THRML_ERR_INVALID_ARG, "top is not within 0 and 1024");
    if (!is_index_type(g.ids_type)) return fail(THRML_ERR_INVALID_ARG, "ids: the element type is not an index type");
    if (!is_float_type(g.teacher_type)) return fail(THRML_ERR_INVALID_ARG, "teacher: the element type is not a float type");
    if (g.ids_pitch < g.top || g.teacher_pitch < g.top) return fail(THRML_ERR_INVALID_ARG, "ids, teacher: the pitch is smaller than top");
    if (!(g.beta >= BETA_MIN && g.beta <= BETA_MAX)) return fail(THRML_ERR_INVALID_ARG, "beta is not within 2^-100 and 2^100");
    if (rows == 0) return THRML_OK;
    if (g.top && (!g.ids || !g.teacher)) return fail(THRML_ERR_INVALID_ARG, "ids, teacher: null pointer");
    if ((mode != GRAD && !g.loss) || (mode != GRAD && !g.lse_out) || (mode == GRAD && !g.lse_in)) return fail(THRML_ERR_INVALID_ARG, "loss, lse: null pointer");
    g.rows = rows;
    return for_type(type, [&](auto e) {
        using T = decltype(e);
        const auto st = static_cast<cudaStream_t>(stream);
        return mode == LOSS ? launch_distill<T, LOSS>(ctx, st, g) : mode == GRAD ? launch_distill<T, GRAD>(ctx, st, g) : launch_distill<T, STEP>(ctx, st, g);
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
    g.per_beta = 1.0f / beta;
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
        return for_type(type, [&](auto e) {
            using T = decltype(e);
            // As many CTAs as hold the row; with few rows, up to eight times as many, so that the GPU is covered.
            const int64_t span = positions<T>(logits, pitch, cols);
            int64_t per_row = (span + ADJUST_SHARE<T> - 1) / ADJUST_SHARE<T>;
            const int64_t most = 8 * per_row;
            while (2 * per_row <= most && rows * per_row < 2 * ctx->sm_count && span / (2 * per_row) >= 256) per_row *= 2;
            const int64_t share = ((span + per_row - 1) / per_row + 63) / 64 * 64;
            if (rows * per_row > INT32_MAX) return fail(THRML_ERR_INVALID_ARG, "too many rows of this length in one call");
            if (out != logits && overlap(Area(out, sizeof(T), rows, cols, out_pitch), Area(logits, sizeof(T), rows, cols, pitch)))
                return fail(THRML_ERR_INVALID_ARG, "out overlaps the logits without being them");
            // half of a full share's positions at a time (long histories) take 4 bytes each, the whole share 2
            const int64_t count_bytes = std::max<int64_t>(2 * share, 4 * std::min<int64_t>(share, ADJUST_SHARE<T> / 2));
            const AdjustArgs g{logits, out, pitch, out_pitch, static_cast<int32_t>(cols), static_cast<int32_t>(share), static_cast<int32_t>(per_row), static_cast<int32_t>(count_bytes / 4), *rules};
            const size_t smem = 16 * ADJUST_PIECES * ADJUST_THREADS + (rules->history ? count_bytes : 0) + (rules->bias_ids ? share / 8 : 0);
            if (int32_t rc = allow_shared<k_adjust<T>>(ctx, 16 * ADJUST_PIECES * ADJUST_THREADS + ADJUST_SHARE<T> * 2 + ADJUST_SHARE<T> / 8)) return rc;
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(static_cast<unsigned>(rows * per_row));
            cfg.blockDim = dim3(ADJUST_THREADS);
            cfg.dynamicSmemBytes = smem;
            cfg.stream = static_cast<cudaStream_t>(stream);
            CU_TRY(cudaLaunchKernelEx(&cfg, k_adjust<T>, g));
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
        // A CTA per row, or a cluster of up to eight where there are few rows for the GPU.
        int64_t per_row = 1;
        while (per_row < 8 && rows * per_row < 2 * ctx->sm_count && cols / (2 * per_row) >= DRAW_THREADS * DRAW_GROUP) per_row *= 2;
        const int64_t share = ((cols + per_row - 1) / per_row + DRAW_GROUP - 1) / DRAW_GROUP * DRAW_GROUP;
        if (rows * per_row > INT32_MAX) return fail(THRML_ERR_INVALID_ARG, "too many rows of this length in one call");
        const DrawArgs g{logits, beta, noise, out, pitch, noise_pitch, static_cast<int32_t>(cols), static_cast<int32_t>(share), static_cast<int32_t>(per_row),
                         static_cast<uint32_t>(row_offset), make_round_keys(key)};
        return for_type(type, [&](auto e) {
            using T = decltype(e);
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(static_cast<unsigned>(rows * per_row));
            cfg.blockDim = dim3(DRAW_THREADS);
            cfg.stream = static_cast<cudaStream_t>(stream);
            cudaLaunchAttribute cluster;
            cluster.id = cudaLaunchAttributeClusterDimension;
            cluster.val.clusterDim = {static_cast<unsigned>(per_row), 1, 1};
            cfg.attrs = &cluster;
            cfg.numAttrs = per_row > 1 ? 1 : 0;
            CU_TRY(cudaLaunchKernelEx(&cfg, noise ? k_draw<T, true> : k_draw<T, false>, g));
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
                           float* loss, float* lse, void* grad, int64_t grad_pitch) {
    return guarded(ctx, [&] {
        DistillArgs g = distill_args(logits, pitch, cols, top, ids, ids_type, ids_pitch, teacher, teacher_type, teacher_pitch, beta, weight);
        g.loss = loss;
        g.lse_out = lse;
        g.grad = grad;
        g.grad_pitch = grad_pitch;
        return distill(ctx, stream, STEP, rows, type, g);
    });
}

}  // extern "C"
