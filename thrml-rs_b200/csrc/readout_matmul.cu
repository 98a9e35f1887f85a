// The readout's 8-bit product: activations quantised with one scale per token, weights with one scale per channel, the sum
// of products exact in 32-bit integers on the tensor cores (tcgen05 kind::i8, accumulators in tensor memory).
#include <algorithm>

#include "readout.cuh"
#include "tensor_core.cuh"

using namespace thrml;
using namespace thrml::readout;

namespace {

template <int N>
__device__ __forceinline__ bool aligned_for(const void* p) { return (reinterpret_cast<uintptr_t>(p) % N) == 0; }

// ---------------------------------------------------------------------------------------------------------
// Rows in 8 bits.
// ---------------------------------------------------------------------------------------------------------
// The integer nearest to x / scale, halves to even, within +-127: what dividing in f64 and rounding gives.  x * (1 / scale)
// is within 2^-15 of the quotient, so only a product that close to a half is decided exactly: x - (h * scale) is one
// rounding, whose sign is right.
__device__ __forceinline__ int32_t quantise(float x, float scale, float inverse) {
    const float t = x * inverse;
    float q = rintf(t);
    if (fabsf(fabsf(t - q) - 0.5f) < 0x1p-12f) {
        const float low = floorf(t), half = low + 0.5f;  // the border between low and low + 1
        const float over = fmaf(-half, scale, x);
        q = over > 0.0f ? low + 1.0f : over < 0.0f ? low : 2.0f * rintf(half * 0.5f);
    }
    return static_cast<int32_t>(fminf(fmaxf(q, -127.0f), 127.0f));
}

// Bound by memory.  A CTA has a row: as many threads as hold it in two 16-byte pieces each (32 to 512; a longer row's rest is
// read a second time), in registers between the maximum and the quotients.  Four pieces and 256 threads are no faster on rows of 4096
// (2048 of them, bf16: 11 us against 10.5) and slower on long ones (256 of 131072: 53 against 32, with all of it in L2; 44 from memory);
// 1024 threads 2048 of 16384: 53 against 34.
constexpr int QUANT_THREADS = 512, QUANT_PIECES = 2;

// A row's scale, from the largest magnitude in it.
struct Scale {
    float scale, lift, lifted, inverse;
    bool zeros;
    __device__ __forceinline__ explicit Scale(float most) {
        scale = __fdiv_rn(most, 127.0f);
        zeros = scale == 0.0f || !(scale < INFINITY);
        lift = scale < 0x1p-100f ? 0x1p100f : 1.0f;  // a power of two: exact, and the reciprocal stays finite
        lifted = scale * lift;
        inverse = 1.0f / lifted;
    }
    __device__ __forceinline__ int32_t quantised(float x) const { return zeros ? 0 : quantise(x * lift, lifted, inverse); }
};

struct QuantArgs {
    const void* x;
    int64_t x_pitch;
    int8_t* q;
    int64_t q_pitch;
    float* scale;
    int32_t cols;
};

template <class T>
__global__ void __launch_bounds__(QUANT_THREADS) k_quantize(const __grid_constant__ QuantArgs g) {
    constexpr int V = VEC<T>;
    __shared__ uint32_t sh[QUANT_THREADS / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, threads = blockDim.x;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(g.x) + row * g.x_pitch;
    int8_t* q = g.q + row * g.q_pitch;
    const Share<T> s(x, g.cols, 0, g.cols + V);
    uint4 raw[QUANT_PIECES];
#pragma unroll
    for (int t = 0; t < QUANT_PIECES; ++t)
        if (tid + t * threads < s.pieces) raw[t] = s.piece(tid + t * threads);
    uint32_t most = 0;  // the bits of |x| order as the magnitudes do, with infinity and then NaN above them
    auto look = [&](const uint4& r) {
        float v[V];
        unpack_16<T>(r, v);
#pragma unroll
        for (int j = 0; j < V; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
    };
    auto edge = [&](auto f) {
        if (s.head + tid < s.first) f(s.head + tid);
        if (s.tail + tid < s.stop) f(s.tail + tid);
    };
#pragma unroll
    for (int t = 0; t < QUANT_PIECES; ++t)
        if (tid + t * threads < s.pieces) look(raw[t]);
    for (int32_t i = tid + QUANT_PIECES * threads; i < s.pieces; i += threads) look(s.piece(i));
    edge([&](int32_t k) { most = max(most, __float_as_uint(to_float(x[k])) & 0x7fffffffu); });
    most = __reduce_max_sync(0xffffffffu, most);
    if ((tid & 31) == 0) sh[tid >> 5] = most;
    __syncthreads();
    for (int w = 0; w < threads / 32; ++w) most = max(most, sh[w]);
    const Scale scale(__uint_as_float(most));
    if (tid == 0) g.scale[row] = scale.scale;
    auto one = [&](float v) { return scale.quantised(v); };
    auto put = [&](int32_t i, const uint4& r) {
        float v[V];
        unpack_16<T>(r, v);
        uint32_t w[V / 4];
        bool near = scale.zeros || scale.lift != 1.0f;
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            uint32_t b[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                // adding 1.5 2^23 rounds to an integer, whose low byte is the sum's; a product next to a half is decided below
                const float y = v[j + t] * scale.inverse, sum = y + 0x1.8p23f;
                near |= fabsf(y - (sum - 0x1.8p23f)) > 0.5f - 0x1p-12f;
                b[t] = __float_as_uint(sum);
            }
            w[j / 4] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        }
        if (near) {
#pragma unroll
            for (int j = 0; j < V; j += 4)
                w[j / 4] = (one(v[j]) & 0xff) | (one(v[j + 1]) & 0xff) << 8 | (one(v[j + 2]) & 0xff) << 16 | static_cast<uint32_t>(one(v[j + 3])) << 24;
        }
        int8_t* to = q + s.first + i * V;
        if (aligned_for<V>(to)) {
            if (V == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[V / 4 - 1]);
            else *reinterpret_cast<uint32_t*>(to) = w[0];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) to[j] = static_cast<int8_t>(w[j / 4] >> (8 * (j % 4)));
        }
    };
#pragma unroll
    for (int t = 0; t < QUANT_PIECES; ++t)
        if (tid + t * threads < s.pieces) put(tid + t * threads, raw[t]);
    for (int32_t i = tid + QUANT_PIECES * threads; i < s.pieces; i += threads) put(i, s.piece(i));
    edge([&](int32_t k) { q[k] = static_cast<int8_t>(one(to_float(x[k]))); });
}

// ---------------------------------------------------------------------------------------------------------
// The product.
// ---------------------------------------------------------------------------------------------------------
constexpr int TILE_N = 128;  // channels of a tile = tensor-memory lanes
constexpr int KB = 128;      // bytes of K per stage: one 128-byte swizzle atom
template <int BM>
constexpr int PROD_THREADS = BM == 16 ? 192 : 320;  // TMA warp, MMA warp, four epilogue warps (eight where there are two or more pieces of 16 tokens)

struct ProductArgs {
    int32_t m, n, k_steps;
    const float* a_scale;
    const float* w_scale;
    const float* bias;
    void* out;
    int64_t out_pitch;
    int* err;
};

template <int BM>
__host__ __device__ constexpr int prod_stages() { return BM == 64 ? 4 : 5; }  // two CTAs an SM: with three or four, calls one behind the other took up to three times as long
template <int BM>
constexpr size_t prod_smem(int split) {
    return 1024 + static_cast<size_t>(prod_stages<BM>()) * (TILE_N + BM) * KB + (split > 1 ? sizeof(int32_t) * TILE_N * BM : 0);
}

// Few tokens of few inputs are quantised by the product's own CTAs (X: their type), each for its part of K: a row's maximum takes
// the whole row, which every CTA reads: 32 KB of f32 in all at most, 16 KB of the 2-byte types.  That saves a launch, and is chosen for
// that: a call with one token, 4096 inputs and channels takes the host 11.7 us instead of 14.3, but the GPU 9.7 instead of 9.0, which
// is what a replayed graph of such calls pays.
constexpr int FEW_VALUES = 8192, FEW_STEPS = 16;  // values of x; steps of K per CTA, whose tokens are held at once
struct FewTokens {
    const void* x;
    int64_t x_pitch;
    int32_t k;
};
template <class X>
__device__ __forceinline__ void quantise_few(const FewTokens& f, int32_t m, int32_t k_first, int32_t k_stop, uint8_t* tokens, float* scales, uint32_t* most, int threads) {
    constexpr int V = VEC<X>, AT_ONCE = FEW_VALUES / V / 192 + 1;
    const int tid = threadIdx.x;
    const int32_t per_row = f.k / V, all = m * per_row;
    auto row_of = [&](int32_t i) { return m == 1 ? 0 : i / per_row; };
    uint4 raw[AT_ONCE];
#pragma unroll
    for (int t = 0; t < AT_ONCE; ++t) {
        const int32_t i = tid + t * threads, row = row_of(i);
        if (i < all) raw[t] = *reinterpret_cast<const uint4*>(static_cast<const X*>(f.x) + row * f.x_pitch + (i - row * per_row) * V);
    }
    for (int32_t i = tid; i < (k_stop - k_first + KB - 1) / KB * 16 * KB / 16; i += threads) reinterpret_cast<uint4*>(tokens)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (tid < 16) most[tid] = 0u;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < AT_ONCE; ++t) {
        const int32_t i = tid + t * threads;
        uint32_t top = 0u;
        if (i < all) {
            float v[V];
            unpack_16<X>(raw[t], v);
#pragma unroll
            for (int j = 0; j < V; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
        }
        if (per_row % 32 == 0) {  // a warp's pieces lie in one row
            top = __reduce_max_sync(0xffffffffu, top);
            if (i < all && (tid & 31) == 0) atomicMax(most + row_of(i), top);
        } else if (i < all) {
            atomicMax(most + row_of(i), top);
        }
    }
    __syncthreads();
    Scale scale(__uint_as_float(most[0]));
    int32_t scaled = 0;  // the row that it is of
#pragma unroll
    for (int t = 0; t < AT_ONCE; ++t) {
        const int32_t i = tid + t * threads, row = row_of(i), k = (i - row * per_row) * V;
        if (i >= all || k < k_first || k >= k_stop) continue;
        if (row != scaled) scale = Scale(__uint_as_float(most[row])), scaled = row;
        float v[V];
        unpack_16<X>(raw[t], v);
        uint32_t w[V / 4];
#pragma unroll
        for (int j = 0; j < V; j += 4)
            w[j / 4] = (scale.quantised(v[j]) & 0xff) | (scale.quantised(v[j + 1]) & 0xff) << 8 | (scale.quantised(v[j + 2]) & 0xff) << 16 | static_cast<uint32_t>(scale.quantised(v[j + 3])) << 24;
        // where TMA would put it: 16-byte chunk c of a 128-byte row r goes to chunk c ^ (r & 7)
        const int32_t at = k - k_first, byte = at % KB;
        uint8_t* to = tokens + at / KB * (16 * KB) + row * KB + (((byte / 16) ^ (row & 7)) * 16 + byte % 16);
        if (V == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[V / 4 - 1]);
        else *reinterpret_cast<uint32_t*>(to) = w[0];
    }
    if (tid < m) scales[tid] = __fdiv_rn(__uint_as_float(most[tid]), 127.0f);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the MMAs read through the asynchronous proxy
}

// A wait that runs out: the roles of a CTA tell each other through a word in its shared memory (and the CTAs of a tile each other),
// which ends their waits and keeps them from writing; the kernel then waits, with the same limit, for the loads and MMAs that it has in
// flight, and raises the context's flag as it ends.  Other launches go on.
__device__ __forceinline__ void tell(dense::SharedWord lost, uint32_t rank, int code) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dense::peer_addr(lost.at, rank)), "r"(code) : "memory");
}
__device__ __forceinline__ void report(int* err, int lost) {
    if (lost) atomicCAS(err, 0, lost);
}

// A CTA computes a tile of TILE_N channels x BM tokens: the channels are the tensor memory's lanes, so a warp's stores run along
// a row of the output, and few tokens still fill the MMA's 128 rows.  The CTAs of a cluster (1, 2, 4 or 8) share a tile:
// each takes a part of K, hands its 32-bit sums over through distributed shared memory, and finishes a part of the tokens.
template <int BM, class T, class X>
__global__ void __launch_bounds__(PROD_THREADS<BM>)
    k_product(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ ProductArgs g, const __grid_constant__ FewTokens few) {
    using namespace dense;
    constexpr int STAGES = prod_stages<BM>();
    constexpr uint32_t W_BYTES = TILE_N * KB, STAGE_BYTES = W_BYTES + BM * KB;
    constexpr uint32_t TMEM_COLS = BM < 32 ? 32 : BM;
    constexpr uint32_t IDESC = make_idesc(2, 1, TILE_N, BM);  // s32 accumulators, signed 8-bit operands
    constexpr bool FEW = !std::is_void<X>::value;
    constexpr uint32_t LOAD_BYTES = FEW ? W_BYTES : STAGE_BYTES;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full;
    __shared__ uint32_t tmem_base_slot;
    __shared__ int lost_word;
    __shared__ uint32_t few_most[FEW ? 16 : 1];
    __shared__ float few_scale[FEW ? 16 : 1];

    const SharedWord lost{smem_u32(&lost_word)};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t split;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(split));
    const uint32_t rank = cluster_rank();
    const int32_t n0 = static_cast<int32_t>(blockIdx.x / split) * TILE_N, m0 = static_cast<int32_t>(blockIdx.y) * BM;
    const int32_t k_begin = static_cast<int32_t>(static_cast<int64_t>(g.k_steps) * rank / split), k_end = static_cast<int32_t>(static_cast<int64_t>(g.k_steps) * (rank + 1) / split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        mbar_init(&acc_full, 1);
        lost_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_base_slot;
    // The sums cross the cluster only after every CTA has started: each warp waits for that when it is done with its part.
    if (split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    auto all_started = [&] {
        __syncwarp();
        if (split > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    };
    // The weights of the first stages do not wait for the tokens to be quantised.
    const int32_t early = min(k_end - k_begin, STAGES);
    int32_t issued = early;  // loads; whether the MMAs' last commit was made: what is to be settled after a wait that ran out
    bool committed = false;
    if (threadIdx.x == 0)
        for (int32_t i = 0; i < early; ++i) {
            mbar_expect_tx(&full_bar[i], LOAD_BYTES);
            tma_load_2d(smem_u32(smem + i * STAGE_BYTES), &map_w, &full_bar[i], (k_begin + i) * KB, n0);
        }
    __syncwarp();
    uint8_t* tokens = smem + STAGES * STAGE_BYTES + (split > 1 ? sizeof(int32_t) * TILE_N * BM : 0);  // FEW: a tile of BM x KB per step
    if constexpr (FEW) quantise_few<X>(few, g.m, k_begin * KB, min(k_end * KB, few.k), tokens, few_scale, few_most, PROD_THREADS<BM>);
    if (FEW) __syncthreads();
    // By plain loads: the kernel that writes the scales may be at work when this one starts.
    auto a_scale = [&](int32_t token) {
        if constexpr (FEW) return few_scale[token];
        else return g.a_scale[token];
    };

    if (warp == 0) {
        if (lane == 0) {
            if (!FEW) {
                asm volatile("griddepcontrol.wait;" ::: "memory");
                for (int32_t i = 0; i < early; ++i) tma_load_2d(smem_u32(smem + i * STAGE_BYTES) + W_BYTES, &map_a, &full_bar[i], (k_begin + i) * KB, m0);
            }
            uint32_t stage = early == STAGES ? 0 : early, phase = early == STAGES ? 1 : 0;
            for (int32_t kt = k_begin + early; kt < k_end; ++kt) {
                if (!mbar_wait(&empty_bar[stage], phase ^ 1u, lost, 1)) break;
                mbar_expect_tx(&full_bar[stage], LOAD_BYTES);
                const uint32_t dst = smem_u32(smem + stage * STAGE_BYTES);
                tma_load_2d(dst, &map_w, &full_bar[stage], kt * KB, n0);
                if (!FEW) tma_load_2d(dst + W_BYTES, &map_a, &full_bar[stage], kt * KB, m0);
                ++issued;
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
        }
        all_started();
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool alive = true;
            for (int32_t kt = k_begin; kt < k_end; ++kt) {
                if (!mbar_wait(&full_bar[stage], phase, lost, 3)) { alive = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t w_addr = smem_u32(smem + stage * STAGE_BYTES);
                const uint64_t dw = make_smem_desc(w_addr), da = make_smem_desc(FEW ? smem_u32(tokens) + (kt - k_begin) * BM * KB : w_addr + W_BYTES);
#pragma unroll
                for (int ks = 0; ks < KB / 32; ++ks)
                    umma<1>(tmem, dw + static_cast<uint64_t>(ks * 2), da + static_cast<uint64_t>(ks * 2), IDESC, kt > k_begin || ks ? 1u : 0u);
                umma_commit(&empty_bar[stage]);
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
            if (alive) umma_commit(&acc_full);
            committed = alive;
        }
        all_started();
    } else {
        const int quarter = warp & 3, ch = quarter * 32 + lane;
        const int32_t col = n0 + ch;
        const float w_scale = col < g.n ? g.w_scale[col] : 0.0f, bias = g.bias && col < g.n ? g.bias[col] : 0.0f;
        T* out = static_cast<T*>(g.out) + col;
        if (!FEW) asm volatile("griddepcontrol.wait;" ::: "memory");  // the tokens' scales
        const bool alive = __all_sync(0xffffffffu, mbar_wait(&acc_full, 0, lost, 4));  // the lanes go on together
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        int32_t* red = reinterpret_cast<int32_t*>(smem + STAGES * STAGE_BYTES);  // [source CTA][token of the share][channel]
        const int32_t share = BM / static_cast<int32_t>(split);
        all_started();
        if (!alive && lane < static_cast<int>(split)) tell(lost, lane, 4);
        for (int c = (warp - 2) >> 2; c < BM / 16; c += (PROD_THREADS<BM> - 64) / 128) {
            uint32_t acc[16];
            tmem_ld16_issue(taddr + c * 16, acc);
            tmem_ld_wait();
            if (split == 1) {
                const int32_t first = m0 + c * 16, left = g.m - first;  // tokens from here on
                if (alive && col < g.n) {
                    float scales[16];  // loaded before the stores, which hold later loads back
#pragma unroll
                    for (int j = 0; j < 16; ++j) scales[j] = j < left ? a_scale(first + j) : 0.0f;
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (j < left) {
                            const float y = __int2float_rn(static_cast<int32_t>(acc[j])) * scales[j] * w_scale;
                            out[(first + j) * g.out_pitch] = from_float<T>(g.bias ? y + bias : y);
                        }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const uint32_t t = c * 16 + j, owner = t / share;
                    const uint32_t at = smem_u32(red + (rank * share + (t - owner * share)) * TILE_N + ch);
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_addr(at, owner)), "r"(acc[j]) : "memory");
                }
            }
        }
    }
    if (split > 1) {
        cluster_sync_all();  // every CTA's sums have arrived
        if (warp >= 2 && !lost.raised()) {
            const int quarter = warp & 3, ch = quarter * 32 + lane;
            const int32_t col = n0 + ch, share = BM / static_cast<int32_t>(split), first = m0 + static_cast<int32_t>(rank) * share;
            const int32_t* red = reinterpret_cast<const int32_t*>(smem + STAGES * STAGE_BYTES);
            const float w_scale = col < g.n ? g.w_scale[col] : 0.0f, bias = g.bias && col < g.n ? g.bias[col] : 0.0f;
            const float held = lane < share && first + lane < g.m ? a_scale(first + lane) : 0.0f;  // a lane for each token: at most 32
            T* out = static_cast<T*>(g.out) + col;
            for (int32_t t = (warp - 2) >> 2; t < share && first + t < g.m; t += (PROD_THREADS<BM> - 64) / 128) {
                int32_t acc = 0;
                for (uint32_t src = 0; src < split; ++src) acc += red[(src * share + t) * TILE_N + ch];
                const float y = __int2float_rn(acc) * __shfl_sync(0xffffffffu, held, t) * w_scale;
                if (col < g.n) out[(first + t) * g.out_pitch] = from_float<T>(g.bias ? y + bias : y);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (lost.raised()) {
        if (threadIdx.x == 0) settle_loads(full_bar, STAGES, issued);
        if (threadIdx.x == 32) {
            if (!committed) umma_commit(&acc_full);
            mbar_settle(&acc_full, 0);
        }
        if (threadIdx.x == 0) report(g.err, lost.value());
        __syncwarp();
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// Many tokens: CTA pairs.  Two CTAs of a cluster share a tile of 256 channels x BM tokens through tcgen05 cta_group::2: each stages its
// own 128 channels and half of the tokens, so the operands, whose way from L2 to the SMs binds 8-bit products, cross it once
// per pair.  Persistent over tiles, two accumulators in tensor memory, so that one tile's epilogue runs under the next one's
// MMAs.  Roles per CTA: TMA warp, MMA warp (the leader's issues for both), eight epilogue warps, two for each quarter of the
// lanes.  Every TMA load counts on the leader's barrier; the leader's commits free the stages and hand the accumulators over in
// both CTAs; epilogue warps of both release an accumulator on the leader's barrier.  All waits are bounded.
constexpr int PAIR_THREADS = 64 + 32 * 8;
constexpr int PAIR_CHANNELS = 256;
template <int BM>
__host__ __device__ constexpr int pair_stages() { return 192 * 1024 / ((TILE_N + BM / 2) * KB); }
template <int BM>
constexpr size_t pair_smem() { return 1024 + static_cast<size_t>(pair_stages<BM>()) * (TILE_N + BM / 2) * KB; }

struct PairArgs {
    ProductArgs p;
    int32_t tiles_m, tiles, group;  // token tiles, all tiles, channel tiles that a wave of pairs walks together
};
// Tile number t: `group` channel tiles by all token tiles, channels innermost, so that the pairs at work at once share operands in L2.
__device__ __forceinline__ void tile_place(const PairArgs& g, int32_t tiles_n, int32_t t, int32_t& tm, int32_t& tn) {
    const int32_t per_band = g.group * g.tiles_m, band = t / per_band, width = min(g.group, tiles_n - band * g.group), in_band = t - band * per_band;
    tm = in_band / width;
    tn = band * g.group + in_band - tm * width;
}

template <int BM, class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
    k_product_pair(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ PairArgs args) {
    using namespace dense;
    constexpr int STAGES = pair_stages<BM>();
    constexpr uint32_t W_BYTES = TILE_N * KB, STAGE_BYTES = W_BYTES + BM / 2 * KB;
    constexpr uint32_t TMEM_COLS = 2 * BM;
    constexpr uint32_t IDESC = make_idesc(2, 1, PAIR_CHANNELS, BM);
    const ProductArgs& g = args.p;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t full_bar[STAGES], empty_bar[STAGES], acc_full[2], acc_empty[2], settle_bar;
    __shared__ uint32_t tmem_base_slot;
    __shared__ int lost_word, peer_issued;
    // Of a warp's half of the tile's tokens: four of them come by one instruction, where each by a load of its own held the epilogue up
    // behind short sums (8192 x 784 -> 4096: 67 -> 49 us; 58 by read-only loads, which memory that k_quantize may be writing rules out).
    __shared__ __align__(16) float token_scales[8][BM / 2];

    const SharedWord lost{smem_u32(&lost_word)};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const int32_t first_tile = blockIdx.x >> 1, tile_step = gridDim.x >> 1, tiles_n = args.tiles / args.tiles_m;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        lost_word = 0;
        mbar_init(&settle_bar, 1);
        for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_base_slot;
    int32_t issued = 0;  // loads of this CTA

    if (warp == 0) {
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool alive = true;
            for (int32_t tile = first_tile; tile < args.tiles && alive; tile += tile_step) {
                int32_t tm, tn;
                tile_place(args, tiles_n, tile, tm, tn);
                const int32_t n0 = tn * PAIR_CHANNELS + static_cast<int32_t>(rank) * TILE_N, m0 = tm * BM + static_cast<int32_t>(rank) * (BM / 2);
                int32_t early = 0;
                if (tile == first_tile) {  // the weights of the first stages do not wait for the kernel that quantises the tokens
                    early = min(g.k_steps, STAGES);
                    for (int32_t i = 0; i < early; ++i) {
                        if (leader) mbar_expect_tx(&full_bar[i], 2 * STAGE_BYTES);
                        tma_load_2d_pair(smem_u32(smem + i * STAGE_BYTES), &map_w, peer_addr(smem_u32(&full_bar[i]), 0), i * KB, n0);
                    }
                    asm volatile("griddepcontrol.wait;" ::: "memory");
                    for (int32_t i = 0; i < early; ++i)
                        tma_load_2d_pair(smem_u32(smem + i * STAGE_BYTES) + W_BYTES, &map_a, peer_addr(smem_u32(&full_bar[i]), 0), i * KB, m0);
                    issued = early;
                    stage = early == STAGES ? 0 : early;
                    phase = early == STAGES ? 1 : 0;
                }
                for (int32_t kt = early; kt < g.k_steps; ++kt) {
                    if (!mbar_wait(&empty_bar[stage], phase ^ 1u, lost, 1)) { alive = false; break; }
                    if (leader) mbar_expect_tx(&full_bar[stage], 2 * STAGE_BYTES);
                    const uint32_t bar = peer_addr(smem_u32(&full_bar[stage]), 0);
                    const uint32_t dst = smem_u32(smem + stage * STAGE_BYTES);
                    tma_load_2d_pair(dst, &map_w, bar, kt * KB, n0);
                    tma_load_2d_pair(dst + W_BYTES, &map_a, bar, kt * KB, m0);
                    ++issued;
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            uint32_t stage = 0, phase = 0, it = 0;
            bool alive = true;
            for (int32_t tile = first_tile; tile < args.tiles && alive; tile += tile_step, ++it) {
                const uint32_t buf = it & 1u;
                if (!mbar_wait(&acc_empty[buf], ((it >> 1) & 1u) ^ 1u, lost, 2)) { alive = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t tmem_d = tmem + buf * BM;
                for (int32_t kt = 0; kt < g.k_steps; ++kt) {
                    if (!mbar_wait(&full_bar[stage], phase, lost, 3)) { alive = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t w_addr = smem_u32(smem + stage * STAGE_BYTES);
                    const uint64_t dw = make_smem_desc(w_addr), da = make_smem_desc(w_addr + W_BYTES);
#pragma unroll
                    for (int ks = 0; ks < KB / 32; ++ks)
                        umma_pair<1>(tmem_d, dw + static_cast<uint64_t>(ks * 2), da + static_cast<uint64_t>(ks * 2), IDESC, (kt | ks) ? 1u : 0u);
                    const uint32_t e = smem_u32(&empty_bar[stage]);
                    umma_commit_pair(e);
                    umma_commit_pair(peer_addr(e, 1));
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
                if (alive) {
                    const uint32_t f = smem_u32(&acc_full[buf]);
                    umma_commit_pair(f);
                    umma_commit_pair(peer_addr(f, 1));
                }
            }
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2, ch = quarter * 32 + lane;
        uint32_t it = 0;
        float* mine = token_scales[warp - 2];
        asm volatile("griddepcontrol.wait;" ::: "memory");  // the tokens' scales
        for (int32_t tile = first_tile; tile < args.tiles; tile += tile_step, ++it) {
            int32_t tm, tn;
            tile_place(args, tiles_n, tile, tm, tn);
            const uint32_t buf = it & 1u;
            const int32_t col = tn * PAIR_CHANNELS + static_cast<int32_t>(rank) * TILE_N + ch, m0 = tm * BM + half * (BM / 2);
            const float w_scale = col < g.n ? g.w_scale[col] : 0.0f, bias = g.bias && col < g.n ? g.bias[col] : 0.0f;
            __syncwarp();  // the last tile's have been read
#pragma unroll
            for (int t = 0; t < BM / 64; ++t) mine[32 * t + lane] = m0 + 32 * t + lane < g.m ? g.a_scale[m0 + 32 * t + lane] : 0.0f;
            __syncwarp();
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (it >> 1) & 1u, lost, 4))) break;  // the lanes go on together
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t taddr = tmem + buf * BM + half * (BM / 2) + (static_cast<uint32_t>(quarter * 32) << 16);
            T* out = static_cast<T*>(g.out) + static_cast<int64_t>(m0) * g.out_pitch + col;
#pragma unroll 1
            for (int c = 0; c < BM / 32; ++c) {
                const int32_t left = g.m - (m0 + c * 16);  // tokens from here on
                uint32_t acc[16];
                tmem_ld16_issue(taddr + c * 16, acc);
                float scales[16];
#pragma unroll
                for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(scales + j) = *reinterpret_cast<const float4*>(mine + c * 16 + j);
                tmem_ld_wait();
                if (col < g.n) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (j < left) {
                            const float y = __int2float_rn(static_cast<int32_t>(acc[j])) * scales[j] * w_scale;
                            out[(c * 16 + j) * g.out_pitch] = from_float<T>(g.bias ? y + bias : y);
                        }
                }
                __syncwarp();
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(peer_addr(smem_u32(&acc_empty[buf]), 0));
        }
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (lane == 0 && lost.raised()) tell(lost, rank ^ 1, lost.value());
    cluster_sync_all();  // no CTA leaves (or frees tensor memory) while its peer can still reach it
    if (lost.raised()) {  // in both CTAs or in none
        if (threadIdx.x == 0 && !leader)
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_addr(smem_u32(&peer_issued), 0)), "r"(issued) : "memory");
        __syncwarp();
        cluster_sync_all();
        if (threadIdx.x == 0 && leader) {  // the barriers of both CTAs' loads are here; of some loads only one has issued its half
            for (int32_t i = peer_issued; i < issued; ++i) mbar_complete_tx(&full_bar[i % STAGES], STAGE_BYTES);
            for (int32_t i = issued; i < peer_issued; ++i) mbar_expect_tx(&full_bar[i % STAGES], STAGE_BYTES);
            settle_loads(full_bar, STAGES, max(issued, peer_issued));
            report(g.err, lost.value());
        }
        if (threadIdx.x == 32 && leader) {
            umma_commit_pair(smem_u32(&settle_bar));
            mbar_settle(&settle_bar, 0);
        }
        __syncwarp();
        cluster_sync_all();
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// Failure-detection self test: a warp waits as the products do, on a barrier that nothing arrives on, and reports as they do.
__global__ void k_lose_wait(int* err) {
    __shared__ uint64_t bar;
    __shared__ int lost_word;
    if (threadIdx.x != 0) return;
    const dense::SharedWord lost{dense::smem_u32(&lost_word)};
    lost_word = 0;
    dense::mbar_init(&bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    dense::mbar_wait(&bar, 0, lost, 7);
    report(err, lost.value());
}

struct Product {
    int64_t m, n, k;
    const int8_t* a;
    int64_t a_pitch;
    const float* a_scale;
    const int8_t* w;
    int64_t w_pitch;
    const float* w_scale;
    const float* bias;
    void* out;
    int32_t out_type;
    int64_t out_pitch;
    bool after_quantising;  // the launch before is k_quantize, which lets this one start early
};

int32_t check_matrix8(const char* what, const void* p, int64_t k, int64_t pitch) {
    if (!p) return fail(THRML_ERR_INVALID_ARG, std::string(what) + ": null pointer");
    if (!aligned_to(p, 16) || pitch % 16) return fail(THRML_ERR_INVALID_ARG, std::string(what) + ": 8-bit rows start on 16-byte boundaries and have a pitch that is a multiple of 16");
    if (pitch < k) return fail(THRML_ERR_INVALID_ARG, std::string(what) + ": the pitch is smaller than a row");
    return THRML_OK;
}

int32_t check_product(const Product& p) {
    if (p.m < 0 || p.m > (1 << 22) || p.n < 0 || p.n > (1 << 24)) return fail(THRML_ERR_INVALID_ARG, "at most 2^22 tokens and 2^24 channels");
    if (p.k < 1 || p.k > 131071) return fail(THRML_ERR_INVALID_ARG, "k is not within 1 and 131071, where sums of 8-bit products fit 32 bits");
    if (!is_float_type(p.out_type)) return fail(THRML_ERR_INVALID_ARG, "out: the element type is not a float type");
    if (p.m == 0 || p.n == 0) return THRML_OK;
    if (p.out_pitch < p.n) return fail(THRML_ERR_INVALID_ARG, "out: the pitch is smaller than a row");
    if (!p.out || !aligned_to(p.out, type_size(p.out_type))) return fail(THRML_ERR_INVALID_ARG, "out: the pointer is null or not aligned to the element");
    if (!p.a_scale || !p.w_scale) return fail(THRML_ERR_INVALID_ARG, "scales: null pointer");
    if (int32_t rc = check_matrix8("a", p.a, p.k, p.a_pitch)) return rc;
    return check_matrix8("w", p.w, p.k, p.w_pitch);
}

int32_t check_apart(const Product& p) {
    const Area out(p.out, type_size(p.out_type), p.m, p.n, p.out_pitch);
    if (overlap(out, Area(p.a, 1, p.m, p.k, p.a_pitch)) || overlap(out, Area(p.w, 1, p.n, p.k, p.w_pitch)) || overlap(out, Area(p.a_scale, 4, 1, p.m, p.m)) ||
        overlap(out, Area(p.w_scale, 4, 1, p.n, p.n)) || overlap(out, Area(p.bias, 4, 1, p.n, p.n)))
        return fail(THRML_ERR_INVALID_ARG, "out overlaps an input");
    return THRML_OK;
}

template <int BM, class T, class X>
int32_t launch_product(thrml_ctx* ctx, cudaStream_t stream, const Product& p, int split, const FewTokens& few) {
    CUtensorMap map_w, map_a;
    if (int32_t rc = make_operand_map(&map_w, const_cast<int8_t*>(p.w), true, p.k, p.n, p.w_pitch, TILE_N)) return rc;
    if (std::is_void<X>::value) {
        if (int32_t rc = make_operand_map(&map_a, const_cast<int8_t*>(p.a), true, p.k, p.m, p.a_pitch, BM)) return rc;
    } else {
        map_a = map_w;  // not used
    }
    constexpr size_t token_bytes = std::is_void<X>::value ? 0 : FEW_STEPS * BM * KB;
    ProductArgs g{static_cast<int32_t>(p.m), static_cast<int32_t>(p.n), static_cast<int32_t>((p.k + KB - 1) / KB), p.a_scale, p.w_scale, p.bias, p.out, p.out_pitch, ctx->wait_flag_dev};
    if (int32_t rc = allow_shared<k_product<BM, T, X>>(ctx, prod_smem<BM>(2) + token_bytes)) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((p.n + TILE_N - 1) / TILE_N * split), static_cast<unsigned>((p.m + BM - 1) / BM));
    cfg.blockDim = dim3(PROD_THREADS<BM>);
    cfg.dynamicSmemBytes = prod_smem<BM>(split) + token_bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {static_cast<unsigned>(split), 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.after_quantising ? 2 : 1;
    CU_TRY(cudaLaunchKernelEx(&cfg, k_product<BM, T, X>, map_w, map_a, g, few));
    return THRML_OK;
}

template <int BM, class T>
int32_t launch_pair(thrml_ctx* ctx, cudaStream_t stream, const Product& p) {
    CUtensorMap map_w, map_a;
    if (int32_t rc = make_operand_map(&map_w, const_cast<int8_t*>(p.w), true, p.k, p.n, p.w_pitch, TILE_N)) return rc;
    if (int32_t rc = make_operand_map(&map_a, const_cast<int8_t*>(p.a), true, p.k, p.m, p.a_pitch, BM / 2)) return rc;
    const int32_t tiles_m = static_cast<int32_t>((p.m + BM - 1) / BM), tiles_n = static_cast<int32_t>((p.n + PAIR_CHANNELS - 1) / PAIR_CHANNELS);
    const PairArgs g{{static_cast<int32_t>(p.m), static_cast<int32_t>(p.n), static_cast<int32_t>((p.k + KB - 1) / KB), p.a_scale, p.w_scale, p.bias, p.out, p.out_pitch, ctx->wait_flag_dev},
                     tiles_m, tiles_m * tiles_n, 8};
    if (int32_t rc = allow_shared<k_product_pair<BM, T>>(ctx, static_cast<int>(pair_smem<BM>()))) return rc;
    const int pairs = std::min(ctx->sm_count / 2, tiles_m * tiles_n);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
    cfg.blockDim = dim3(PAIR_THREADS);
    cfg.dynamicSmemBytes = pair_smem<BM>();
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = p.after_quantising ? 1 : 0;
    CU_TRY(cudaLaunchKernelEx(&cfg, k_product_pair<BM, T>, map_w, map_a, g));
    return THRML_OK;
}

// K is split while that takes no more than the SMs.
int split_of(const thrml_ctx* ctx, int64_t tiles, int64_t k_steps) {
    int split = 1;
    while (split < 8 && 2 * tiles * split <= ctx->sm_count && 2 * split <= k_steps) split *= 2;
    return split;
}

template <class T>
int32_t product(thrml_ctx* ctx, cudaStream_t stream, const Product& p) {
    // Up to 64 tokens, and up to a wave of two CTAs an SM, the operands' way from memory binds, and many CTAs keep more of them
    // in flight (4096 inputs, 65536 channels: 16 tokens 47 us, in pairs 58; 64 tokens 51, in pairs 61; 4096 channels: 128 tokens
    // 15, in pairs 20; 512 tokens 19, in pairs 22).  Beyond, pairs: with 256 tokens a tile unless 128 need fewer rounds for the
    // half of the work each.
    const int bm = p.m <= 16 ? 16 : p.m <= 32 ? 32 : 64;
    const int64_t tiles = (p.n + TILE_N - 1) / TILE_N * ((p.m + bm - 1) / bm), k_steps = (p.k + KB - 1) / KB;
    if (p.m > 64 && tiles > 2 * ctx->sm_count) {
        const auto rounds = [&](int64_t width) { return ((p.n + PAIR_CHANNELS - 1) / PAIR_CHANNELS * ((p.m + width - 1) / width) + ctx->sm_count / 2 - 1) / (ctx->sm_count / 2); };
        return 2 * rounds(256) <= rounds(128) ? launch_pair<256, T>(ctx, stream, p) : launch_pair<128, T>(ctx, stream, p);
    }
    const int split = split_of(ctx, tiles, k_steps);
    if (bm == 16) return launch_product<16, T, void>(ctx, stream, p, split, {});
    if (bm == 32) return launch_product<32, T, void>(ctx, stream, p, split, {});
    return launch_product<64, T, void>(ctx, stream, p, split, {});
}

int32_t run_product(thrml_ctx* ctx, void* stream, const Product& p) {
    if (p.m == 0 || p.n == 0) return THRML_OK;
    return for_type(p.out_type, [&](auto e) { return product<decltype(e)>(ctx, static_cast<cudaStream_t>(stream), p); });
}

struct Quant {
    int64_t rows, cols;
    const void* x;
    int32_t x_type;
    int64_t x_pitch;
    int8_t* q;
    int64_t q_pitch;
    float* scale;
};

int32_t check_quant(const Quant& z) {
    if (z.rows < 0 || z.rows > INT32_MAX || z.cols < 1 || z.cols > (1 << 30)) return fail(THRML_ERR_INVALID_ARG, "x: the number of rows or columns is out of range");
    if (!is_float_type(z.x_type)) return fail(THRML_ERR_INVALID_ARG, "x: the element type is not a float type");
    if (z.x_pitch < z.cols || z.q_pitch < z.cols) return fail(THRML_ERR_INVALID_ARG, "x, q: the pitch is smaller than a row");
    if (z.rows && (!z.x || !z.q || !z.scale)) return fail(THRML_ERR_INVALID_ARG, "x, q, scale: null pointer");
    if (!aligned_to(z.x, type_size(z.x_type))) return fail(THRML_ERR_INVALID_ARG, "x: the pointer is not aligned to the element");
    return THRML_OK;
}

int32_t run_quant(void* stream, const Quant& z) {
    if (z.rows == 0) return THRML_OK;
    const QuantArgs g{z.x, z.x_pitch, z.q, z.q_pitch, z.scale, static_cast<int32_t>(z.cols)};
    return for_type(z.x_type, [&](auto e) {
        int threads = 32;
        while (threads < QUANT_THREADS && static_cast<int64_t>(threads) * QUANT_PIECES * VEC<decltype(e)> < z.cols) threads *= 2;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned>(z.rows));
        cfg.blockDim = dim3(static_cast<unsigned>(threads));
        cfg.stream = static_cast<cudaStream_t>(stream);
        CU_TRY(cudaLaunchKernelEx(&cfg, k_quantize<decltype(e)>, g));
        return THRML_OK;
    });
}

// The whole of thrml_linear_i8 in one launch, where x is small enough (and its rows made of whole 16-byte pieces).
int32_t run_few(thrml_ctx* ctx, void* stream, const Product& p, const Quant& z, bool& done) {
    const int64_t vec = 16 / static_cast<int64_t>(type_size(z.x_type)), tiles = (p.n + TILE_N - 1) / TILE_N, k_steps = (p.k + KB - 1) / KB;
    const int split = split_of(ctx, tiles, k_steps);
    done = p.m <= 16 && p.m * p.k <= FEW_VALUES && (k_steps + split - 1) / split <= FEW_STEPS && p.k % vec == 0 && z.x_pitch % vec == 0 && aligned_to(z.x, 16) && tiles <= ctx->sm_count;
    if (!done) return THRML_OK;
    const FewTokens few{z.x, z.x_pitch, static_cast<int32_t>(p.k)};
    return for_type(p.out_type, [&](auto e) {
        return for_type(z.x_type, [&](auto x) { return launch_product<16, decltype(e), decltype(x)>(ctx, static_cast<cudaStream_t>(stream), p, split, few); });
    });
}

}  // namespace

extern "C" {

int32_t thrml_quantize_rows_i8(thrml_ctx* ctx, void* stream, int64_t rows, int64_t cols, const void* x, int32_t x_type, int64_t x_pitch, int8_t* q, int64_t q_pitch,
                               float* scale) {
    return guarded(ctx, [&]() -> int32_t {
        const Quant z{rows, cols, x, x_type, x_pitch, q, q_pitch, scale};
        if (int32_t rc = check_quant(z)) return rc;
        return run_quant(stream, z);
    });
}

int32_t thrml_matmul_i8(thrml_ctx* ctx, void* stream, int64_t m, int64_t n, int64_t k, const int8_t* a, int64_t a_pitch, const float* a_scale, const int8_t* w,
                        int64_t w_pitch, const float* w_scale, const float* bias, void* out, int32_t out_type, int64_t out_pitch) {
    return guarded(ctx, [&]() -> int32_t {
        const Product p{m, n, k, a, a_pitch, a_scale, w, w_pitch, w_scale, bias, out, out_type, out_pitch, false};
        if (int32_t rc = check_product(p)) return rc;
        if (int32_t rc = check_apart(p)) return rc;
        return run_product(ctx, stream, p);
    });
}

int32_t thrml_linear_i8(thrml_ctx* ctx, void* stream, int64_t m, int64_t n, int64_t k, const void* x, int32_t x_type, int64_t x_pitch, int8_t* q, int64_t q_pitch,
                        float* scale, const int8_t* w, int64_t w_pitch, const float* w_scale, const float* bias, void* out, int32_t out_type, int64_t out_pitch) {
    return guarded(ctx, [&]() -> int32_t {
        const Product p{m, n, k, q, q_pitch, scale, w, w_pitch, w_scale, bias, out, out_type, out_pitch, true};
        if (int32_t rc = check_product(p)) return rc;
        const Quant z{m, k, x, x_type, x_pitch, q, q_pitch, scale};
        if (int32_t rc = check_quant(z)) return rc;
        if (int32_t rc = check_apart(p)) return rc;
        if (m == 0 || n == 0) return THRML_OK;
        // CTAs that quantise the tokens themselves read x while others write
        if (overlap(Area(out, type_size(out_type), m, n, out_pitch), Area(x, type_size(x_type), m, k, x_pitch))) return fail(THRML_ERR_INVALID_ARG, "out overlaps x");
        bool done = false;
        Product alone = p;
        alone.after_quantising = false;
        if (int32_t rc = run_few(ctx, stream, alone, z, done)) return rc;
        if (done) return THRML_OK;
        if (int32_t rc = run_quant(stream, z)) return rc;
        return run_product(ctx, stream, p);
    });
}

int32_t thrml_debug_lose_wait(thrml_ctx* ctx, void* stream) {
    return guarded(ctx, [&]() -> int32_t {
        k_lose_wait<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>(ctx->wait_flag_dev);
        CU_TRY(cudaGetLastError());
        return THRML_OK;
    });
}

}  // extern "C"
