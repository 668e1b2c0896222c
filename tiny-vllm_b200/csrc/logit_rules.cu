// Rules on logits, before a token is drawn from them: for token v of a row whose request holds slot s,
//
//   x = logit(v)
//   x = x > 0 ? x / repetition : x * repetition                       if v is among the request's tokens (prompt or answer)
//   x = x - frequency * count(v) - presence * (count(v) > 0)          count: occurrences in the answer alone
//   x = x + (sum of the request's biases of v)
//   x = -inf                                                          if the request's mask has a zero bit at v
//
// in float32, rounded once to the type of the logits.  Biases come behind the penalties, so that one adds what it says whether its token
// was seen or not (before them, a penalty for repetition would divide or multiply it too).  The counts are made anew from the request's tokens in every call:
// a CTA takes one slice of one row, counts the tokens that fall into it in shared memory (a word a token: the count, one
// bit for "in the prompt", one for "has a bias"), and then passes over its slice once.  Integer atomics and one thread a
// logit: the result does not depend on the order in which anything runs.
//
// Bound by reading and writing the logits; the loads of the slice are issued first, so that the chain slot -> lengths ->
// tokens -> counts runs under them.  64 rows x 151,936 float32 with 4,001 tokens and 300 biases each take 23 us, 3.4 TB/s (a copy of the
// logits alone 13.5: every CTA goes over its row's tokens), 24 rows with 900 tokens and masks 8.4 us, 3.5 TB/s; one row 3.0 us, which is
// the chain.
#include "common.cuh"

namespace {

constexpr int THREADS = 256;
// Tokens of the vocabulary a CTA takes.  Every CTA of a row goes over all of its history, so slices are large once their CTAs fill the GPU
// (64 rows x 151,936 with 4,001 tokens: 4096 a CTA 23 us, 2048 30; 24 rows with 900: 8.4, 9.3) and small before (one row 3.6 us, 3.0; 7
// rows x 32,003: 4.8, 3.9).
constexpr int LARGE_SLICE = 4096, SMALL_SLICE = 2048;
constexpr int MAX_BIASES = 1024;                   // biases of a slot
constexpr int BIASES_EACH = MAX_BIASES / THREADS;  // ... and of a thread
constexpr uint32_t HAS_BIAS = 1u << 31, IN_PROMPT = 1u << 30, COUNT = IN_PROMPT - 1;

struct Rules {
    const int* slots;                              // [rows]; one outside [0, slot_count): no rules
    const float* penalties;                        // [slot_count, 3] repetition, presence, frequency
    const int* lengths;                            // [slot_count, 2] tokens, of them the prompt's
    const int* history;                            // [slot_count, room]
    const int* bias_tokens;                        // [slot_count, biases] or null; -1: none
    const float* bias_values;
    const uint32_t* masks;                         // [mask_count, mask_words] or null
    const int* mask_rows;                          // [slot_count]; one outside [0, mask_count): every token is allowed
    int slot_count, room, biases, mask_count, mask_words;
};

template <typename T, int VEC> __device__ __forceinline__ void load_vec(const T* p, float* v) {
    if constexpr (VEC == 1) {
        v[0] = to_float<T>(*p);
    } else if constexpr (sizeof(T) == 4) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
        unpack_bf16x8(*reinterpret_cast<const uint4*>(p), v);
    }
}
template <typename T, int VEC> __device__ __forceinline__ void store_vec(T* p, const float* v) {
    if constexpr (VEC == 1) *p = from_float<T>(v[0]);
    else if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint4*>(p) = pack_bf16x8(v);
}

// logits may be out itself (every thread reads what it will write before it writes): plain pointers
template <typename T, int VEC, int SLICE>
__global__ void __launch_bounds__(THREADS, VEC == 1 ? 4 : 5)
logit_rules_kernel(const T* logits, int64_t row_stride, T* out, int64_t out_stride, int vocab, int slices, Rules rules) {
    __shared__ __align__(16) uint32_t words[SLICE];
    __shared__ int any_twice;
    extern __shared__ float bias[];                // [SLICE] where there are biases
    constexpr int PASSES = SLICE / (THREADS * VEC);
    const int tid = threadIdx.x;
    const int row = blockIdx.x / slices, begin = (blockIdx.x % slices) * SLICE;
    const int count = min(SLICE, vocab - begin);
    const T* x = logits + (int64_t)row * row_stride + begin;
    T* y = out + (int64_t)row * out_stride + begin;

    float v[PASSES][VEC];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int at = (p * THREADS + tid) * VEC;
        if (at + VEC <= count) load_vec<T, VEC>(x + at, v[p]);
        else
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[p][e] = at + e < count ? to_float<T>(x[at + e]) : 0.0f;
    }
    const int slot = rules.slots[row];
    for (int i = 4 * tid; i < SLICE; i += 4 * THREADS) *reinterpret_cast<uint4*>(words + i) = make_uint4(0, 0, 0, 0);
    if (tid == 0) any_twice = 0;
    __syncthreads();
    const bool ruled = (unsigned)slot < (unsigned)rules.slot_count;       // the same for the whole CTA
    float repetition = 1.0f, presence = 0.0f, frequency = 0.0f;
    const uint32_t* mask = nullptr;
    uint32_t allowed[PASSES];                      // the mask's words of this thread's tokens
    bool counted = false;
    const bool biased = ruled && rules.biases > 0;
    if (ruled) {
        // (everything that the slot leads to, side by side)
        int bias_token[BIASES_EACH];
        const int* tokens = rules.bias_tokens + (int64_t)slot * rules.biases;
        const float* values = rules.bias_values + (int64_t)slot * rules.biases;
#pragma unroll
        for (int n = 0; n < BIASES_EACH; ++n)
            bias_token[n] = tid + n * THREADS < rules.biases ? __ldcg(tokens + tid + n * THREADS) : -1;
        repetition = rules.penalties[3 * (int64_t)slot];
        presence = rules.penalties[3 * (int64_t)slot + 1];
        frequency = rules.penalties[3 * (int64_t)slot + 2];
        const int total = min(max(rules.lengths[2 * (int64_t)slot], 0), rules.room);
        const int prompt = min(max(rules.lengths[2 * (int64_t)slot + 1], 0), total);
        if (rules.masks) {
            const int m = rules.mask_rows[slot];
            if ((unsigned)m < (unsigned)rules.mask_count) {
                mask = rules.masks + (int64_t)m * rules.mask_words;
#pragma unroll
                for (int p = 0; p < PASSES; ++p) {
                    const int at = (p * THREADS + tid) * VEC;
                    if (at < count) allowed[p] = __ldg(mask + ((begin + at) >> 5));
                }
            }
        }
        // without a penalty for repetition the prompt is not looked at
        const int first = repetition == 1.0f ? (presence == 0.0f && frequency == 0.0f ? total : prompt) : 0;
        counted = first < total;
        const int* history = rules.history + (int64_t)slot * rules.room;
        // (in batches, so that the loads of one do not wait for the counts of the one before)
        constexpr int BATCH = 8;
        for (int i0 = first + tid; i0 < total; i0 += BATCH * THREADS) {
            int token[BATCH];
#pragma unroll
            for (int n = 0; n < BATCH; ++n) token[n] = i0 + n * THREADS < total ? __ldcg(history + i0 + n * THREADS) : -1;
#pragma unroll
            for (int n = 0; n < BATCH; ++n) {
                const unsigned at = (unsigned)token[n] - (unsigned)begin;
                if (token[n] >= 0 && at < (unsigned)count) {
                    if (i0 + n * THREADS >= prompt) atomicAdd(words + at, 1u);
                    else atomicOr(words + at, IN_PROMPT);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < BIASES_EACH; ++n) {
            const unsigned at = (unsigned)bias_token[n] - (unsigned)begin;
            if (bias_token[n] >= 0 && at < (unsigned)count) {
                if (atomicOr(words + at, HAS_BIAS) & HAS_BIAS) any_twice = 1;
                else bias[at] = __ldcg(values + tid + n * THREADS);
            }
        }
        if (counted || biased) __syncthreads();
        if (biased && any_twice) {
            // a token named more than once: its first entry adds them all up, in their order
#pragma unroll
            for (int n = 0; n < BIASES_EACH; ++n) {
                const int i = tid + n * THREADS, token = bias_token[n];
                const unsigned at = (unsigned)token - (unsigned)begin;
                if (token < 0 || at >= (unsigned)count) continue;
                bool first_entry = true;
                float sum = 0.0f;
                for (int j = 0; j < rules.biases && first_entry; ++j)
                    if (tokens[j] == token) {
                        if (j < i) first_entry = false;
                        else sum = __fadd_rn(sum, values[j]);
                    }
                if (first_entry) bias[at] = sum;
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int at = (p * THREADS + tid) * VEC;
        if (at >= count) break;
        if (counted || biased) {
            uint32_t word[VEC];
            if constexpr (VEC == 1) word[0] = words[at];
            else
#pragma unroll
                for (int e = 0; e < VEC; e += 4) *reinterpret_cast<uint4*>(word + e) = *reinterpret_cast<const uint4*>(words + at + e);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (word[e] == 0) continue;
                float f = v[p][e];
                if (word[e] & ~HAS_BIAS) {
                    f = f > 0.0f ? __fdiv_rn(f, repetition) : __fmul_rn(f, repetition);
                    const uint32_t times = word[e] & COUNT;
                    if (times) f = __fsub_rn(__fsub_rn(f, __fmul_rn(frequency, (float)times)), presence);
                }
                if (word[e] & HAS_BIAS) f = __fadd_rn(f, bias[at + e]);
                v[p][e] = f;
            }
        }
        if (mask) {
            const uint32_t bits = allowed[p] >> (at & 31);                      // (a slice starts at a whole word, VEC divides 32)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (!(bits >> e & 1u)) v[p][e] = -INFINITY;
        }
        if (at + VEC <= count) store_vec<T, VEC>(y + at, v[p]);
        else
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (at + e < count) y[at + e] = from_float<T>(v[p][e]);
    }
}

// lengths[slot] grows by one for every row that holds the slot, and the rows' tokens join its history, in the order of the
// rows.  A full history stays as it is.  One CTA: a row counts those before it that hold its slot.
__global__ void append_tokens_kernel(const int* slots, const int* tokens, int rows, int* lengths, int* history, int slot_count,
                                     int room) {
    extern __shared__ int held[];
    for (int i = threadIdx.x; i < rows; i += blockDim.x) held[i] = slots[i];
    __syncthreads();
    for (int i = threadIdx.x; i < rows; i += blockDim.x) {
        const int slot = held[i];
        if ((unsigned)slot >= (unsigned)slot_count) continue;
        int place = min(max(lengths[2 * (int64_t)slot], 0), room);
        for (int j = 0; j < i; ++j) place += held[j] == slot;
        if (place < room) history[(int64_t)slot * room + place] = tokens[i];
    }
    __syncthreads();                               // every length has been read
    for (int i = threadIdx.x; i < rows; i += blockDim.x) {
        const int slot = held[i];
        if ((unsigned)slot >= (unsigned)slot_count) continue;
        int more = 1;
        bool last = true;
        for (int j = 0; j < rows; ++j) {
            more += j < i && held[j] == slot;
            last = last && !(j > i && held[j] == slot);
        }
        // a slot's last row alone writes its length
        if (last) lengths[2 * (int64_t)slot] = min(min(max(lengths[2 * (int64_t)slot], 0), room) + more, room);
    }
}

}  // namespace

// The call's arguments as the Python side packs them.
struct RulesCall {
    const void* logits;
    long long row_stride;
    void* out;
    long long out_stride;
    const int* slots;
    const float* penalties;
    const int* lengths;
    const int* history;
    const int* bias_tokens;
    const float* bias_values;
    const uint32_t* masks;
    const int* mask_rows;
    int rows, vocab, slot_count, room, biases, mask_count, mask_words, dtype;
};

namespace {
template <typename T, int VEC, int SLICE> int launch_slices(const RulesCall& c, const Rules& rules, cudaStream_t stream) {
    const int slices = (c.vocab + SLICE - 1) / SLICE;
    if ((long long)c.rows * slices > 0x7fffffffLL) return TVB_BAD_ARGUMENT;
    const size_t shared = rules.biases > 0 ? SLICE * 4 : 0;
    logit_rules_kernel<T, VEC, SLICE><<<c.rows * slices, THREADS, shared, stream>>>((const T*)c.logits, c.row_stride, (T*)c.out, c.out_stride, c.vocab,
                                                                            slices, rules);
    return tvb_last_error();
}
template <typename T, int VEC> int launch_rules(const RulesCall& c, const Rules& rules, cudaStream_t stream) {
    return (long long)c.rows * ((c.vocab + LARGE_SLICE - 1) / LARGE_SLICE) <= 148 ? launch_slices<T, VEC, SMALL_SLICE>(c, rules, stream)
                                                                                   : launch_slices<T, VEC, LARGE_SLICE>(c, rules, stream);
}
}  // namespace

extern "C" int tvb_logit_rules(const RulesCall* call, void* stream) {
    const RulesCall& c = *call;
    if (c.rows <= 0 || c.vocab <= 0) return 0;
    if (c.slot_count < 0 || c.room < 0 || c.biases < 0 || c.biases > MAX_BIASES || (c.biases > 0 && (!c.bias_tokens || !c.bias_values)) ||
        (c.masks && (!c.mask_rows || (long long)c.mask_words * 32 < c.vocab)))
        return TVB_BAD_ARGUMENT;
    const Rules rules{c.slots, c.penalties, c.lengths, c.history, c.bias_tokens, c.bias_values, c.masks, c.mask_rows,
                      c.slot_count, c.room, c.biases, c.mask_count, c.mask_words};
    cudaStream_t s = (cudaStream_t)stream;
    const int size = c.dtype == TVB_F32 ? 4 : 2;
    const bool wide = !(((uintptr_t)c.logits | (uintptr_t)c.out) & 15) && c.row_stride * size % 16 == 0 && c.out_stride * size % 16 == 0;
    if (c.dtype == TVB_F32) return wide ? launch_rules<float, 4>(c, rules, s) : launch_rules<float, 1>(c, rules, s);
    if (c.dtype == TVB_BF16) return wide ? launch_rules<bf16, 8>(c, rules, s) : launch_rules<bf16, 1>(c, rules, s);
    return TVB_BAD_ARGUMENT;
}

extern "C" int tvb_append_tokens(const int* slots, const int* tokens, int rows, int* lengths, int* history, int slot_count, int room,
                                 void* stream) {
    if (rows <= 0) return 0;
    if (rows > 8192 || slot_count < 0 || room < 0) return TVB_BAD_ARGUMENT;
    const int threads = rows >= 256 ? 256 : (rows + 31) / 32 * 32;
    append_tokens_kernel<<<1, threads, rows * 4, (cudaStream_t)stream>>>(slots, tokens, rows, lengths, history, slot_count, room);
    return tvb_last_error();
}
