// Attention over the paged cache for tokens of which groups have their first keys in common: several answers to one prompt,
// or requests behind one system prompt.  softmax(q K^T scale) V over the keys 0 .. position of every token, where the keys
// below the group's shared length are read once for a tile of the group's query rows (tokens x query heads of one key/value
// head) instead of once a token.
//
// Softmax over a union of key ranges from the ranges' own results: a range gives its maximum m, l = sum exp(s - m) and
// O = sum exp(s - m) v, and ranges join as l = sum l_i exp(m_i - m), O = sum O_i exp(m_i - m).  The launches:
//   attend_shared   pieces of the shared keys, a tile of query rows each; m, l and O go to float32 scratch;
//   attend_own      what every token has behind them, a CTA a token, kv head and piece; to the scratch too;
//   join            every row's pieces in their order, and the result.
// The second does not need the first: launched programmatically it runs beside it (every CTA of the first waits for the kernel before,
// so what that wrote is there for both), and one of its CTAs waits for the first's end, so that the third has both behind it.  Where
// no keys are shared and no token's are cut, attend_own is all there is and stores the result itself.
//
// bfloat16, as a rule: tcgen05.mma for the shared pieces of head sizes 64 and 128 (attention_shared_tc.cuh), mma.sync on tiles that
// tensor-map copies bring for tokens' own keys, and for shared pieces of head size 256 (attention_own_tma.cuh).  Pages of other
// sizes, and 64 query rows of head size 256: mma.sync m16n8k16 over tiles that cp.async brings; a warp of a shared piece has 16
// query rows and every key, the warps of a token's own piece share the keys of a tile among them.  P is rounded to bfloat16 for the
// second product, whose operands are of one type (V's; a second part of P would double that product), the denominator sums what was not rounded: results are 0.0020 to 0.0023 off 64 bits on the whole, where the last rounding
// alone is 0.0017 off.  float32: the float32 cores.
//
// Bound by reading keys and values while a group has few query rows, by the shared pieces' products once it has many: 60 tokens with up
// to 431 keys of their own behind 6,144, 32 / 8 heads of size 128, take 28 us for 93 MB, 3.3 TB/s; three groups of 13 with up to 777 behind
// 2,896, 64 / 8 heads, 31 us for 112 MB, 3.6 TB/s.  What it is above the reading: 3 us before the first key arrives, 3 us for the join,
// and SMs that wait for the slowest piece.  float32, two groups of 5 behind 608 keys, 16 / 8 heads: 13.5 us for 16 MB.
#include "common.cuh"

namespace {

constexpr int THREADS = 128, WARPS = 4;
constexpr int KEYS = 64;                        // keys of a bfloat16 tile
constexpr int KEYS32 = 32;                      // keys of a float32 tile
constexpr int MAX_SHARED_PIECES = 64, MAX_OWN_PIECES = 64;
constexpr float LOG2E = 1.4426950408889634f;

struct Attend {
    const void* q;
    int64_t q_stride;
    const void* keys;                           // [pages, kv heads, page size, D]
    const void* values;
    const int* tables;                          // [rows, width]
    const int* token_row;                       // [tokens]
    const int* positions;                       // [tokens]
    const int* group_starts;                    // [groups + 1]
    const int* shared_lens;                     // [groups]
    float* part_o;                              // [tokens, q heads, shared and own pieces, D]; null: attend_own stores the result
    float* part_ml;                             // [tokens, q heads, shared and own pieces, 2]
    void* out;
    int64_t out_stride;
    int tokens, rows, width, groups, pages, page_size, num_q, num_kv;
    int shared_pieces, own_pieces, own_tiles;   // shared_pieces 0: every token reads all of its keys by itself
    float scale_log2;
};

struct Range { int first, end; };

// V neighbouring float32 (2, 4 or 8), from where another kernel may have written them
template <int V> __device__ __forceinline__ void load_lane(const float* from, float (&v)[V]) {
    if constexpr (V == 2) {
        const float2 f = __ldcg(reinterpret_cast<const float2*>(from));
        v[0] = f.x; v[1] = f.y;
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 f = __ldcg(reinterpret_cast<const float4*>(from + i));
            v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
        }
    }
}

// piece c of n keys in up to `pieces`: whole tiles of 64, of the shared keys whole blocks of 128
__device__ __forceinline__ int piece_keys(int n, int pieces) { return max(KEYS, ((n + pieces - 1) / pieces + KEYS - 1) / KEYS * KEYS); }
__device__ __forceinline__ int shared_piece_keys(int n, int pieces) { return max(2 * KEYS, ((n + pieces - 1) / pieces + 2 * KEYS - 1) / (2 * KEYS) * 2 * KEYS); }

// (__ldcg: plain loads may be served by an L1 that a kernel before filled, and attend_own starts without waiting)
__device__ __forceinline__ int shared_of_group(const Attend& a, int group) {
    return (int)min((int64_t)max(__ldcg(a.shared_lens + group), 0), (int64_t)a.width * a.page_size);
}
// The groups of a warp's lanes, 32 at a time: where the starts fall, a group begins (and ends) no earlier than the largest before it, so
// that no token stands in two groups, whatever the starts are, and no row has two writers.  `upto`: the end of the groups before.  (The
// rare case apart: inline it costs 0.2 us of 6.9 where no group is looked at, 0.3 of 31.1 in three groups of 13.)
__device__ __noinline__ int2 raise_starts(int start, int end, int upto) {
    int top = start;
    for (int d = 1; d < 32; d <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, top, d);
        if ((int)(threadIdx.x & 31) >= d) top = max(top, other);
    }
    start = max(top, upto);
    return make_int2(start, max(start, end));
}
__device__ __forceinline__ void keep_ascending(int& start, int& end, int& upto) {
    if (__any_sync(0xffffffffu, start > end || start < upto)) {
        const int2 raised = raise_starts(start, end, upto);
        start = raised.x;
        end = raised.y;
    }
    upto = __shfl_sync(0xffffffffu, end, 31);
}
// What a token reads: the row of its table (-1: it is none), its keys, and how many of them its group reads for it (those it
// shares if it reads them all, else none).  A whole warp asks, 32 groups at a time, all loads side by side.
struct Facts { int row, keys, shared; };
__device__ __forceinline__ Facts facts_of(const Attend& a, int token) {
    const int lane = threadIdx.x & 31;
    Facts f{__ldcg(a.token_row + token), __ldcg(a.positions + token), 0};
    int upto = 0;
    if (a.shared_pieces > 0)
        for (int g0 = 0; g0 < a.groups; g0 += 32) {
            int start = 0x7fffffff, end = 0x7fffffff, shared = 0;
            if (g0 + lane < a.groups) {
                start = max(__ldcg(a.group_starts + g0 + lane), 0);
                end = max(__ldcg(a.group_starts + g0 + lane + 1), 0);
                shared = shared_of_group(a, g0 + lane);
            }
            keep_ascending(start, end, upto);
            const uint32_t found = __ballot_sync(0xffffffffu, start <= token && token < end);
            if (found) {
                f.shared = __shfl_sync(0xffffffffu, shared, __ffs(found) - 1);
                break;
            }
        }
    if ((unsigned)f.row >= (unsigned)a.rows || f.keys < 0) f.row = -1;
    f.keys = (int)min((int64_t)f.keys + 1, (int64_t)a.width * a.page_size);
    if (f.keys < f.shared) f.shared = 0;
    return f;
}

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4_at(uint32_t* r, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans_at(uint32_t* r, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t* r, const bf16* p) { ldmatrix_x4_at(r, smem_address(p)); }
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t* r, const bf16* p) { ldmatrix_x4_trans_at(r, smem_address(p)); }

// One piece: ROWS query rows (token, head) of one kv head over the keys [range.first, range.end) of the request with this
// block table.
struct Piece {
    Range range;
    const int* table;
    int kv_head, slot, keys;                    // slot: which of the shared pieces it is; keys: the group's shared ones
    int token0, rows, row0;                     // row r: token token0 + (row0 + r) / heads, head (row0 + r) % heads
};

// The piece of the shared keys that this CTA has: `tile` query rows; false: none.
__device__ __forceinline__ bool find_shared_piece(const Attend& a, int tile_rows, Piece& p) {
    const int heads = a.num_q / a.num_kv, lane = threadIdx.x & 31;
    int item = blockIdx.x;
    const int piece = item % a.shared_pieces;
    item /= a.shared_pieces;
    p.kv_head = item % a.num_kv;
    int tile = item / a.num_kv;
    // the group that has the tile: 32 groups at a time
    int groups_upto = 0;
    for (int g0 = 0; g0 < a.groups; g0 += 32) {
        int start = a.tokens, end = a.tokens, shared = 0;
        if (g0 + lane < a.groups) {
            start = min(max(__ldcg(a.group_starts + g0 + lane), 0), a.tokens);
            end = min(max(__ldcg(a.group_starts + g0 + lane + 1), 0), a.tokens);
            shared = shared_of_group(a, g0 + lane);
        }
        keep_ascending(start, end, groups_upto);
        const int count = shared > 0 ? ((end - start) * heads + tile_rows - 1) / tile_rows : 0;
        int upto = count;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += other;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, upto > tile);
        if (past == 0) { tile -= __shfl_sync(0xffffffffu, upto, 31); continue; }
        const int at = __ffs(past) - 1;
        tile -= __shfl_sync(0xffffffffu, upto - count, at);
        start = __shfl_sync(0xffffffffu, start, at);
        end = __shfl_sync(0xffffffffu, end, at);
        const int n = __shfl_sync(0xffffffffu, shared, at), per = shared_piece_keys(n, a.shared_pieces);
        p.range = Range{piece * per, min(n, (piece + 1) * per)};
        if (p.range.first >= n) return false;
        // the table of the first token that reads all of the shared keys
        int row = -1;
        for (int token = start; token < end && row < 0; token += 32) {
            int mine = -1, position = -1;
            if (token + lane < end) {
                mine = __ldcg(a.token_row + token + lane);
                position = __ldcg(a.positions + token + lane);
            }
            const uint32_t reads = __ballot_sync(0xffffffffu, (unsigned)mine < (unsigned)a.rows && position >= n - 1);
            if (reads) row = __shfl_sync(0xffffffffu, mine, __ffs(reads) - 1);
        }
        if (row < 0) return false;
        p.keys = n;
        p.table = a.tables + (int64_t)row * a.width;
        p.token0 = start;
        p.row0 = tile * tile_rows;
        p.rows = min(tile_rows, (end - start) * heads - p.row0);
        p.slot = piece;
        return true;
    }
    return false;
}

// The piece of a token's own keys that this CTA has, up to `tile` of its query heads; false: none (p.rows rows of the token are
// there, though, for the first of its pieces: the token is padding, or has no keys but shared ones).
__device__ __forceinline__ bool find_own_piece(const Attend& a, int tile_rows, Piece& p) {
    int item = blockIdx.x;
    const int piece = item % a.own_pieces;
    item /= a.own_pieces;
    const int tile = item % a.own_tiles;
    item /= a.own_tiles;
    p.kv_head = item % a.num_kv;
    p.token0 = item / a.num_kv;
    p.row0 = tile * tile_rows;
    p.rows = min(tile_rows, a.num_q / a.num_kv - p.row0);
    p.slot = a.shared_pieces + piece;
    const Facts f = facts_of(a, p.token0);
    if (f.row < 0) return false;
    const int n = f.keys - f.shared, per = piece_keys(n, a.own_pieces);
    p.range = Range{f.shared + min(n, piece * per), f.shared + min(n, (piece + 1) * per)};
    p.table = a.tables + (int64_t)f.row * a.width;
    return p.range.first < p.range.end;
}
__device__ __forceinline__ int token_of(const Attend& a, const Piece& p, int r, int& head) {
    const int heads = a.num_q / a.num_kv, at = p.row0 + r;
    head = p.kv_head * heads + at % heads;
    return p.token0 + at / heads;
}
__device__ __forceinline__ int64_t part_of(const Attend& a, int token, int head, int slot) {
    return ((int64_t)token * a.num_q + head) * (a.shared_pieces + a.own_pieces) + slot;
}
// a token that takes part in its group's pieces: it is one, and reads all of the shared keys
__device__ __forceinline__ bool takes_part(const Attend& a, const Piece& p, int token) {
    const int row = __ldcg(a.token_row + token), position = __ldcg(a.positions + token);
    return (unsigned)row < (unsigned)a.rows && position >= p.keys - 1;          // (no table is shorter than the shared keys)
}
// place of a key's row in the cache, in rows of D (of which there are less than 2^31); -1: no such page
__device__ __forceinline__ int row_in(const Attend& a, const Piece& p, int page, int key) {
    return (unsigned)page < (unsigned)a.pages ? (page * a.num_kv + p.kv_head) * a.page_size + key % a.page_size : -1;
}
__device__ __forceinline__ int cache_row(const Attend& a, const Piece& p, int key) {
    return row_in(a, p, __ldcg(p.table + key / a.page_size), key);
}

// ----------------------------------------------------------- joining the pieces
// What the warps of an attend_own CTA end with, in shared memory: their rows' O [WARPS][OWN][D] and (m, l) [WARPS][OWN][2].
template <int D, int OWN> struct Ends {
    static constexpr int PITCH = D + 4, FLOATS = WARPS * OWN * (PITCH + 2);
    float* o;
    float* ml;
    __device__ __forceinline__ explicit Ends(float* at) : o(at), ml(at + WARPS * OWN * PITCH) {}
};

template <typename T, int V> __device__ __forceinline__ void store_lane(T* to, const float (&v)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = from_float<T>(v[e]);
}

// Every warp has stored its share (the barrier is here): a warp a row, the warps' shares as one piece, or as the result; `rows`: whose.
template <typename T, int D, int OWN>
__device__ __forceinline__ void finish_own(const Attend& a, const Piece& p, const Ends<D, OWN>& ends, uint32_t rows = ~0u) {
    using E = Ends<D, OWN>;
    constexpr int V = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    for (int r = warp; warp < WARPS && r < p.rows; r += WARPS) {
        if (!(rows >> r & 1)) continue;
        float top = -INFINITY, total = 0.0f, sum[V] = {};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, ends.ml[2 * (w * OWN + r)]);
        const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = exp2f(ends.ml[2 * (w * OWN + r)] - ref);
            total = fmaf(f, ends.ml[2 * (w * OWN + r) + 1], total);
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] = fmaf(f, ends.o[(w * OWN + r) * E::PITCH + lane * V + e], sum[e]);
        }
        int head;
        const int token = token_of(a, p, r, head);
        if (a.part_o) {
            const int64_t part = part_of(a, token, head, p.slot);
            store_lane(a.part_o + part * D + lane * V, sum);
            if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + part * 2) = make_float2(top, total);
        } else {
            const float inverse = total == 0.0f ? 0.0f : 1.0f / total;          // no key is seen: zeros
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] *= inverse;
            store_lane(reinterpret_cast<T*>(a.out) + token * a.out_stride + head * D + lane * V, sum);
        }
    }
}

// The kernels' waits (see the top).
__device__ __forceinline__ void start_own(const Attend& a) {
    if (a.shared_pieces == 0) pdl_wait();
    pdl_launch_dependents();
}
__device__ __forceinline__ void end_own(const Attend& a) {
    if (a.shared_pieces > 0 && blockIdx.x + 1 == gridDim.x) pdl_wait();
}
// The rows of a CTA without keys, where nobody joins pieces: zeros.
template <typename T, int D> __device__ __forceinline__ void store_zeros(const Attend& a, const Piece& p) {
    if (a.part_o) return;
    for (int i = threadIdx.x; i < p.rows * D; i += blockDim.x) {
        int head;
        const int token = token_of(a, p, i / D, head);
        reinterpret_cast<T*>(a.out)[token * a.out_stride + head * D + i % D] = from_float<T>(0.0f);
    }
}

// a warp a row: a token's query head
template <typename T, int D> __global__ void __launch_bounds__(THREADS) join_kernel(Attend a) {
    constexpr int V = D / 32, EACH = (MAX_SHARED_PIECES + MAX_OWN_PIECES) / 32, AHEAD = 8;      // values, parts of a lane; pieces in flight
    const int lane = threadIdx.x & 31;
    const int64_t at = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    const int token = (int)(at / a.num_q), head = (int)(at % a.num_q), slots = a.shared_pieces + a.own_pieces;
    // which pieces there are: by what was there before attend_shared, so before this waits
    int shared_used = 0, own_used = 0;
    if (token < a.tokens) {
        const Facts f = facts_of(a, token);
        if (f.row >= 0) {
            const int own = f.keys - f.shared;
            if (f.shared > 0) shared_used = (f.shared - 1) / shared_piece_keys(f.shared, a.shared_pieces) + 1;
            if (own > 0) own_used = (own - 1) / piece_keys(own, a.own_pieces) + 1;
        }
    }
    const int parts = shared_used + own_used, gap = a.shared_pieces - shared_used;
    pdl_wait();
    pdl_launch_dependents();
    if (token >= a.tokens) return;
    const int64_t first = part_of(a, token, head, 0);
    float m[EACH], weight[EACH], top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const float2 v = lane + 32 * i < slots ? __ldcg(reinterpret_cast<const float2*>(a.part_ml) + first + lane + 32 * i) : make_float2(0, 0);
        m[i] = v.x; weight[i] = v.y;
    }
    float v[AHEAD][V];
    const float* from = a.part_o + first * D + lane * V;
    auto load = [&](int part) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int slot = part + j < shared_used ? part + j : part + j + gap;
            if (part + j < parts) load_lane<V>(from + (int64_t)slot * D, v[j]);
        }
    };
    load(0);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int slot = lane + 32 * i;
        const bool used = slot < shared_used || (slot >= a.shared_pieces && slot < a.shared_pieces + own_used);
        if (!used) { m[i] = -INFINITY; weight[i] = 0.0f; }
        top = fmaxf(top, m[i]);
    }
    top = warp_max(top);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        m[i] = exp2f(m[i] - ref);
        total = fmaf(m[i], weight[i], total);
    }
    total = warp_sum(total);
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;                  // a token that is none, or sees no key: zeros
#pragma unroll
    for (int i = 0; i < EACH; ++i) m[i] *= inverse;
    float sum[V] = {};
    for (int part = 0; part < parts; part += AHEAD) {
        if (part > 0) load(part);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int slot = part + j < shared_used ? part + j : part + j + gap;
            float w = __shfl_sync(0xffffffffu, m[0], slot & 31);
#pragma unroll
            for (int i = 1; i < EACH; ++i) {
                const float other = __shfl_sync(0xffffffffu, m[i], slot & 31);
                if (slot >> 5 == i) w = other;
            }
            if (part + j < parts)
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e] = fmaf(w, v[j][e], sum[e]);
        }
    }
    store_lane(reinterpret_cast<T*>(a.out) + token * a.out_stride + head * D + lane * V, sum);
}

// ------------------------------------------------------------------ bfloat16
template <int D> struct Tiles {
    static constexpr int PITCH = D + 8;
    static constexpr int TILE = KEYS * PITCH;                                   // elements of a K or V tile
    static constexpr int bytes(int rows) { return (rows + 4 * KEYS) * PITCH * 2 + 3 * KEYS * 4 + 3 * 2 * 4 + 64; }
};

// A piece of the shared keys, 64 query rows, 16 a warp: for what the kernel of attention_shared_tc.cuh does not take.
template <int D>
__device__ __forceinline__ void attend_shared_piece(const Attend& a, const Piece& p, unsigned char* raw) {
    constexpr int PITCH = Tiles<D>::PITCH, ROWS = 64, NK = KEYS;
    bf16* q_s = reinterpret_cast<bf16*>(raw);                                   // [ROWS][PITCH]
    bf16* k_s = q_s + ROWS * PITCH;                                              // [2][KEYS][PITCH]
    bf16* v_s = k_s + 2 * Tiles<D>::TILE;
    // of a tile's keys: the place of their rows (-1: none), and which there are.  Three tiles of them: one warp may look up
    // those of a tile while another still reads the bits of the one two before.
    int* at_s = reinterpret_cast<int*>(v_s + 2 * Tiles<D>::TILE);               // [3][KEYS]
    uint32_t* there_s = reinterpret_cast<uint32_t*>(at_s + 3 * KEYS);           // [3][2]
    bool* takes_s = reinterpret_cast<bool*>(there_s + 6);                       // [ROWS] tokens that take part
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const bf16* keys = reinterpret_cast<const bf16*>(a.keys);
    const bf16* values = reinterpret_cast<const bf16*>(a.values);
    const int tiles = (p.range.end - p.range.first + KEYS - 1) / KEYS;

    // (a page's number is asked for a tile before it is looked at)
    auto page_of = [&](int tile) -> int {
        const int key = p.range.first + tile * KEYS + tid;
        return tid < KEYS && key < p.range.end ? __ldcg(p.table + key / a.page_size) : -1;
    };
    auto place = [&](int tile, int page) {                                      // the first two warps
        const int slot = tile % 3;
        if (tid < KEYS) {
            const int key = p.range.first + tile * KEYS + tid;
            const int at = key < p.range.end ? row_in(a, p, page, key) : -1;
            at_s[slot * KEYS + tid] = at;
            const uint32_t there = __ballot_sync(0xffffffffu, at >= 0);
            if (lane == 0) there_s[slot * 2 + warp] = there;
        }
    };
    auto load = [&](int tile) {
        const int buffer = tile & 1, slot = tile % 3;
        constexpr int WORDS = D / 8;
#pragma unroll 4
        for (int i = tid; i < KEYS * WORDS; i += THREADS) {
            const int key = i / WORDS, word = i % WORDS;
            const int at = at_s[slot * KEYS + key];
            const int64_t from = (int64_t)max(at, 0) * D + word * 8;
            cp_async_16(k_s + buffer * Tiles<D>::TILE + key * PITCH + word * 8, keys + from, at >= 0);
            cp_async_16(v_s + buffer * Tiles<D>::TILE + key * PITCH + word * 8, values + from, at >= 0);
        }
        cp_async_commit();
    };
    const int first_page = page_of(0);
    int next_page = page_of(1);
    if (tid < ROWS) {
        int head;
        takes_s[tid] = tid < p.rows && takes_part(a, p, token_of(a, p, tid, head));
    }
#pragma unroll 4
    for (int i = tid; i < ROWS * (D / 8); i += THREADS) {
        const int r = i / (D / 8), word = i % (D / 8);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < p.rows) {
            int head;
            const int token = token_of(a, p, r, head);
            v = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.q) + token * a.q_stride + head * D + word * 8));
        }
        *reinterpret_cast<uint4*>(q_s + r * PITCH + word * 8) = v;
    }
    place(0, first_page);
    __syncthreads();
    if (tiles > 0) load(0);
    const bf16* q_rows = q_s + warp * 16 * PITCH + (lane & 15) * PITCH + (lane >> 4) * 8;
    uint32_t q_frag[D <= 128 ? D / 16 : 1][4];
    if constexpr (D <= 128)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) ldmatrix_x4(q_frag[ks], q_rows + ks * 16);

    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    for (int tile = 0; tile < tiles; ++tile) {
        const int buffer = tile & 1;
        if (tile + 1 < tiles) {
            place(tile + 1, next_page);
            next_page = page_of(tile + 2);
        }
        cp_async_wait<0>();
        __syncthreads();                                                        // the tile is there; places of the next too
        if (tile + 1 < tiles) load(tile + 1);
        const bf16* k_tile = k_s + buffer * Tiles<D>::TILE;
        const bf16* v_tile = v_s + buffer * Tiles<D>::TILE;
        float s[NK / 8][4];
#pragma unroll
        for (int n = 0; n < NK / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t q_now[4];
            if constexpr (D > 128) ldmatrix_x4(q_now, q_rows + ks * 16);
            const uint32_t (&q4)[4] = D <= 128 ? q_frag[D <= 128 ? ks : 0] : q_now;
#pragma unroll
            for (int np = 0; np < NK / 16; ++np) {
                uint32_t b[4];
                const int matrix = lane >> 3;
                ldmatrix_x4(b, k_tile + (np * 16 + (matrix >> 1) * 8 + (lane & 7)) * PITCH + ks * 16 + (matrix & 1) * 8);
                mma_16816(s[2 * np], q4, b[0], b[1]);
                mma_16816(s[2 * np + 1], q4, b[2], b[3]);
            }
        }
        const uint64_t there = (uint64_t)there_s[tile % 3 * 2] | (uint64_t)there_s[tile % 3 * 2 + 1] << 32;
        float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < NK / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[n][i] *= a.scale_log2;
                if (~there != 0 && !(there >> (n * 8 + 2 * t4 + (i & 1)) & 1)) s[n][i] = -INFINITY;
                most[i >> 1] = fmaxf(most[i >> 1], s[n][i]);
            }
        float subtract[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 1));
            most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 2));
            const float now = fmaxf(m[h], most[h]);
            subtract[h] = now == -INFINITY ? 0.0f : now;                        // no inf - inf where no key was seen yet
            const float factor = exp2_unit(m[h] - subtract[h]);
            m[h] = now;
            l[h] *= factor;
            most[h] = factor;
        }
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] *= most[i >> 1];
#pragma unroll
        for (int kk = 0; kk < NK / 16; ++kk) {
            uint32_t weights[4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int n = 2 * kk + half;
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = exp2_unit(s[n][i] - subtract[i >> 1]);
                    l[i >> 1] += w[i];
                }
                weights[2 * half] = pack_bf16x2(w[0], w[1]);
                weights[2 * half + 1] = pack_bf16x2(w[2], w[3]);
            }
#pragma unroll
            for (int dp = 0; dp < D / 16; ++dp) {
                uint32_t b[4];
                const int matrix = lane >> 3;
                ldmatrix_x4_trans(b, v_tile + (kk * 16 + (matrix & 1) * 8 + (lane & 7)) * PITCH + dp * 16 + (matrix >> 1) * 8);
                mma_16816(o[2 * dp], weights, b[0], b[1]);
                mma_16816(o[2 * dp + 1], weights, b[2], b[3]);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = warp * 16 + g + 8 * h;
        if (r >= p.rows || !takes_s[r]) continue;
        int head;
        const int token = token_of(a, p, r, head);
        const int64_t part = part_of(a, token, head, p.slot);
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(a.part_o + part * D + n * 8 + 2 * t4) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        if (t4 == 0) *reinterpret_cast<float2*>(a.part_ml + part * 2) = make_float2(m[h], l[h]);
    }
}

template <int D> __global__ void __launch_bounds__(THREADS) attend_shared_bf16_kernel(Attend a) {
    extern __shared__ __align__(16) unsigned char raw[];
    pdl_wait();
    pdl_launch_dependents();
    Piece p;
    if (find_shared_piece(a, 64, p)) attend_shared_piece<D>(a, p, raw);
}

// A token's own keys: up to 16 of its query heads (one tile of the instruction), tiles of 32 keys, eight a warp, in a ring of three.
template <int D> struct OwnTiles {
    static constexpr int KEYS = 32, RING = 3, PITCH = D + 8, TILE = KEYS * PITCH;
    static constexpr int RING_BYTES = (16 + 2 * RING * KEYS) * PITCH * 2, END_BYTES = Ends<D, 16>::FLOATS * 4;
    static constexpr int BYTES = (RING_BYTES > END_BYTES ? RING_BYTES : END_BYTES) + 8 * KEYS * 4 + 8 * 4;
    static constexpr int CTAS = D == 64 ? 6 : D == 128 ? 4 : 2;                 // on an SM
};
__device__ __forceinline__ void mma_1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(b0));
}

template <int D> __global__ void __launch_bounds__(THREADS, OwnTiles<D>::CTAS) attend_own_bf16_kernel(Attend a) {
    using S = OwnTiles<D>;
    constexpr int PITCH = S::PITCH, WORDS = D / 8;
    extern __shared__ __align__(16) unsigned char raw[];
    start_own(a);
    Piece p;
    if (!find_own_piece(a, 16, p)) {
        store_zeros<bf16, D>(a, p);
        end_own(a);
        return;
    }
    bf16* q_s = reinterpret_cast<bf16*>(raw);                                   // [16][PITCH]
    bf16* k_s = q_s + 16 * PITCH;                                               // [RING][KEYS][PITCH]
    bf16* v_s = k_s + S::RING * S::TILE;
    // of a tile's keys: the place of their rows (-1: none), and which there are; eight places, of which four are in use at once: the last
    // is looked up while a slow warp is still at the first
    int* at_s = reinterpret_cast<int*>(raw + S::BYTES - 8 * S::KEYS * 4 - 8 * 4);                // [8][KEYS]
    uint32_t* there_s = reinterpret_cast<uint32_t*>(at_s + 8 * S::KEYS);        // [8]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const bf16* keys = reinterpret_cast<const bf16*>(a.keys);
    const bf16* values = reinterpret_cast<const bf16*>(a.values);
    const int tiles = (p.range.end - p.range.first + S::KEYS - 1) / S::KEYS;
    // the first warp; a page's number is asked for a tile before it is looked at
    auto page_of = [&](int tile) -> int {
        const int key = p.range.first + tile * S::KEYS + lane;
        return warp == 0 && key < p.range.end ? __ldcg(p.table + key / a.page_size) : -1;
    };
    auto place = [&](int tile, int page) {
        if (warp != 0) return;
        const int key = p.range.first + tile * S::KEYS + lane;
        const int at = key < p.range.end ? row_in(a, p, page, key) : -1;
        at_s[(tile & 7) * S::KEYS + lane] = at;
        const uint32_t there = __ballot_sync(0xffffffffu, at >= 0);
        if (lane == 0) there_s[tile & 7] = there;
    };
    auto load = [&](int tile) {
        if (tile < tiles) {
            bf16* k_to = k_s + tile % S::RING * S::TILE;
            bf16* v_to = v_s + tile % S::RING * S::TILE;
#pragma unroll 4
            for (int i = tid; i < S::KEYS * WORDS; i += THREADS) {
                const int key = i / WORDS, word = i % WORDS;
                const int at = at_s[(tile & 7) * S::KEYS + key];
                const int64_t from = (int64_t)max(at, 0) * D + word * 8;
                cp_async_16(k_to + key * PITCH + word * 8, keys + from, at >= 0);
                cp_async_16(v_to + key * PITCH + word * 8, values + from, at >= 0);
            }
        }
        cp_async_commit();
    };
    {
        int pages[S::RING - 1];
#pragma unroll
        for (int i = 0; i < S::RING - 1; ++i) pages[i] = page_of(i);
        for (int i = tid; i < 16 * WORDS; i += THREADS) {
            const int r = i / WORDS, word = i % WORDS;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < p.rows) {
                int head;
                const int token = token_of(a, p, r, head);
                v = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.q) + token * a.q_stride + head * D + word * 8));
            }
            *reinterpret_cast<uint4*>(q_s + r * PITCH + word * 8) = v;
        }
#pragma unroll
        for (int i = 0; i < S::RING - 1; ++i) place(i, pages[i]);
    }
    int next_page = page_of(S::RING - 1);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S::RING - 1; ++i) load(i);
    const bf16* q_rows = q_s + (lane & 15) * PITCH + (lane >> 4) * 8;
    uint32_t q_frag[D <= 128 ? D / 16 : 1][4];
    if constexpr (D <= 128)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) ldmatrix_x4(q_frag[ks], q_rows + ks * 16);
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    for (int tile = 0; tile < tiles; ++tile) {
        place(tile + S::RING - 1, next_page);
        next_page = page_of(tile + S::RING);
        cp_async_wait<S::RING - 2>();
        __syncthreads();                        // the tile is there, the places of the one after next too, the one before is through
        load(tile + S::RING - 1);
        const int at = (warp * 8 + (lane & 7)) * PITCH + (lane >> 3) * 8;       // of this warp's keys, 32 values at a time
        const bf16* k_tile = k_s + tile % S::RING * S::TILE + at;
        const bf16* v_tile = v_s + tile % S::RING * S::TILE + at;
        float s[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
            uint32_t b[4];
            ldmatrix_x4(b, k_tile + ks * 32);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t q_now[4];
                if constexpr (D > 128) ldmatrix_x4(q_now, q_rows + (2 * ks + half) * 16);
                const uint32_t (&q4)[4] = D <= 128 ? q_frag[D <= 128 ? 2 * ks + half : 0] : q_now;
                mma_16816(s[half], q4, b[2 * half], b[2 * half + 1]);
            }
        }
        const uint32_t there = there_s[tile & 7] >> (warp * 8);
        float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[0][i] = there >> (2 * t4 + (i & 1)) & 1 ? (s[0][i] + s[1][i]) * a.scale_log2 : -INFINITY;
            most[i >> 1] = fmaxf(most[i >> 1], s[0][i]);
        }
        float subtract[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 1));
            most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 2));
            const float now = fmaxf(m[h], most[h]);
            subtract[h] = now == -INFINITY ? 0.0f : now;                        // no inf - inf where no key was seen yet
            most[h] = exp2_unit(m[h] - subtract[h]);
            m[h] = now;
            l[h] *= most[h];
        }
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = exp2_unit(s[0][i] - subtract[i >> 1]);
            l[i >> 1] += w[i];
        }
        const uint32_t w_lo = pack_bf16x2(w[0], w[1]), w_hi = pack_bf16x2(w[2], w[3]);
        if (__any_sync(0xffffffffu, most[0] != 1.0f || most[1] != 1.0f))
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][i] *= most[i >> 1];
#pragma unroll
        for (int dp = 0; dp < D / 32; ++dp) {
            uint32_t b[4];
            ldmatrix_x4_trans(b, v_tile + dp * 32);
#pragma unroll
            for (int j = 0; j < 4; ++j) mma_1688(o[4 * dp + j], w_lo, w_hi, b[j]);
        }
    }
    cp_async_wait<0>();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    const Ends<D, 16> ends(reinterpret_cast<float*>(raw));                      // over the tiles
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h, at = warp * 16 + r;
        if (r >= p.rows) continue;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(ends.o + at * Ends<D, 16>::PITCH + n * 8 + 2 * t4) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        if (t4 == 0) *reinterpret_cast<float2*>(ends.ml + 2 * at) = make_float2(m[h], l[h]);
    }
    finish_own<bf16, D, 16>(a, p, ends);
    end_own(a);
}

// ------------------------------------------------------------------- float32
// 16 query rows, four a warp: a lane has a key of the tile for the scores, D / 32 values of every row for the sums.
template <int D>
__global__ void __launch_bounds__(THREADS) attend_shared_f32_kernel(Attend a) {
    constexpr int PITCH = D + 4, VALUES = D / 32;
    extern __shared__ __align__(16) float tiles_s[];
    float* k_s = tiles_s;                                                       // [KEYS32][PITCH]
    float* v_s = k_s + KEYS32 * PITCH;
    float* q_s = v_s + KEYS32 * PITCH;                                          // [16][D]
    __shared__ uint32_t there_s;
    __shared__ bool takes_s[16];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_launch_dependents();
    Piece p;
    if (!find_shared_piece(a, 16, p)) return;
    const float* keys = reinterpret_cast<const float*>(a.keys);
    const float* values = reinterpret_cast<const float*>(a.values);
    if (tid < 16) {
        int head;
        takes_s[tid] = tid < p.rows && takes_part(a, p, token_of(a, p, tid, head));
    }
    for (int i = tid; i < 16 * (D / 4); i += THREADS) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float4 v = make_float4(0, 0, 0, 0);
        if (r < p.rows) {
            int head;
            const int token = token_of(a, p, r, head);
            v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + token * a.q_stride + head * D + d);
        }
        *reinterpret_cast<float4*>(q_s + r * D + d) = v;
    }
    float o[4][VALUES] = {}, m[4], l[4] = {};
#pragma unroll
    for (int r = 0; r < 4; ++r) m[r] = -INFINITY;
    const bool works = warp * 4 < p.rows;
    for (int key0 = p.range.first; key0 < p.range.end; key0 += KEYS32) {
        __syncthreads();                                                        // the tile before is through
        // a warp brings the keys warp, warp + 4, ..
        for (int key = warp; key < KEYS32; key += WARPS) {
            const int64_t at = key0 + key < p.range.end ? cache_row(a, p, key0 + key) : -1;
            for (int d = lane * 4; d < D; d += 128) {
                const float4 zero = make_float4(0, 0, 0, 0);
                *reinterpret_cast<float4*>(k_s + key * PITCH + d) = at < 0 ? zero : *reinterpret_cast<const float4*>(keys + at * D + d);
                *reinterpret_cast<float4*>(v_s + key * PITCH + d) = at < 0 ? zero : *reinterpret_cast<const float4*>(values + at * D + d);
            }
        }
        if (warp == 0) {
            const uint32_t there = __ballot_sync(0xffffffffu, key0 + lane < p.range.end && cache_row(a, p, key0 + lane) >= 0);
            if (lane == 0) there_s = there;
        }
        __syncthreads();
        if (!works) continue;
        float s[4] = {};
#pragma unroll 8
        for (int d = 0; d < D; d += 4) {
            const float4 kv = *reinterpret_cast<const float4*>(k_s + lane * PITCH + d);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4 qv = *reinterpret_cast<const float4*>(q_s + (warp * 4 + r) * D + d);
                s[r] = fmaf(qv.x, kv.x, s[r]); s[r] = fmaf(qv.y, kv.y, s[r]);
                s[r] = fmaf(qv.z, kv.z, s[r]); s[r] = fmaf(qv.w, kv.w, s[r]);
            }
        }
        const bool there = there_s >> lane & 1;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            s[r] = there ? s[r] * a.scale_log2 : -INFINITY;
            const float now = fmaxf(m[r], warp_max(s[r])), subtract = now == -INFINITY ? 0.0f : now;
            const float factor = exp2f(m[r] - subtract);
            m[r] = now;
            s[r] = exp2f(s[r] - subtract);
            l[r] = l[r] * factor + s[r];                                        // a lane's own share
#pragma unroll
            for (int e = 0; e < VALUES; ++e) o[r][e] *= factor;
        }
#pragma unroll 8
        for (int key = 0; key < KEYS32; ++key) {
            float v[VALUES];
#pragma unroll
            for (int e = 0; e < VALUES; ++e) v[e] = v_s[key * PITCH + e * 32 + lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float w = __shfl_sync(0xffffffffu, s[r], key);
#pragma unroll
                for (int e = 0; e < VALUES; ++e) o[r][e] = fmaf(w, v[e], o[r][e]);
            }
        }
    }
    if (!works) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float total = warp_sum(l[r]);
        if (warp * 4 + r >= p.rows || !takes_s[warp * 4 + r]) continue;
        int head;
        const int token = token_of(a, p, warp * 4 + r, head);
        const int64_t part = part_of(a, token, head, p.slot);
#pragma unroll
        for (int e = 0; e < VALUES; ++e) a.part_o[part * D + e * 32 + lane] = o[r][e];
        if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + part * 2) = make_float2(m[r], total);
    }
}

// Up to four query heads of a token: a warp takes every fourth key, a lane D / 32 neighbouring values of it.
template <int D>
__global__ void __launch_bounds__(THREADS) attend_own_f32_kernel(Attend a) {
    constexpr int OWN = 4, V = D / 32, AHEAD = D <= 128 ? 4 : 2;                // keys of a warp in flight
    using E = Ends<D, OWN>;
    extern __shared__ __align__(16) unsigned char raw[];
    start_own(a);
    Piece p;
    if (!find_own_piece(a, OWN, p)) {
        store_zeros<float, D>(a, p);
        end_own(a);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* keys = reinterpret_cast<const float*>(a.keys);
    const float* values = reinterpret_cast<const float*>(a.values);
    float q[OWN][V] = {}, o[OWN][V] = {}, m[OWN], l[OWN] = {};
#pragma unroll
    for (int r = 0; r < OWN; ++r) {
        m[r] = -INFINITY;
        if (r >= p.rows) continue;
        int head;
        const int token = token_of(a, p, r, head);
        load_lane<V>(reinterpret_cast<const float*>(a.q) + token * a.q_stride + head * D + lane * V, q[r]);
    }
    // The warp's keys are p.range.first + warp + 4 n; a lane looks up where every 32nd of them lies, and those of the next 32 meanwhile.
    const int mine = max(0, (p.range.end - p.range.first - warp + WARPS - 1) / WARPS);
    auto place = [&](int n) -> int { return n < mine ? cache_row(a, p, p.range.first + warp + WARPS * n) : -1; };
    int places = place(lane), next_places = place(lane + 32);
    float k[2][AHEAD][V], v[2][AHEAD][V];       // of these keys, and of the next
    uint32_t there[2];
    auto fetch = [&](int n, int buffer, int from) {                              // from: the places of keys n / 32 * 32 ..
        there[buffer] = 0;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int64_t at = __shfl_sync(0xffffffffu, from, (n + i) & 31);
            if (at >= 0) {
                there[buffer] |= 1u << i;
                load_lane<V>(keys + at * D + lane * V, k[buffer][i]);
                load_lane<V>(values + at * D + lane * V, v[buffer][i]);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) k[buffer][i][e] = v[buffer][i][e] = 0.0f;
            }
        }
    };
    auto take = [&](int buffer) {
#pragma unroll
        for (int r = 0; r < OWN; ++r) {
            if (r >= p.rows) continue;
            float s[AHEAD], now = m[r];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                float dot = 0.0f;
#pragma unroll
                for (int e = 0; e < V; ++e) dot = fmaf(q[r][e], k[buffer][i][e], dot);
                s[i] = warp_sum(dot) * a.scale_log2;
                if (!(there[buffer] >> i & 1)) s[i] = -INFINITY;
                now = fmaxf(now, s[i]);
            }
            const float subtract = now == -INFINITY ? 0.0f : now, factor = exp2f(m[r] - subtract);
            m[r] = now;
            l[r] *= factor;
#pragma unroll
            for (int e = 0; e < V; ++e) o[r][e] *= factor;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const float w = exp2f(s[i] - subtract);
                l[r] += w;
#pragma unroll
                for (int e = 0; e < V; ++e) o[r][e] = fmaf(w, v[buffer][i][e], o[r][e]);
            }
        }
    };
    fetch(0, 0, places);
    for (int n = 0; n < mine; n += 2 * AHEAD) {
        fetch(n + AHEAD, 1, places);            // (AHEAD divides 16: the same 32 keys)
        take(0);
        if ((n + 2 * AHEAD) % 32 == 0) {
            places = next_places;
            next_places = place(n + 2 * AHEAD + 32 + lane);
        }
        fetch(n + 2 * AHEAD, 0, places);
        take(1);
    }
    const E ends(reinterpret_cast<float*>(raw));
#pragma unroll
    for (int r = 0; r < OWN; ++r) {
        const int at = warp * OWN + r;
#pragma unroll
        for (int i = 0; i < V; ++i) ends.o[at * E::PITCH + lane * V + i] = o[r][i];
        if (lane == 0) { ends.ml[2 * at] = m[r]; ends.ml[2 * at + 1] = l[r]; }
    }
    finish_own<float, D, OWN>(a, p, ends);
    end_own(a);
}

#include "attention_shared_tc.cuh"
#include "attention_own_tma.cuh"

// ------------------------------------------------------------------ host side
long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

struct Plan {
    long long shared_items, own_items;
    int shared_pieces, own_pieces, own_tiles;
    int pieces() const { return shared_pieces + own_pieces; }   // of a row; with 1 there is nothing to join
    int tile_tokens;                            // tokens of a tile on the tensor cores of the fifth generation; 0: the other kernels
    bool by_sixteen;                            // shared pieces in tiles of 16 query rows, by attend_own_tma_kernel
};

// Into how many pieces the keys are cut, none shorter than MIN_KEYS: the tokens' own for about four CTAs an SM; the shared ones, on the
// tensor cores, for one CTA on as many SMs as are their share of the work (a block of 128 keys takes a tile 1.2 us, a token's own
// keys come in at 47 KB a us and SM), LEAST_SMS at least, so that attend_own's CTAs run on the others meanwhile (60 tokens with up to
// 431 keys behind 6,144: 31.1 us with 96, 28.2 with 64, 31.2 with 48; three groups of 13 with up to 777 behind 2,896, 64 / 8 heads:
// 39.7, 31.3, 31.3; 64 tokens with up to 64 behind 8,192, 64 / 8 heads: 42 with 148, 53 with 100, 87 with 74).
Plan plan_of(int tokens, int groups, int num_q, int num_kv, int head_dim, int pages, int page_size, long long max_shared, long long max_own, int dtype) {
    constexpr int MIN_KEYS = 128, SMS = 148, LEAST_SMS = 64;
    const int heads = num_q / num_kv;
    Plan p;
    p.tile_tokens = dtype == TVB_BF16 && pages > 0 && tc_takes(head_dim, heads, page_size) ? TC_ROWS / heads : 0;
    // Head size 256, whose 64 query rows leave a tile of keys no room to be ahead: 16 rows, if a group has no more as a rule (8 / 4 heads,
    // three groups, us 16 rows / 64: 4 tokens behind 5,808 keys 22 / 32, four of 7 behind 368 11.8 / 13.4; 11 tokens, two tiles of 16,
    // behind 4,320 33.7 / 32.3).
    p.by_sixteen = dtype == TVB_BF16 && head_dim == 256 && pages > 0 && own_tma_takes(page_size) && (long long)tokens * heads <= 16ll * max(groups, 1);
    // CTAs' tiles: at most, and as a rule
    long long tiles = 0, usual = 1;
    // Up to so many values (32 MB of bfloat16) the tokens read the shared keys by themselves, in one launch or two: the third
    // and the reading in pieces cost more (16 / 8 heads, head size 128, us alone / shared: 2 tokens behind 2,048 keys 9.8 / 13.6, 4 12 /
    // 13.5, 8 behind 1,024 12.5 / 12.3, 16 behind 512 12.7 / 11.6; float32 8 behind 1,024 25 / 37, 16 behind 512 33 / 36).
    constexpr long long FEW_VALUES = 1ll << 23;
    const bool alone = (long long)tokens * num_kv * head_dim * max_shared <= FEW_VALUES;
    if (alone) max_own += max_shared;
    if (groups > 0 && max_shared > 0 && !alone) {
        const long long in_tile = p.tile_tokens > 0 ? p.tile_tokens * heads : dtype == TVB_F32 || p.by_sixteen ? 16 : 64;
        tiles = groups + (long long)tokens * heads / in_tile;
        usual = max((long long)groups, ceil_div((long long)tokens * heads, in_tile));
    }
    auto pieces_of = [&](long long ctas, long long items, long long keys, int most) {
        const long long wanted = items > 0 ? max(1ll, ctas / items) : 1;
        return (int)max(1ll, min(min(wanted, ceil_div(max(keys, 1ll), MIN_KEYS)), (long long)most));
    };
    p.own_tiles = (int)ceil_div(heads, dtype == TVB_F32 ? 4 : 16);
    const double own_us = (double)tokens * num_kv * max_own * head_dim * (dtype == TVB_F32 ? 8 : 4) / 47e3;
    const double shared_us = 1.2 * usual * num_kv * (max_shared / 128.0);
    const int share = max(LEAST_SMS, (int)(SMS * shared_us / (shared_us + own_us + 1e-9)));
    // (the other kernels: a round of their CTAs; head size 256, 33 tokens behind 4,320: 32 us in one round, 45 in three)
    const int others = dtype == TVB_BF16 && head_dim == 256 ? SMS : 3 * SMS;
    p.shared_pieces = tiles > 0 ? pieces_of(p.tile_tokens > 0 ? share : others, usual * num_kv, max_shared, MAX_SHARED_PIECES) : 0;
    p.own_pieces = pieces_of(4 * SMS, (long long)tokens * num_kv * p.own_tiles, max_own, MAX_OWN_PIECES);
    if (tiles == 0 && dtype == TVB_BF16 && max_own <= 2 * MIN_KEYS) p.own_pieces = 1;            // not worth the launch that joins them
    p.shared_items = tiles * num_kv * p.shared_pieces;
    p.own_items = (long long)tokens * num_kv * p.own_tiles * p.own_pieces;
    return p;
}

template <typename K> int launch(K kernel, long long grid, size_t shared, int pdl, cudaStream_t stream, const Attend& a) {
    if (shared > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
        if (e != cudaSuccess) return (int)e;
    }
    TvbLaunch at(dim3((unsigned)grid), dim3(THREADS), shared, stream, pdl);
    const cudaError_t e = cudaLaunchKernelEx(&at.config, kernel, a);
    return e == cudaSuccess ? tvb_last_error() : (int)e;
}

template <int D> int launch_shared(const Attend& a, const Plan& p, int dtype, int pdl, cudaStream_t s) {
    if (dtype == TVB_F32)
        return launch(attend_shared_f32_kernel<D>, p.shared_items, (size_t)(2 * KEYS32 * (D + 4) + 16 * D) * 4, pdl, s, a);
    if constexpr (D <= 128)
        if (p.tile_tokens > 0) return launch_shared_tc<D>(a, p.shared_items, p.tile_tokens, pdl, s);
    if constexpr (D == 256)
        if (p.by_sixteen) return launch_own_tma<D, true>(a, p.shared_items, pdl, s);
    return launch(attend_shared_bf16_kernel<D>, p.shared_items, Tiles<D>::bytes(64), pdl, s, a);
}
template <int D> int launch_all(const Attend& a, const Plan& p, int dtype, int pdl, cudaStream_t s) {
    int e = p.shared_items > 0 ? launch_shared<D>(a, p, dtype, pdl, s) : 0;
    if (e) return e;
    if (dtype == TVB_F32) e = launch(attend_own_f32_kernel<D>, p.own_items, (size_t)Ends<D, 4>::FLOATS * 4, pdl, s, a);
    else if (a.pages > 0 && own_tma_takes(a.page_size)) e = launch_own_tma<D, false>(a, p.own_items, pdl, s);
    else e = launch(attend_own_bf16_kernel<D>, p.own_items, OwnTiles<D>::BYTES, pdl, s, a);
    if (e || !a.part_o) return e;
    const long long joins = ceil_div((long long)a.tokens * a.num_q, WARPS);
    return dtype == TVB_F32 ? launch(join_kernel<float, D>, joins, 0, pdl, s, a) : launch(join_kernel<bf16, D>, joins, 0, pdl, s, a);
}

}  // namespace

// float32 of scratch, and the launches that a call takes in `launches`
extern "C" long long tvb_attention_shared_scratch(int tokens, int groups, int num_q, int num_kv, int head_dim, int pages, int page_size,
                                                  int max_shared, int max_own, int dtype, int* launches) {
    *launches = 0;
    if (tokens <= 0 || num_kv <= 0) return 0;
    const Plan p = plan_of(tokens, groups, num_q, num_kv, head_dim, pages, page_size, max_shared, max_own, dtype);
    *launches = p.pieces() > 1 ? 2 + (p.shared_items > 0) : 1;
    return p.pieces() > 1 ? (long long)tokens * num_q * p.pieces() * (head_dim + 2) : 0;
}

// 0, or which bounded wait gave up in some launch since the last call; reading clears it.  Synchronises.
extern "C" int tvb_attention_shared_status() {
    int value = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&value, tvb_attention_shared_status_word, sizeof(int)) != cudaSuccess) return -1;
    if (value != 0) cudaMemcpyToSymbol(tvb_attention_shared_status_word, &zero, sizeof(int));
    return value;
}

// The call's arguments as the Python side packs them.
struct SharedCall {
    const void* q;
    long long q_stride;
    const void* keys;
    const void* values;
    const int* tables;
    const int* token_row;
    const int* positions;
    const int* group_starts;
    const int* shared_lens;
    float* scratch;
    void* out;
    long long out_stride;
    int rows, width, groups, tokens, pages, page_size, num_q, num_kv, head_dim, max_shared, max_own, dtype, pdl;
    float scale;
};

extern "C" int tvb_attention_shared(const SharedCall* call, void* stream) {
    const SharedCall& c = *call;
    if (c.tokens <= 0) return 0;
    if ((c.dtype != TVB_F32 && c.dtype != TVB_BF16) || c.num_kv <= 0 || c.num_q <= 0 || c.num_q % c.num_kv || c.page_size <= 0 || c.groups < 0 ||
        c.rows < 0 || c.width < 0 || c.max_shared < 0 || c.max_own < 0 || (long long)c.width * c.page_size > 0x7fffffffLL - 4096 ||
        (long long)c.pages * c.num_kv * c.page_size > 0x7fffffffLL || (((uintptr_t)c.q | (uintptr_t)c.keys | (uintptr_t)c.values) & 15) ||
        c.q_stride * (c.dtype == TVB_F32 ? 4 : 2) % 16)
        return TVB_BAD_ARGUMENT;                // (loads of 16 bytes)
    const Plan p = plan_of(c.tokens, c.groups, c.num_q, c.num_kv, c.head_dim, c.pages, c.page_size, c.max_shared, c.max_own, c.dtype);
    if (p.shared_items > 0x7fffffffLL || p.own_items > 0x7fffffffLL || (long long)c.tokens * c.num_q * p.pieces() > 0x7fffffffLL ||
        (p.pieces() > 1 && !c.scratch))
        return TVB_BAD_ARGUMENT;
    Attend a{c.q, c.q_stride, c.keys, c.values, c.tables, c.token_row, c.positions, c.group_starts, c.shared_lens,
             p.pieces() > 1 ? c.scratch : nullptr, nullptr, c.out, c.out_stride, c.tokens, c.rows, c.width, c.groups, c.pages, c.page_size,
             c.num_q, c.num_kv, p.shared_pieces, p.own_pieces, p.own_tiles, c.scale * LOG2E};
    a.part_ml = c.scratch + (long long)c.tokens * c.num_q * p.pieces() * c.head_dim;
    cudaStream_t s = (cudaStream_t)stream;
    if (c.head_dim == 64) return launch_all<64>(a, p, c.dtype, c.pdl, s);
    if (c.head_dim == 128) return launch_all<128>(a, p, c.dtype, c.pdl, s);
    if (c.head_dim == 256) return launch_all<256>(a, p, c.dtype, c.pdl, s);
    return TVB_BAD_ARGUMENT;
}
