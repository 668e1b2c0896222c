// Low-rank adapters of many requests beside a shared projection: row t of y = x W^T becomes
//
//   y[t] + s_a (x[t] A_a^T) B_a^T        a = ids[t]; rows whose number names no adapter stay as they are
//
// with A [adapters, rank, k] and B [adapters, n, rank].  Two kernels: `shrink` makes u = s x A^T (float32 sums over k in
// pieces that the CTAs of a cluster add in order, through distributed shared memory), `expand` takes u through B and adds
// it to y.  Rows come in any order; a tile of rows goes once over every adapter that one of its rows has.
//
// bfloat16: mma.sync m16n8k16 (the products are a hundredth of the projection's: what counts is that A, B, x and y come in
// with enough of them in flight).  Few rows (see rows_go): 16 rows of one adapter a CTA, as they lie or sorted, straight into
// registers: a thread takes 16 bytes, eight neighbouring k, of each row, and which k a fragment's place stands for is permuted
// alike in both operands.  More rows go 64 a CTA through a ring in shared memory: tensor-map copies fill it where types, ranks and
// alignment allow (adapters_tma.cuh, which has its own `expand` too), else cp.async.  u leaves in two bfloat16 whose sum is u
// to 2^-16 of it, so that no rounding of u is seen beside that of a bfloat16 result.  A row takes the sums of its own adapter
// alone: what other adapters hold, infinities among them, does not reach it.
// float32: the float32 cores.
//
// Bound by the latency of their chains of loads (ids, A and x, u, B and y) for few rows: one row 1024 -> 4096 of rank 16 takes 4.4 us
// beside a projection of 2.7, 48 rows 4096 -> 6144 with 13 adapters of rank 16 10 us beside 11.5 (7 MB, 1 us at the speed of HBM).
// Bound by the traffic of x and y and the instructions between it for many: adapters_tma.cuh.  float32, 301 rows 1024 -> 2048 of
// rank 8: 8 to 10 us beside 25 to 28.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int THREADS = 128, WARPS = 4;
constexpr int MAX_RANK = 256;
constexpr int MAX_SPLITS = 8;                   // pieces of k: the CTAs of a cluster

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// values at, .., at + 7 of a row of `size` (zeros past its end, or where the row is not there) in loads of WIDTH, of which size is a
// multiple and on which the row lies; L2: past L1
template <int WIDTH, bool L2 = false> __device__ __forceinline__ uint4 load_8(const bf16* row, int at, int size, bool there) {
    if constexpr (WIDTH == 8) {
        const uint4* from = reinterpret_cast<const uint4*>(row + at);
        return !there || at >= size ? make_uint4(0, 0, 0, 0) : L2 ? __ldcg(from) : *from;
    } else if constexpr (WIDTH == 4) {
        const uint2* from = reinterpret_cast<const uint2*>(row + at);
        const uint2 lo = !there || at >= size ? make_uint2(0, 0) : L2 ? __ldcg(from) : *from;
        const uint2 hi = !there || at + 4 >= size ? make_uint2(0, 0) : L2 ? __ldcg(from + 1) : from[1];
        return make_uint4(lo.x, lo.y, hi.x, hi.y);
    } else {
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned short* from = reinterpret_cast<const unsigned short*>(row) + at + e;
            h[e] = !there || at + e >= size ? 0u : L2 ? (uint32_t)__ldcg(from) : (uint32_t)*from;
        }
        return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t* r, const bf16* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_address(p)) : "memory");
}

// What both kernels agree on: u as `hi` and `lo` rows [m][2][padded rank] (bfloat16), or [m][rank] (float32).
__device__ __forceinline__ int padded_rank(int rank) { return (rank + 15) / 16 * 16; }

// u of a row and rank: scaled, in two parts; places behind the rank are zeros.  The head of a number that bfloat16 would round to
// infinity is the largest one it has, and an infinite u has no rest (infinity - infinity).
constexpr float BF16_MOST = 3.3895313892515355e38f;
__device__ __forceinline__ void store_u(bf16* u, int row, int rank, int padded, float value) {
    const bool infinite = isinf(value);
    const bf16 hi = from_float<bf16>(infinite ? value : value > BF16_MOST ? BF16_MOST : value < -BF16_MOST ? -BF16_MOST : value);
    u[((int64_t)row * 2) * padded + rank] = hi;
    u[((int64_t)row * 2 + 1) * padded + rank] = from_float<bf16>(infinite ? 0.0f : value - to_float<bf16>(hi));
}
// Sums of products of u's two parts with a B that is infinite, or of an infinite u, hold infinity - infinity or 0 * infinity where the
// definition has infinity.  So a thread makes those of its sums that are not finite (the i-th is of column column_of(i), of which there
// are n) again from u itself and the adapter's B.
template <int COLUMNS, typename F>
__device__ __forceinline__ void mend_sums(float (&sums)[COLUMNS], const bf16* u, int padded, const bf16* b, int rank, int n, const F& column_of) {
    float zero = 0.0f;
#pragma unroll
    for (int i = 0; i < COLUMNS; ++i) zero = fmaf(sums[i], 0.0f, zero);
    if (zero == 0.0f) return;
    uint32_t again = 0;
#pragma unroll
    for (int i = 0; i < COLUMNS; ++i)
        if (column_of(i) < n && !isfinite(sums[i])) {
            again |= 1u << i;
            sums[i] = 0.0f;
        }
    if (again == 0) return;                     // (columns that are none)
#pragma unroll 1
    for (int r = 0; r < rank; ++r) {
        const float value = to_float<bf16>(u[r]) + to_float<bf16>(u[padded + r]);
#pragma unroll
        for (int i = 0; i < COLUMNS; ++i)
            if (again >> i & 1u) sums[i] = fmaf(value, to_float<bf16>(b[(int64_t)column_of(i) * rank + r]), sums[i]);
    }
}

struct Shrink {
    const bf16* x;
    int64_t ldx;
    const bf16* down;
    const int* ids;
    const float* scales;                        // [adapters] or null
    bf16* u;
    int m, k, rank, adapters;
    int splits, per_split;                      // pieces of k (CTAs of a cluster); blocks of 32 (few rows) or stages in each
};

// The adapters of a tile's rows, each once, in the order of the rows; `ids` of the rows (-1: none).  All threads call.
template <int ROWS> __device__ __forceinline__ int find_adapters(const int* all, int m, int adapters, int row0, int* ids, int* distinct) {
    static_assert(ROWS <= 64, "two warps");
    __shared__ int counts[2];
    const int tid = threadIdx.x;
    if (tid < ROWS) {
        const int id = row0 + tid < m ? __ldcg(all + row0 + tid) : -1;
        ids[tid] = (unsigned)id < (unsigned)adapters ? id : -1;
    }
    if (tid < 2) counts[tid] = 0;
    __syncthreads();
    // as a rule all rows have one
    if (__syncthreads_and(tid >= ROWS || ids[tid] == ids[0])) {
        if (tid == 0) distinct[0] = ids[0];
        __syncthreads();
        return ids[0] >= 0 ? 1 : 0;
    }
    bool first = false;
    uint32_t firsts = 0;
    if (tid < 64) {                             // whole warps
        if (tid < ROWS && ids[tid] >= 0) {
            first = true;
            for (int j = 0; j < tid; ++j) first = first && ids[j] != ids[tid];
        }
        firsts = __ballot_sync(0xffffffffu, first);
        if ((tid & 31) == 0) counts[tid >> 5] = __popc(firsts);
    }
    __syncthreads();
    if (first) distinct[(tid >= 32 ? counts[0] : 0) + __popc(firsts & ((1u << (tid & 31)) - 1u))] = ids[tid];
    __syncthreads();
    return counts[0] + counts[1];
}

// ---- few rows: 16 rows, 16 ranks and a piece of k a CTA, its warps share the piece; the CTAs of a cluster have the pieces
struct FewShared {
    float met[WARPS][16][16];
    float pieces[MAX_SPLITS][16 * 16];          // of the cluster's first CTA
};
// u of up to 16 rows of one adapter (lane group g: rows g and g + 8), 16 ranks of it; `row_of` says which row the i-th is, -1: none
// of this adapter.  The cluster's first barrier has been arrived at, and the one that ends this is left to be waited for.
template <bool WIDE, typename R> __device__ __forceinline__ void shrink_rows(const Shrink& s, int adapter, int rank0, const R& row_of, FewShared& shared) {
    constexpr int NR = 2, AHEAD = 4;            // groups of 8 ranks; blocks of 32 k in flight
    cg::cluster_group cluster = cg::this_cluster();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % s.splits, ranks = s.rank - rank0, padded = padded_rank(s.rank);
    const int end = min((s.k + 31) / 32, (split + 1) * s.per_split);
    const bf16* down = s.down + ((int64_t)adapter * s.rank + rank0) * s.k;
    const int lo_row = row_of(g), hi_row = row_of(g + 8);
    const bf16* lo = s.x + max(lo_row, 0) * s.ldx;
    const bf16* hi = s.x + max(hi_row, 0) * s.ldx;
    float sums[NR][4] = {};
    for (int b0 = split * s.per_split + warp; b0 < end; b0 += AHEAD * WARPS) {
        uint4 xl[AHEAD], xh[AHEAD], w[AHEAD][NR];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int b = b0 + i * WARPS, at = b * 32 + 8 * t;
            xl[i] = load_8<WIDE ? 8 : 1>(lo, at, s.k, lo_row >= 0 && b < end);
            xh[i] = load_8<WIDE ? 8 : 1>(hi, at, s.k, hi_row >= 0 && b < end);
#pragma unroll
            for (int j = 0; j < NR; ++j)
                w[i][j] = load_8<WIDE ? 8 : 1>(down + (int64_t)(8 * j + g) * s.k, at, s.k, 8 * j + g < ranks && b < end);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                mma_16816(sums[j], xl[i].x, xh[i].x, xl[i].y, xh[i].y, w[i][j].x, w[i][j].y);
                mma_16816(sums[j], xl[i].z, xh[i].z, xl[i].w, xh[i].w, w[i][j].z, w[i][j].w);
            }
    }
#pragma unroll
    for (int j = 0; j < NR; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) shared.met[warp][e < 2 ? g : g + 8][8 * j + 2 * t + (e & 1)] = sums[j][e];
    __syncthreads();
    cluster_wait();                             // the first CTA runs, and is through with the pieces before
    float* first_pieces = cluster.map_shared_rank(&shared.pieces[0][0], 0);
    for (int i = threadIdx.x; i < 16 * 8 * NR; i += THREADS) {
        const int row = i / (8 * NR), rank = i % (8 * NR);
        float sum = shared.met[0][row][rank];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) sum += shared.met[w][row][rank];
        first_pieces[split * 16 * 8 * NR + i] = sum;
    }
    cluster_arrive();
    cluster_wait();
    if (split == 0) {
        const float scale = s.scales ? s.scales[adapter] : 1.0f;
        for (int i = threadIdx.x; i < 16 * 8 * NR; i += THREADS) {
            const int rank = i % (8 * NR), row = row_of(i / (8 * NR));
            if (row < 0) continue;
            float sum = shared.pieces[0][i];
            for (int p = 1; p < s.splits; ++p) sum += shared.pieces[p][i];
            store_u(s.u, row, rank0 + rank, padded, rank < ranks ? sum * scale : 0.0f);
        }
    }
    cluster_arrive();
}

// The adapters of 16 rows as they lie, in the order of the rows.  A whole warp makes one.
constexpr int BARE = -1, NO_ROW = -2;           // what a row without an adapter has, and a place without a row
struct TileAdapters {
    int id;                                     // of row `lane`
    uint32_t alike, leaders;                    // lanes with the same, the first ones of each
    // with_bare: rows without an adapter count as another one
    __device__ __forceinline__ TileAdapters(const int* all, int m, int adapters, int row0, bool with_bare) {
        const int lane = threadIdx.x & 31;
        id = NO_ROW;
        if (lane < 16 && row0 + lane < m) {
            id = __ldcg(all + row0 + lane);
            if ((unsigned)id >= (unsigned)adapters) id = BARE;
        }
        alike = __match_any_sync(0xffffffffu, id);
        leaders = __ballot_sync(0xffffffffu, id >= (with_bare ? BARE : 0) && (alike & ((1u << lane) - 1u)) == 0);
    }
    __device__ __forceinline__ void pass(int n) {
        for (; n > 0; --n) leaders &= leaders - 1;
    }
    // the next one's number (NO_ROW: there is none), and which of the rows have it
    __device__ __forceinline__ int next(uint32_t& rows) const {
        const int leader = leaders ? __ffs(leaders) - 1 : 31;
        rows = __shfl_sync(0xffffffffu, alike, leader);
        return __shfl_sync(0xffffffffu, id, leader);
    }
};

// rows as they lie, the blockIdx.z-th of their adapters
template <bool WIDE> __global__ void __launch_bounds__(THREADS) shrink_few_kernel(Shrink s) {
    __shared__ FewShared shared;
    cluster_arrive_relaxed();
    const int rank0 = blockIdx.x / s.splits * 16, row0 = blockIdx.y * 16;
    pdl_wait();
    pdl_launch_dependents();
    TileAdapters tile(s.ids, s.m, s.adapters, row0, false);
    tile.pass(blockIdx.z);
    uint32_t rows;
    const int adapter = tile.next(rows);
    if (adapter >= 0)                           // the same for the whole cluster
        shrink_rows<WIDE>(s, adapter, rank0, [&](int i) { return rows >> i & 1 ? row0 + i : -1; }, shared);
    cluster_wait();
}

// ---- some more rows, and more than a few adapters: chunks of up to 16 rows with one adapter
//
// The rows of a decode step come in any order (as its requests were admitted).  Every CTA sorts them by their adapters for itself,
// in shared memory, and takes chunks of rows that share one, so that an adapter is read once for 16 of them however they lie.
// Adapters come in the order of their first rows, and their rows as they lie, so that all CTAs agree.
constexpr int MAX_SORTED_ROWS = 512, TABLE = 2 * MAX_SORTED_ROWS, SORTED_BLOCKS = MAX_SORTED_ROWS / 32;
static_assert(SORTED_BLOCKS == 16 && TABLE == 1 << 10, "a byte of a uint4 a block of 32 rows, 10 bits of a hash");
struct Sorted {
    uint4 counts[TABLE];                        // rows of a hashed adapter in every block of 32 rows, a byte each
    int keys[TABLE];                            // the adapter, -1: none; then its first chunk and, << 16, place
    int of_rows[MAX_SORTED_ROWS];               // a row's adapter, -1: none
    int slots[MAX_SORTED_ROWS];                 // a row's place in the table, and how many rows before have its adapter << 16
    int sums[SORTED_BLOCKS];
    int ids[MAX_SORTED_ROWS];                   // a chunk's adapter
    int starts[MAX_SORTED_ROWS];                // its place among the sorted rows, and how many they are << 16
    unsigned short rows[MAX_SORTED_ROWS];       // sorted
    __device__ __forceinline__ int row(int chunk, int i) const { return i < starts[chunk] >> 16 ? rows[(starts[chunk] & 0xffff) + i] : -1; }
};
// How many chunks there are; with_bare: rows without an adapter have number `adapters`.  All threads call.  (Loops as they are: code that
// runs once is read as slowly as it is long.)
__device__ __forceinline__ int sort_rows(const int* all, int m, int adapters, bool with_bare, Sorted& c) {
    const int tid = threadIdx.x, lane = tid & 31, padded = (m + 31) / 32 * 32;
    const uint32_t lower = (1u << lane) - 1u;
#pragma unroll 1
    for (int row = tid; row < padded; row += THREADS) {
        const int id = row < m ? __ldcg(all + row) : -1;
        c.of_rows[row] = row < m && (unsigned)id >= (unsigned)adapters && with_bare ? adapters : (unsigned)id < (unsigned)adapters ? id : -1;
    }
#pragma unroll 1
    for (int i = tid; i < TABLE; i += THREADS) {
        c.keys[i] = -1;
        c.counts[i] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
#pragma unroll 1
    for (int row = tid; row < padded; row += THREADS) {                         // (whole warps)
        const int id = c.of_rows[row];
        const uint32_t alike = __match_any_sync(0xffffffffu, id);
        const int rank = __popc(alike & lower);
        int at = (int)((uint32_t)id * 0x9e3779b1u >> 22);
        if (id >= 0 && rank == 0) {
            for (;;) {                          // half of the table at least stays empty
                const int held = atomicCAS(c.keys + at, -1, id);
                if (held == -1 || held == id) break;
                at = (at + 1) & (TABLE - 1);
            }
            reinterpret_cast<unsigned char*>(c.counts + at)[row / 32] = (unsigned char)__popc(alike);
        }
        c.slots[row] = __shfl_sync(0xffffffffu, at, __ffs(alike) - 1) | rank << 16;
    }
    __syncthreads();
    // rows and chunks of the adapters that begin at a row, added up over the rows
#pragma unroll 1
    for (int row = tid; row < padded; row += THREADS) {
        const int block = row / 32, slot = c.slots[row] & 0xffff;
        int sum = 0;
        if (c.of_rows[row] >= 0) {
            const uint4 of = c.counts[slot];
            const uint32_t words[4] = {of.x, of.y, of.z, of.w};
            uint32_t before = 0, total = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int bytes = block - 4 * w;
                total = __dp4a(words[w], 0x01010101u, total);
                before = __dp4a(bytes >= 4 ? words[w] : bytes <= 0 ? 0u : words[w] & ((1u << (8 * bytes)) - 1u), 0x01010101u, before);
            }
            const int rank = (c.slots[row] >> 16) + before;
            c.slots[row] = slot | rank << 16;
            if (rank == 0) sum = (total + 15) / 16 | total << 16;
        }
        const int own = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += other;
        }
        if (own) c.keys[slot] = sum - own;      // (behind the sums of the blocks before)
        if (lane == 31) c.sums[block] = sum;
    }
    __syncthreads();
    int upto = 0;
#pragma unroll 1
    for (int block = 0; block < padded / 32; ++block) {
        const int row = block * 32 + lane;
        if (block % WARPS == tid / 32 && c.of_rows[row] >= 0 && c.slots[row] >> 16 == 0) c.keys[c.slots[row]] += upto;
        upto += c.sums[block];
    }
    __syncthreads();
#pragma unroll 1
    for (int row = tid; row < padded; row += THREADS) {
        const int id = c.of_rows[row];
        if (id < 0) continue;
        const int slot = c.slots[row] & 0xffff, rank = c.slots[row] >> 16, at = c.keys[slot], place = (at >> 16) + rank;
        c.rows[place] = (unsigned short)row;
        if (rank % 16 == 0) {
            const uint4 of = c.counts[slot];
            const int total = __dp4a(of.x, 0x01010101u, __dp4a(of.y, 0x01010101u, __dp4a(of.z, 0x01010101u, __dp4a(of.w, 0x01010101u, 0u))));
            c.ids[(at & 0xffff) + rank / 16] = id;
            c.starts[(at & 0xffff) + rank / 16] = place | min(16, total - rank) << 16;
        }
    }
    __syncthreads();
    return upto & 0xffff;
}

template <bool WIDE> __global__ void __launch_bounds__(THREADS) shrink_sorted_kernel(Shrink s) {
    __shared__ FewShared shared;
    __shared__ Sorted sorted;
    cluster_arrive_relaxed();
    const int rank_chunks = (s.rank + 15) / 16;
    pdl_wait();
    pdl_launch_dependents();
    const int items = sort_rows(s.ids, s.m, s.adapters, false, sorted) * rank_chunks;
    for (int item = blockIdx.x / s.splits; item < items; item += gridDim.x / s.splits) {          // the same for the whole cluster
        const int chunk = item / rank_chunks;
        shrink_rows<WIDE>(s, sorted.ids[chunk], item % rank_chunks * 16, [&](int i) { return sorted.row(chunk, i); }, shared);
    }
    cluster_wait();
}

// ---- more rows: 64 rows and RANKS ranks a CTA, 16 rows a warp; stages of 64 k
constexpr int STAGE_K = 64, STAGES = 4, STAGE_PITCH = STAGE_K + 8;
template <int RANKS> struct ManyShared {
    static constexpr int STAGE = (64 + RANKS) * STAGE_PITCH;                    // elements
    static constexpr int SUM_PITCH = RANKS + 4;
    static constexpr int RING_BYTES = STAGES * STAGE * 2, SUM_BYTES = 64 * SUM_PITCH * 4;
    static constexpr int BYTES = RING_BYTES > SUM_BYTES ? RING_BYTES : SUM_BYTES;
};
template <int RANKS, bool WIDE>
__global__ void __launch_bounds__(THREADS) shrink_many_kernel(Shrink s) {
    using Shared = ManyShared<RANKS>;
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ int ids[64], distinct[64];
    bf16* ring = reinterpret_cast<bf16*>(raw);
    float* sums_s = reinterpret_cast<float*>(raw);                              // [64][SUM_PITCH], over the ring
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % s.splits, rank0 = blockIdx.x / s.splits * RANKS, ranks = min(RANKS, s.rank - rank0);
    const int row0 = blockIdx.y * 64, padded = padded_rank(s.rank);
    const int first = split * s.per_split, stages = max(0, min((s.k + STAGE_K - 1) / STAGE_K, first + s.per_split) - first);
    pdl_wait();
    pdl_launch_dependents();
    const int count = find_adapters<64>(s.ids, s.m, s.adapters, row0, ids, distinct);
    for (int d = blockIdx.z; d < count; d += gridDim.z) {                       // the same for the whole cluster
        const int adapter = distinct[d];
        const bf16* down = s.down + ((int64_t)adapter * s.rank + rank0) * s.k;
        auto load = [&](int stage) {
            if (stage < stages) {
                bf16* x_s = ring + stage % STAGES * Shared::STAGE;
                bf16* a_s = x_s + 64 * STAGE_PITCH;
                const int k0 = (first + stage) * STAGE_K;
                for (int i = tid; i < (64 + RANKS) * (STAGE_K / 8); i += THREADS) {
                    const int row = i / (STAGE_K / 8), at = k0 + i % (STAGE_K / 8) * 8;
                    const bool of_x = row < 64;
                    const bool there = of_x ? ids[row] == adapter : row - 64 < ranks;
                    const bf16* from = of_x ? s.x + (int64_t)(there ? row0 + row : 0) * s.ldx : down + (int64_t)(there ? row - 64 : 0) * s.k;
                    bf16* to = (of_x ? x_s + row * STAGE_PITCH : a_s + (row - 64) * STAGE_PITCH) + i % (STAGE_K / 8) * 8;
                    if constexpr (WIDE) cp_async_16(to, from + (at < s.k ? at : 0), there && at < s.k);
                    else *reinterpret_cast<uint4*>(to) = load_8<1>(from, at, s.k, there);
                }
            }
            cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) load(i);
        float sums[RANKS / 8][4] = {};
        for (int stage = 0; stage < stages; ++stage) {
            cp_async_wait<STAGES - 2>();
            __syncthreads();                    // the stage is there, and the one that the next load overwrites is through
            load(stage + STAGES - 1);
            const bf16* x_s = ring + stage % STAGES * Shared::STAGE + (warp * 16 + (lane & 15)) * STAGE_PITCH + (lane >> 4) * 8;
            const bf16* a_s = ring + stage % STAGES * Shared::STAGE + 64 * STAGE_PITCH;
#pragma unroll
            for (int kk = 0; kk < STAGE_K / 16; ++kk) {
                uint32_t a[4];
                ldmatrix_x4(a, x_s + kk * 16);
#pragma unroll
                for (int j = 0; j < RANKS / 16; ++j) {
                    uint32_t b[4];
                    const int matrix = lane >> 3;
                    ldmatrix_x4(b, a_s + (j * 16 + (matrix >> 1) * 8 + (lane & 7)) * STAGE_PITCH + kk * 16 + (matrix & 1) * 8);
                    mma_16816(sums[2 * j], a[0], a[1], a[2], a[3], b[0], b[1]);
                    mma_16816(sums[2 * j + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
                }
            }
        }
        cp_async_wait<0>();
        __syncthreads();
#pragma unroll
        for (int j = 0; j < RANKS / 8; ++j)
#pragma unroll
            for (int half = 0; half < 2; ++half)
                *reinterpret_cast<float2*>(sums_s + (warp * 16 + g + 8 * half) * Shared::SUM_PITCH + 8 * j + 2 * t) =
                    make_float2(sums[j][2 * half], sums[j][2 * half + 1]);
        cluster_arrive();
        cluster_wait();
        // a CTA adds the pieces of its share of the rows
        const float scale = s.scales ? s.scales[adapter] : 1.0f;
        const int share = 64 / s.splits;
        for (int i = tid; i < share * RANKS; i += THREADS) {
            const int row = split * share + i / RANKS, rank = i % RANKS;
            if (ids[row] != adapter || rank0 + rank >= padded) continue;
            float piece[MAX_SPLITS];
#pragma unroll
            for (int p = 0; p < MAX_SPLITS; ++p)
                piece[p] = p < s.splits ? cluster.map_shared_rank(sums_s, p)[row * Shared::SUM_PITCH + rank] : 0.0f;
            float sum = piece[0];
#pragma unroll
            for (int p = 1; p < MAX_SPLITS; ++p) sum += piece[p];
            store_u(s.u, row0 + row, rank0 + rank, padded, rank < ranks ? sum * scale : 0.0f);
        }
        cluster_arrive();                       // nobody reads these sums any more
        cluster_wait();
    }
}

struct Expand {
    const void* u;
    const void* up;                             // [adapters, n, rank]
    const int* ids;
    const void* y;
    int64_t ldy;
    void* out;                                  // y itself where their types are the same
    int64_t ldo;
    int m, n, rank, adapters;
};

// A warp has 16 rows of y with one adapter and walks over tiles of 32 columns: the rows' u stays in registers, y and B of the next tile
// are asked for before this one's products.  A thread takes 16 bytes, eight neighbouring ranks, of a row of B and of u (which rank
// a fragment's place stands for is permuted alike in both).  The columns of an n-tile are spread so that a thread holds eight
// neighbours of y: place c of tile j is column (c / 2) * 8 + 2 j + c % 2.
//
// All that comes from before `shrink` (whose threads wait for it before they let this kernel start) may be read before `shrink` is
// through: ids, and where EARLY says so the first tiles of y and B, past L1.  u may not, and nothing is written before.
// B is read in loads of WIDTH, and a tile of y in 16-byte words where WIDE.  O is Y, and y becomes the result; or y is float32, the
// result bfloat16 elsewhere, and rows without an adapter (BARE) are rounded into it too.
template <typename Y, typename O, int WIDTH, bool WIDE, bool EARLY>
__device__ __forceinline__ void expand_rows(const Expand& s, int adapter, const int (&row)[2], const bool (&there)[2], int first_tile, int end, int step) {
    constexpr int NT = 4, STEPS = 2, WORDS = sizeof(Y) / 2;                     // steps of 32 ranks held; 16-byte words of eight values of y
    const int padded = padded_rank(s.rank), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const bool has = adapter >= 0;
    const bf16* b = reinterpret_cast<const bf16*>(s.up) + (int64_t)max(adapter, 0) * s.n * s.rank;
    const bf16* u[2];
    const Y* y[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        u[h] = reinterpret_cast<const bf16*>(s.u) + (int64_t)row[h] * 2 * padded;
        y[h] = reinterpret_cast<const Y*>(s.y) + row[h] * s.ldy + 8 * t;
    }
    uint4 held[STEPS][2][2];                    // u of rows g + 8 h, its heads and its rests
    auto load_u = [&](int r0) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int at = r0 + 32 * k + 8 * t;
                    held[k][h][q] = has && there[h] && at < padded ? *reinterpret_cast<const uint4*>(u[h] + q * padded + at) : make_uint4(0, 0, 0, 0);
                }
    };
    uint4 old[2][WORDS];                        // of y
    auto load_y = [&](int tile) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (!there[h]) continue;
            const Y* from = y[h] + tile * 32;
            const int left = s.n - tile * 32 - 8 * t;
            if (WIDE && left >= 8) {
#pragma unroll
                for (int q = 0; q < WORDS; ++q) old[h][q] = __ldcg(reinterpret_cast<const uint4*>(from) + q);
            } else if constexpr (sizeof(Y) == 2) {
                uint32_t v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = e < left ? (uint32_t)__ldcg(reinterpret_cast<const unsigned short*>(from) + e) : 0u;
                old[h][0] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
            } else {
                uint32_t v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = e < left ? __ldcg(reinterpret_cast<const uint32_t*>(from) + e) : 0u;
                old[h][0] = make_uint4(v[0], v[1], v[2], v[3]);
                old[h][WORDS - 1] = make_uint4(v[4], v[5], v[6], v[7]);
            }
        }
    };
    uint4 w[STEPS][NT];
    auto load_b = [&](int tile, int r0) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int at = tile * 32 + (g >> 1) * 8 + 2 * j + (g & 1);
                w[k][j] = load_8<WIDTH, EARLY>(b + (int64_t)at * s.rank, r0 + 32 * k + 8 * t, s.rank, has && at < s.n);
            }
    };
    load_y(first_tile);
    load_b(first_tile, 0);
    if (EARLY) {
        pdl_wait();
        pdl_launch_dependents();
    }
    load_u(0);
    for (int tile = first_tile; tile < end; tile += step) {
        float sums[NT][4] = {};
        for (int r0 = 0; r0 < padded; r0 += 32 * STEPS) {
            if (padded > 32 * STEPS && (r0 > 0 || tile != first_tile)) {
                load_u(r0);
                if (r0 > 0) load_b(tile, r0);
            }
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                if (r0 + 32 * k >= padded) break;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const uint4 &lo = held[k][0][q], &hi = held[k][1][q];
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        mma_16816(sums[j], lo.x, hi.x, lo.y, hi.y, w[k][j].x, w[k][j].y);
                        mma_16816(sums[j], lo.z, hi.z, lo.w, hi.w, w[k][j].z, w[k][j].w);
                    }
                }
            }
        }
        uint4 now[2][WORDS];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < WORDS; ++q) now[h][q] = old[h][q];
        if (tile + step < end) {
            load_y(tile + step);
            load_b(tile + step, 0);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (!there[h]) continue;
            O* to = reinterpret_cast<O*>(s.out) + row[h] * s.ldo + 8 * t + tile * 32;
            float add[8];
#pragma unroll
            for (int j = 0; j < NT; ++j) { add[2 * j] = sums[j][2 * h]; add[2 * j + 1] = sums[j][2 * h + 1]; }
            mend_sums(add, u[h], padded, b, s.rank, s.n, [&](int i) { return tile * 32 + 8 * t + i; });
            float v[8];
            if constexpr (sizeof(Y) == 2) {
                unpack_bf16x8(now[h][0], v);
            } else {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const uint4 word = now[h][q];
                    v[4 * q] = __uint_as_float(word.x); v[4 * q + 1] = __uint_as_float(word.y);
                    v[4 * q + 2] = __uint_as_float(word.z); v[4 * q + 3] = __uint_as_float(word.w);
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) add[e] += v[e];
            const int left = s.n - tile * 32 - 8 * t;
            if (WIDE && left >= 8) {
                if constexpr (sizeof(O) == 2) {
                    *reinterpret_cast<uint4*>(to) = pack_bf16x8(add);
                } else {
#pragma unroll
                    for (int q = 0; q < 2; ++q)
                        reinterpret_cast<float4*>(to)[q] = make_float4(add[4 * q], add[4 * q + 1], add[4 * q + 2], add[4 * q + 3]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < left) to[e] = from_float<O>(add[e]);
            }
        }
    }
}

// few rows: 16 rows as they lie, the blockIdx.z-th of their adapters, a tile of 32 columns a warp
template <typename Y, typename O, int WIDTH, bool WIDE>
__global__ void __launch_bounds__(THREADS, 4) expand_few_kernel(Expand s) {
    const int tile = blockIdx.x * WARPS + (threadIdx.x >> 5), row0 = blockIdx.y * 16, g = (threadIdx.x & 31) >> 2;
    TileAdapters of_tile(s.ids, s.m, s.adapters, row0, sizeof(Y) != sizeof(O));
    of_tile.pass(blockIdx.z);
    uint32_t rows;
    const int adapter = of_tile.next(rows);
    if (adapter != NO_ROW && tile * 32 < s.n && (sizeof(Y) != sizeof(O) || adapter >= 0)) {
        const bool there[2] = {(bool)(rows >> g & 1), (bool)(rows >> (g + 8) & 1)};
        const int row[2] = {there[0] ? row0 + g : 0, there[1] ? row0 + g + 8 : 0};
        expand_rows<Y, O, WIDTH, WIDE, true>(s, adapter, row, there, tile, tile + 1, 1);
    } else {
        pdl_wait();                             // (a warp that has nothing to do waits too: what follows relies on this kernel's end)
        pdl_launch_dependents();
    }
}

// rows sorted into chunks: a chunk and a strip of its columns a CTA, as many strips as fill the GPU; the warps take every fourth tile
// of the strip
template <typename Y, typename O, int WIDTH, bool WIDE>
__global__ void __launch_bounds__(THREADS, 4) expand_sorted_kernel(Expand s) {
    __shared__ Sorted sorted;
    const int warp = threadIdx.x >> 5, g = (threadIdx.x & 31) >> 2, tiles = (s.n + 31) / 32;
    const int count = sort_rows(s.ids, s.m, s.adapters, sizeof(Y) != sizeof(O), sorted);
    const int strips = max(1, min((tiles + WARPS - 1) / WARPS, (int)gridDim.x / max(count, 1))), per = (tiles + strips - 1) / strips;
    for (int item = blockIdx.x; item < count * strips; item += gridDim.x) {
        const int chunk = item % count, first = item / count * per + warp, end = min(tiles, (item / count + 1) * per);
        int row[2] = {sorted.row(chunk, g), sorted.row(chunk, g + 8)};
        const bool there[2] = {row[0] >= 0, row[1] >= 0};
        row[0] = max(row[0], 0);
        row[1] = max(row[1], 0);
        const int adapter = sorted.ids[chunk] < s.adapters ? sorted.ids[chunk] : BARE;
        if (first < end) expand_rows<Y, O, WIDTH, WIDE, true>(s, adapter, row, there, first, end, WARPS);
    }
    pdl_wait();                                 // (see above)
    pdl_launch_dependents();
}

// more rows: the warps of a CTA have 16 rows each as they lie and the same columns, whose B they find in L1; one adapter of the rows
// after another
template <typename Y, typename O, int WIDTH, bool WIDE>
__global__ void __launch_bounds__(THREADS, 4) expand_many_kernel(Expand s) {
    constexpr int ROWS = 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    const int row0 = (blockIdx.y * WARPS + warp) * ROWS, tiles = (s.n + 31) / 32;
    TileAdapters of_tile(s.ids, s.m, s.adapters, row0, sizeof(Y) != sizeof(O));
    of_tile.pass(blockIdx.z);
    pdl_wait();
    pdl_launch_dependents();
    for (; of_tile.leaders; of_tile.pass(gridDim.z)) {
        uint32_t rows;
        const int adapter = of_tile.next(rows);
        const bool there[2] = {(bool)(rows >> g & 1), (bool)(rows >> (g + 8) & 1)};
        const int row[2] = {there[0] ? row0 + g : 0, there[1] ? row0 + g + 8 : 0};
        expand_rows<Y, O, WIDTH, WIDE, false>(s, adapter, row, there, blockIdx.x, tiles, gridDim.x);
    }
}

// ---- float32: a warp makes four ranks of a row over its piece of k
struct Shrink32 {
    const float* x;
    int64_t ldx;
    const float* down;
    const int* ids;
    const float* scales;
    float* u;                                   // [m, rank]
    int m, k, rank, adapters, splits, per_split;
};
template <int VEC> __global__ void __launch_bounds__(THREADS) shrink_f32_kernel(Shrink32 s) {
    __shared__ float pieces[MAX_SPLITS][WARPS][4];                              // of the cluster's first CTA
    cg::cluster_group cluster = cg::this_cluster();
    cluster_arrive_relaxed();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_row = s.splits * ((s.rank + 4 * WARPS - 1) / (4 * WARPS)), place = blockIdx.x % per_row;
    const int row = blockIdx.x / per_row, split = place % s.splits, rank0 = (place / s.splits * WARPS + warp) * 4;
    pdl_wait();
    pdl_launch_dependents();
    const int id = s.ids[row];
    const bool any = (unsigned)id < (unsigned)s.adapters;                       // the same for the whole cluster
    float sums[4] = {};
    if (any && rank0 < s.rank) {
        const float* x = s.x + (int64_t)row * s.ldx;
        const float* down = s.down + ((int64_t)id * s.rank + rank0) * s.k;
        const int end = min(s.k, (split + 1) * s.per_split);
#pragma unroll 2
        for (int at = split * s.per_split + lane * VEC; at < end; at += 32 * VEC) {
            float v[VEC], w[4][VEC];
            load_values<VEC>(x + at, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) load_values<VEC>(down + (int64_t)(rank0 + j < s.rank ? j : 0) * s.k + at, w[j]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) sums[j] = fmaf(v[e], w[j][e], sums[j]);
        }
    }
    cluster_wait();                             // the first CTA runs
    float* first_pieces = cluster.map_shared_rank(&pieces[0][0][0], 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float sum = warp_sum(sums[j]);
        if (lane == j) first_pieces[(split * WARPS + warp) * 4 + j] = sum;
    }
    cluster_arrive();
    cluster_wait();
    if (split != 0 || !any || lane >= 4 || rank0 + lane >= s.rank) return;
    float sum = pieces[0][warp][lane];
    for (int p = 1; p < s.splits; ++p) sum += pieces[p][warp][lane];
    s.u[(int64_t)row * s.rank + rank0 + lane] = s.scales ? sum * s.scales[id] : sum;
}

// a thread makes one column of 16 rows
template <int VEC> __global__ void __launch_bounds__(THREADS) expand_f32_kernel(Expand s) {
    constexpr int ROWS = 16;
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ int ids[ROWS], distinct[ROWS];
    float* u = reinterpret_cast<float*>(raw);                                   // [ROWS][rank]
    const int row0 = blockIdx.y * ROWS, rows = min(ROWS, s.m - row0), column = blockIdx.x * THREADS + threadIdx.x;
    // before `shrink` is through (see expand_rows): the adapters, y, and B on its way into L2
    const int count = find_adapters<ROWS>(s.ids, s.m, s.adapters, row0, ids, distinct);
    float* y = reinterpret_cast<float*>(s.out) + (int64_t)row0 * s.ldo + column;
    float old[ROWS];
#pragma unroll
    for (int row = 0; row < ROWS; ++row) old[row] = column < s.n && ids[row] >= 0 ? __ldcg(y + row * s.ldo) : 0.0f;
    if (column < s.n)
        for (int d = 0; d < count; ++d)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const float*>(s.up) + ((int64_t)distinct[d] * s.n + column) * s.rank));
    pdl_wait();
    pdl_launch_dependents();
    for (int i = threadIdx.x; i < rows * s.rank; i += THREADS) u[i] = reinterpret_cast<const float*>(s.u)[(int64_t)row0 * s.rank + i];
    __syncthreads();
    if (column >= s.n) return;
    for (int d = 0; d < count; ++d) {
        const int adapter = distinct[d];
        const float* b = reinterpret_cast<const float*>(s.up) + ((int64_t)adapter * s.n + column) * s.rank;
        float total[ROWS] = {};
#pragma unroll 2
        for (int r = 0; r < s.rank; r += VEC) {
            float w[VEC];
            load_values<VEC>(b + r, w);
#pragma unroll
            for (int row = 0; row < ROWS; ++row)
                if (ids[row] == adapter)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) total[row] = fmaf(u[row * s.rank + r + e], w[e], total[row]);
        }
#pragma unroll
        for (int row = 0; row < ROWS; ++row)
            if (ids[row] == adapter) y[row * s.ldo] = old[row] + total[row];
    }
}

#include "adapters_tma.cuh"

// ------------------------------------------------------------------ host side
// How the rows go: 16 as they lie, sorted by their adapters, or 64 as they lie.  Where there are few adapters, or few rows, the ones a
// tile meets are read side by side quickly enough; sorting costs 2 us for 48 rows, 8 for 512.  Measured (4096 -> 4096, rank 16, us FEW /
// SORTED / MANY): 32 adapters in random order, 48 rows 9.0 / 10.2 / 70, 96 rows 13.4 / 11.2 / 76, 256 rows 33 / 14.7 / 79, 512 rows
// 60 / 22.7 / 102; one after another, 48 rows 8.2 / 10.6 / 80, 96 rows 10.0 / 10.8 / 57, 256 rows 15.0 / 13.5 / 23, 512 rows 24.7 /
// 18.7 / 18.3; 4 adapters in random order, 192 rows 9.8 / 10.4 / 14.4, 256 rows 11.4 / 12.4 / 14.7, 512 rows 21.3 / 19.2 / 19.5; one
// after another, 192 rows 6.6 / 10.3 / 8.9, 256 rows 7.4 / 11.9 / 7.5, 512 rows 10.9 / 18.6 / 8.3.
enum Rows { FEW, SORTED, MANY };
Rows rows_go(int m, int adapters) { return adapters > 8 && m >= 96 && m <= MAX_SORTED_ROWS ? SORTED : m <= 192 ? FEW : MANY; }

int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <typename K, typename S> int launch(K kernel, dim3 grid, size_t shared, int cluster, int pdl, cudaStream_t stream, const S& s) {
    if (shared > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
        if (e != cudaSuccess) return (int)e;
    }
    TvbLaunch at(grid, dim3(THREADS), shared, stream, pdl, cluster);
    const cudaError_t e = cudaLaunchKernelEx(&at.config, kernel, s);
    return e == cudaSuccess ? tvb_last_error() : (int)e;
}

template <int RANKS> int launch_many(const Shrink& a, int chunks, bool wide, int pdl, cudaStream_t s) {
    const dim3 grid(a.splits * chunks, ceil_div(a.m, 64), min(2, a.adapters));
    return wide ? launch(shrink_many_kernel<RANKS, true>, grid, ManyShared<RANKS>::BYTES, a.splits, pdl, s, a)
                : launch(shrink_many_kernel<RANKS, false>, grid, ManyShared<RANKS>::BYTES, a.splits, pdl, s, a);
}

template <typename Y, typename O, int WIDTH, bool WIDE> int launch_expand(const Expand& a, Rows rows_are, int pdl, cudaStream_t s) {
    const int tiles = ceil_div(a.n, 32), each = min(a.adapters, 16) + (sizeof(Y) != sizeof(O));   // (what 16 rows have, at most)
    if (rows_are == FEW)
        return launch(expand_few_kernel<Y, O, WIDTH, WIDE>, dim3(ceil_div(tiles, WARPS), ceil_div(a.m, 16), min(min(16, a.m), each)), 0, 0, pdl, s, a);
    if (rows_are == SORTED)                     // one round of CTAs, four an SM
        return launch(expand_sorted_kernel<Y, O, WIDTH, WIDE>, dim3((unsigned)min((long long)a.m * ceil_div(tiles, WARPS), 4ll * 148)), 0, 0, pdl, s, a);
    // several rounds of CTAs, which walk over the columns (4,099 rows x 4,096 of rank 64: 41 us with three CTAs an SM, 34 with six, 33 with twelve)
    const int rows = ceil_div(a.m, 16 * WARPS);
    return launch(expand_many_kernel<Y, O, WIDTH, WIDE>, dim3(min(tiles, max(1, 12 * 148 / rows)), rows, min(2, each)), 0, 0, pdl, s, a);
}
// by how B and y lie
template <typename Y, typename O> int launch_expand(const Expand& a, Rows rows_are, int pdl, cudaStream_t s) {
    const uintptr_t up = (uintptr_t)a.up, y = (uintptr_t)a.y;
    if (a.rank % 8 == 0 && !(up & 15)) {
        if constexpr (sizeof(Y) == sizeof(O))
            if (!(y & 15) && a.ldy * sizeof(Y) % 16 == 0) return launch_expand<Y, O, 8, true>(a, rows_are, pdl, s);
        return launch_expand<Y, O, 8, false>(a, rows_are, pdl, s);
    }
    return a.rank % 4 == 0 && !(up & 7) ? launch_expand<Y, O, 4, false>(a, rows_are, pdl, s) : launch_expand<Y, O, 1, false>(a, rows_are, pdl, s);
}

}  // namespace

namespace {

int shrink(const void* x, long long ldx, const void* down, const int* ids, const float* scales, void* u, int m, int k, int rank,
           int adapters, int dtype, int pdl, cudaStream_t s) {
    if (dtype == TVB_F32) {
        const bool wide = k % 4 == 0 && ldx % 4 == 0 && !(((uintptr_t)x | (uintptr_t)down) & 15);
        // pieces of at least 512 k, and not more CTAs than eight an SM
        const int chunks = ceil_div(rank, 4 * WARPS);
        int splits = 1;
        while (splits < MAX_SPLITS && k / splits >= 1024 && (long long)m * chunks * splits < 8 * 148) splits *= 2;
        const long long ctas = (long long)m * splits * chunks;
        if (ctas > 0x7fffffffLL) return TVB_BAD_ARGUMENT;
        const Shrink32 a{(const float*)x, ldx, (const float*)down, ids, scales, (float*)u, m, k, rank, adapters, splits,
                         ceil_div(ceil_div(k, splits), 4) * 4};
        const dim3 grid((unsigned)ctas);
        return wide ? launch(shrink_f32_kernel<4>, grid, 0, splits, pdl, s, a) : launch(shrink_f32_kernel<1>, grid, 0, splits, pdl, s, a);
    }
    if (dtype != TVB_BF16) return TVB_BAD_ARGUMENT;
    const bool wide = k % 8 == 0 && ldx % 8 == 0 && !(((uintptr_t)x | (uintptr_t)down) & 15);
    Shrink a{(const bf16*)x, ldx, (const bf16*)down, ids, scales, (bf16*)u, m, k, rank, adapters, 1, 0};
    const Rows rows_are = rows_go(m, adapters);
    if (rows_are != MANY) {
        // a warp keeps a block of 32 k at least
        while (a.splits < MAX_SPLITS && a.splits * 2 * WARPS <= ceil_div(k, 32)) a.splits *= 2;
        a.per_split = ceil_div(ceil_div(k, 32), a.splits);
        const int chunks = ceil_div(rank, 16);
        if (rows_are == FEW) {
            const dim3 grid(a.splits * chunks, ceil_div(m, 16), min(min(16, m), adapters));
            return wide ? launch(shrink_few_kernel<true>, grid, 0, a.splits, pdl, s, a) : launch(shrink_few_kernel<false>, grid, 0, a.splits, pdl, s, a);
        }
        const dim3 grid(a.splits * (unsigned)min((long long)m * chunks, 4ll * 148 / a.splits));   // one round of clusters
        return wide ? launch(shrink_sorted_kernel<true>, grid, 0, a.splits, pdl, s, a) : launch(shrink_sorted_kernel<false>, grid, 0, a.splits, pdl, s, a);
    }
    // pieces of k while the CTAs still have one round on the GPU (three an SM)
    const int chunks = rank <= 16 ? 1 : ceil_div(rank, 64), stages = ceil_div(k, STAGE_K);
    while (a.splits < MAX_SPLITS && a.splits * 4 <= stages && (long long)ceil_div(m, 64) * chunks * a.splits * 2 <= 3 * 148) a.splits *= 2;
    a.per_split = ceil_div(stages, a.splits);
    return rank <= 16 ? launch_many<16>(a, chunks, wide, pdl, s) : launch_many<64>(a, chunks, wide, pdl, s);
}

// dtype: of x, A and B; y_dtype and out_dtype: both float32, both bfloat16 with bfloat16, or float32 and bfloat16 with it
int expand(const Expand& a, int dtype, int y_dtype, int out_dtype, int pdl, cudaStream_t s) {
    if (dtype == TVB_F32) {
        if (y_dtype != TVB_F32 || out_dtype != TVB_F32) return TVB_BAD_ARGUMENT;
        const dim3 grid(ceil_div(a.n, THREADS), ceil_div(a.m, 16));
        const size_t shared = 16 * (size_t)a.rank * 4;
        return a.rank % 4 == 0 && !((uintptr_t)a.up & 15) ? launch(expand_f32_kernel<4>, grid, shared, 0, pdl, s, a)
                                                         : launch(expand_f32_kernel<1>, grid, shared, 0, pdl, s, a);
    }
    if (dtype != TVB_BF16) return TVB_BAD_ARGUMENT;
    const Rows rows_are = rows_go(a.m, a.adapters);
    if (y_dtype == TVB_BF16 && out_dtype == TVB_BF16) return launch_expand<bf16, bf16>(a, rows_are, pdl, s);
    if (y_dtype != TVB_F32) return TVB_BAD_ARGUMENT;
    if (out_dtype == TVB_F32) return launch_expand<float, float>(a, rows_are, pdl, s);
    return out_dtype == TVB_BF16 ? launch_expand<float, bf16>(a, rows_are, pdl, s) : TVB_BAD_ARGUMENT;
}

}  // namespace

// The call's arguments as the Python side packs them.
struct AdaptersCall {
    const void* x;
    long long ldx;
    const void* down;
    const void* up;
    const int* ids;
    const float* scales;
    void* u;                                    // scratch: m rows of rank float32, for bfloat16 of the rank filled up to sixteens
    const void* y;
    long long ldy;
    void* out;                                  // y itself, or a bfloat16 result of a float32 y
    long long ldo;
    int m, n, k, rank, adapters, dtype, y_dtype, out_dtype, pdl;
};

extern "C" int tvb_add_adapters(const AdaptersCall* call, void* stream) {
    const AdaptersCall& c = *call;
    if (c.m <= 0 || c.n <= 0 || c.adapters <= 0) return 0;
    if (c.k <= 0 || c.rank <= 0 || c.rank > MAX_RANK || ceil_div(c.m, 16) > 65535) return TVB_BAD_ARGUMENT;
    if (c.y_dtype == c.out_dtype && (c.out != c.y || c.ldo != c.ldy)) return TVB_BAD_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    const bool many = c.dtype == TVB_BF16 && rows_go(c.m, c.adapters) == MANY;
    const int e = many && shrink_tma_takes(c.x, c.ldx, c.down, c.k, c.rank, c.adapters)
                      ? shrink_tma(Shrink{(const bf16*)c.x, c.ldx, (const bf16*)c.down, c.ids, c.scales, (bf16*)c.u, c.m, c.k, c.rank, c.adapters, 1, 0}, c.pdl, s)
                      : shrink(c.x, c.ldx, c.down, c.ids, c.scales, c.u, c.m, c.k, c.rank, c.adapters, c.dtype, c.pdl, s);
    if (e) return e;
    const Expand a{c.u, c.up, c.ids, c.y, c.ldy, c.out, c.ldo, c.m, c.n, c.rank, c.adapters};
    return many && c.out_dtype == TVB_BF16 && expand_tma_takes(c.up, c.y, c.ldy, c.n, c.rank, c.adapters, c.y_dtype)
               ? expand_tma(a, c.pdl, s)
               : expand(a, c.dtype, c.y_dtype, c.out_dtype, c.pdl, s);
}

// 0, or which bounded wait gave up in some launch since the last call; reading clears it.  Synchronises.
extern "C" int tvb_adapters_status() {
    int value = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&value, tvb_adapters_status_word, sizeof(int)) != cudaSuccess) return -1;
    if (value != 0) cudaMemcpyToSymbol(tvb_adapters_status_word, &zero, sizeof(int));
    return value;
}
