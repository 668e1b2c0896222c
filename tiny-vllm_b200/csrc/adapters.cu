// Low-rank adapters of many requests beside a shared projection: row t of y = x W^T becomes
//
//   y[t] + s_a (x[t] A_a^T) B_a^T        a = ids[t]; rows whose number names no adapter stay as they are
//
// with A [adapters, rank, k] and B [adapters, n, rank].  Two kernels: `shrink` makes u = x A^T (float32, summed over k in
// pieces that are added in order), `expand` takes u through B and adds it to y.  Rows come in any order; a tile of rows
// goes once over every adapter that one of its rows has.
//
// bfloat16: mma.sync m16n8k16 straight from global memory to registers (the products are a hundredth of the projection's,
// and a rank of 16 is one step of k: there is nothing for a pipeline through shared memory to hide behind).  A thread
// loads 16 bytes, eight neighbouring k, of each row; which k a fragment's place stands for is permuted alike in both
// operands.  u enters the second product as two bfloat16 whose sum is u to 2^-17 of it, so that no rounding of u is seen
// beside that of the result.  A row takes the sums of its own adapter alone: what other adapters hold, infinities among
// them, does not reach it.
// float32: the float32 cores.
//
// Bound by reading A, B and x and by reading and writing y.
#include "common.cuh"

namespace {

constexpr int THREADS = 128, WARPS = 4;
constexpr int MAX_RANK = 256;

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// values at, .., at + 7 of a row of `size` (zeros past its end, or where the row is not there)
template <bool WIDE> __device__ __forceinline__ uint4 load_8(const bf16* row, int at, int size, bool there) {
    if constexpr (WIDE) {                       // size is a multiple of 8, the row lies on 16 bytes
        return there && at < size ? *reinterpret_cast<const uint4*>(row + at) : make_uint4(0, 0, 0, 0);
    } else {
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = there && at + e < size ? (uint32_t)reinterpret_cast<const unsigned short*>(row)[at + e] : 0u;
        return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
}
template <bool WIDE> __device__ __forceinline__ uint2 load_4(const bf16* row, int at, int size, bool there) {
    if constexpr (WIDE) {                       // size is a multiple of 4, the row lies on 8 bytes
        return there && at < size ? *reinterpret_cast<const uint2*>(row + at) : make_uint2(0, 0);
    } else {
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = there && at + e < size ? (uint32_t)reinterpret_cast<const unsigned short*>(row)[at + e] : 0u;
        return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    }
}

struct Shrink {
    const bf16* x;
    int64_t ldx;
    const bf16* down;
    const int* ids;
    float* part;                                // [splits, m, rank]
    int m, k, rank, adapters;
    int splits, blocks_per_split;               // blocks of 32 k
};

// One pass over k blocks first, first + step, .. < end: sums[j] += 16 rows of x times 8 ranks from 8 j on.
template <int NR, bool WIDE>
__device__ __forceinline__ void shrink_pass(const Shrink& s, const bf16* lo, const bf16* hi, bool lo_there, bool hi_there, const bf16* down,
                                            int ranks, int first, int step, int end, float (&sums)[NR][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr int AHEAD = NR <= 2 ? 4 : 2;      // blocks in flight
    for (int b0 = first; b0 < end; b0 += AHEAD * step) {
        uint4 xl[AHEAD], xh[AHEAD], w[AHEAD][NR];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int b = b0 + i * step, at = b * 32 + 8 * t;
            xl[i] = load_8<WIDE>(lo, at, s.k, lo_there && b < end);
            xh[i] = load_8<WIDE>(hi, at, s.k, hi_there && b < end);
#pragma unroll
            for (int j = 0; j < NR; ++j)
                w[i][j] = load_8<WIDE>(down + (int64_t)(8 * j + g) * s.k, at, s.k, 8 * j + g < ranks && b < end);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                mma_16816(sums[j], xl[i].x, xh[i].x, xl[i].y, xh[i].y, w[i][j].x, w[i][j].y);
                mma_16816(sums[j], xl[i].z, xh[i].z, xl[i].w, xh[i].w, w[i][j].z, w[i][j].w);
            }
    }
}

// BY_ROWS: a warp has 16 rows of its own, over all k of the split, and goes through their adapters in turn.  Else: the CTA
// has 16 rows and the blockIdx.z-th of their adapters; its warps share k and meet in shared memory.
template <int NR, bool BY_ROWS, bool WIDE>
__global__ void __launch_bounds__(THREADS) shrink_kernel(Shrink s) {
    __shared__ float met[BY_ROWS ? 1 : WARPS][16][8 * NR];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % s.splits, rank0 = blockIdx.x / s.splits * 8 * NR, ranks = s.rank - rank0;
    const int row0 = BY_ROWS ? (blockIdx.y * WARPS + warp) * 16 : blockIdx.y * 16;
    const int first = split * s.blocks_per_split, end = min((s.k + 31) / 32, first + s.blocks_per_split);
    pdl_wait();
    pdl_launch_dependents();
    if (BY_ROWS && row0 >= s.m) return;
    // lanes 0 .. 15: a row's adapter, and the rows that share it
    int id = -1;
    if (lane < 16 && row0 + lane < s.m) {
        id = s.ids[row0 + lane];
        if ((unsigned)id >= (unsigned)s.adapters) id = -1;
    }
    const uint32_t alike = __match_any_sync(0xffffffffu, id);
    uint32_t leaders = __ballot_sync(0xffffffffu, id >= 0 && (alike & ((1u << lane) - 1u)) == 0);
    if constexpr (!BY_ROWS) {
        for (int d = 0; d < (int)blockIdx.z; ++d) leaders &= leaders - 1;
        if (leaders == 0) return;               // the whole CTA
        leaders &= -leaders;
    }
    const int lo_row = row0 + g, hi_row = row0 + g + 8;
    const bf16* lo = s.x + (int64_t)lo_row * s.ldx;
    const bf16* hi = s.x + (int64_t)hi_row * s.ldx;
    while (leaders) {
        const int leader = __ffs(leaders) - 1;
        leaders &= leaders - 1;
        const int adapter = __shfl_sync(0xffffffffu, id, leader);
        const uint32_t rows = __shfl_sync(0xffffffffu, alike, leader);
        const bf16* down = s.down + ((int64_t)adapter * s.rank + rank0) * s.k;
        const bool lo_there = rows >> g & 1, hi_there = rows >> (g + 8) & 1;
        float sums[NR][4] = {};
        shrink_pass<NR, WIDE>(s, lo, hi, lo_there, hi_there, down, ranks, BY_ROWS ? first : first + warp, BY_ROWS ? 1 : WARPS, end, sums);
        if constexpr (BY_ROWS) {
#pragma unroll
            for (int j = 0; j < NR; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int rank = 8 * j + 2 * t + (e & 1);
                    if ((e < 2 ? lo_there : hi_there) && rank < ranks)
                        s.part[((int64_t)split * s.m + (e < 2 ? lo_row : hi_row)) * s.rank + rank0 + rank] = sums[j][e];
                }
        } else {
#pragma unroll
            for (int j = 0; j < NR; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) met[warp][e < 2 ? g : g + 8][8 * j + 2 * t + (e & 1)] = sums[j][e];
            __syncthreads();
            for (int i = threadIdx.x; i < 16 * 8 * NR; i += THREADS) {
                const int row = i / (8 * NR), rank = i % (8 * NR);
                if (!(rows >> row & 1) || rank >= ranks) continue;
                float sum = met[0][row][rank];
#pragma unroll
                for (int w = 1; w < WARPS; ++w) sum += met[w][row][rank];
                s.part[((int64_t)split * s.m + row0 + row) * s.rank + rank0 + rank] = sum;
            }
        }
    }
}

struct Expand {
    const float* part;
    const void* up;                             // [adapters, n, rank]
    const int* ids;
    const float* scales;                        // [adapters] or null
    void* y;
    int64_t ldy;
    int m, n, rank, adapters, splits;
};

// u of a tile's rows, scaled, from its pieces in order; what a row without an adapter has is of no account
template <typename F> __device__ __forceinline__ void gather_u(const Expand& s, int row0, int rows, const int* ids, F&& put) {
    for (int i = threadIdx.x; i < rows * s.rank; i += blockDim.x) {
        const int row = i / s.rank, rank = i % s.rank;
        float sum = 0.0f;
        if (ids[row] >= 0) {
            const float* at = s.part + ((int64_t)row0 + row) * s.rank + rank;
            for (int p = 0; p < s.splits; ++p) sum += at[(int64_t)p * s.m * s.rank];
            if (s.scales) sum *= s.scales[ids[row]];
        }
        put(row, rank, sum);
    }
}

// the numbers of a tile's rows (-1: none), and the tile's adapters, each once, in `distinct`
template <int ROWS> __device__ __forceinline__ int find_adapters(const Expand& s, int row0, int* ids, int* distinct, int* count) {
    const int tid = threadIdx.x;
    if (tid == 0) *count = 0;
    if (tid < ROWS) {
        int id = row0 + tid < s.m ? s.ids[row0 + tid] : -1;
        ids[tid] = (unsigned)id < (unsigned)s.adapters ? id : -1;
    }
    __syncthreads();
    if (tid < ROWS && ids[tid] >= 0) {
        bool first = true;
        for (int j = 0; j < tid; ++j) first = first && ids[j] != ids[tid];
        // (in any order: a row adds the sums of one adapter)
        if (first) distinct[atomicAdd(count, 1)] = ids[tid];
    }
    __syncthreads();
    return *count;
}

// A tile of 16 MT rows and 128 columns of y, 32 columns a warp.  The columns of an n-tile are spread so that a thread holds
// eight neighbours of y: place c of tile j is column (c / 2) * 8 + 2 j + c % 2.
template <int MT, typename Y, bool WIDE>
__global__ void __launch_bounds__(THREADS) expand_kernel(Expand s) {
    constexpr int ROWS = 16 * MT, NT = 4;
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ int ids[ROWS], distinct[ROWS], distinct_count;
    const int padded = (s.rank + 15) / 16 * 16, pitch = padded + 8;
    bf16* u_hi = reinterpret_cast<bf16*>(raw);                                  // [ROWS][pitch]
    bf16* u_lo = u_hi + ROWS * pitch;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row0 = blockIdx.y * ROWS, n0 = blockIdx.x * 128 + warp * 32;
    const int rows = min(ROWS, s.m - row0);
    const bf16* up = reinterpret_cast<const bf16*>(s.up);
    pdl_wait();
    pdl_launch_dependents();
    const int count = find_adapters<ROWS>(s, row0, ids, distinct, &distinct_count);
    if (count == 0) return;
    for (int i = threadIdx.x; i < ROWS * pitch; i += THREADS) { u_hi[i] = from_float<bf16>(0.0f); u_lo[i] = from_float<bf16>(0.0f); }
    __syncthreads();
    gather_u(s, row0, rows, ids, [&](int row, int rank, float u) {
        const bf16 hi = from_float<bf16>(u);
        u_hi[row * pitch + rank] = hi;
        u_lo[row * pitch + rank] = from_float<bf16>(u - to_float<bf16>(hi));
    });
    __syncthreads();
    float total[MT][NT][4] = {};
    for (int d = 0; d < count; ++d) {
        const int adapter = distinct[d];
        const bf16* b = up + (int64_t)adapter * s.n * s.rank;
        float sums[MT][NT][4] = {};
        for (int r0 = 0; r0 < padded; r0 += 16) {
            uint2 w[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int column = n0 + (g >> 1) * 8 + 2 * j + (g & 1);
                w[j] = load_4<WIDE>(b + (int64_t)column * s.rank, r0 + 4 * t, s.rank, column < s.n);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const bf16* at = u_hi + (16 * i + g) * pitch + r0 + 4 * t;
                const uint2 hl = *reinterpret_cast<const uint2*>(at), hh = *reinterpret_cast<const uint2*>(at + 8 * pitch);
                const bf16* rest = at + ROWS * pitch;
                const uint2 ll = *reinterpret_cast<const uint2*>(rest), lh = *reinterpret_cast<const uint2*>(rest + 8 * pitch);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    mma_16816(sums[i][j], hl.x, hh.x, hl.y, hh.y, w[j].x, w[j].y);
                    mma_16816(sums[i][j], ll.x, lh.x, ll.y, lh.y, w[j].x, w[j].y);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const bool lo = ids[16 * i + g] == adapter, hi = ids[16 * i + g + 8] == adapter;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < 2 ? lo : hi) total[i][j][e] = sums[i][j][e];
        }
    }
    const int column = n0 + 8 * t;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int row = 16 * i + g + 8 * half;
            if (row >= rows || ids[row] < 0) continue;
            Y* y = reinterpret_cast<Y*>(s.y) + (int64_t)(row0 + row) * s.ldy + column;
            float add[8];
#pragma unroll
            for (int j = 0; j < NT; ++j) { add[2 * j] = total[i][j][2 * half]; add[2 * j + 1] = total[i][j][2 * half + 1]; }
            if (WIDE && column + 8 <= s.n) {
                if constexpr (sizeof(Y) == 2) {
                    float old[8];
                    unpack_bf16x8(*reinterpret_cast<const uint4*>(y), old);
#pragma unroll
                    for (int e = 0; e < 8; ++e) add[e] += old[e];
                    *reinterpret_cast<uint4*>(y) = pack_bf16x8(add);
                } else {
                    const float4 a = reinterpret_cast<const float4*>(y)[0], c = reinterpret_cast<const float4*>(y)[1];
                    reinterpret_cast<float4*>(y)[0] = make_float4(a.x + add[0], a.y + add[1], a.z + add[2], a.w + add[3]);
                    reinterpret_cast<float4*>(y)[1] = make_float4(c.x + add[4], c.y + add[5], c.z + add[6], c.w + add[7]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (column + e < s.n) y[e] = from_float<Y>(to_float<Y>(y[e]) + add[e]);
            }
        }
}

// ---- float32: a warp makes four ranks of a row over its split of k
struct Shrink32 {
    const float* x;
    int64_t ldx;
    const float* down;
    const int* ids;
    float* part;
    int m, k, rank, adapters, splits, per_split;
};
template <int VEC> __global__ void __launch_bounds__(THREADS) shrink_f32_kernel(Shrink32 s) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_row = s.splits * ((s.rank + 4 * WARPS - 1) / (4 * WARPS)), place = blockIdx.x % per_row;
    const int row = blockIdx.x / per_row, split = place % s.splits, rank0 = (place / s.splits * WARPS + warp) * 4;
    pdl_wait();
    pdl_launch_dependents();
    const int id = s.ids[row];
    if ((unsigned)id >= (unsigned)s.adapters || rank0 >= s.rank) return;
    const float* x = s.x + (int64_t)row * s.ldx;
    const float* down = s.down + ((int64_t)id * s.rank + rank0) * s.k;
    const int end = min(s.k, (split + 1) * s.per_split);
    float sums[4] = {};
    for (int at = split * s.per_split + lane * VEC; at < end; at += 32 * VEC) {
        float v[VEC], w[VEC];
        load_values<VEC>(x + at, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (rank0 + j >= s.rank) break;
            load_values<VEC>(down + (int64_t)j * s.k + at, w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) sums[j] = fmaf(v[e], w[e], sums[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float sum = warp_sum(sums[j]);
        if (lane == j && rank0 + j < s.rank) s.part[((int64_t)split * s.m + row) * s.rank + rank0 + j] = sum;
    }
}

// a thread makes one column of 16 rows
template <int VEC> __global__ void __launch_bounds__(THREADS) expand_f32_kernel(Expand s) {
    constexpr int ROWS = 16;
    extern __shared__ __align__(16) unsigned char raw[];
    __shared__ int ids[ROWS], distinct[ROWS], distinct_count;
    float* u = reinterpret_cast<float*>(raw);                                   // [ROWS][pitch]
    const int pitch = (s.rank + 3) / 4 * 4;
    const int row0 = blockIdx.y * ROWS, rows = min(ROWS, s.m - row0), column = blockIdx.x * THREADS + threadIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    const int count = find_adapters<ROWS>(s, row0, ids, distinct, &distinct_count);
    if (count == 0) return;
    gather_u(s, row0, rows, ids, [&](int row, int rank, float v) { u[row * pitch + rank] = v; });
    __syncthreads();
    if (column >= s.n) return;
    for (int d = 0; d < count; ++d) {
        const float* b = reinterpret_cast<const float*>(s.up) + ((int64_t)distinct[d] * s.n + column) * s.rank;
        float sums[ROWS] = {};
        for (int r = 0; r < s.rank; r += VEC) {
            float w[VEC];
            load_values<VEC>(b + r, w);
#pragma unroll
            for (int row = 0; row < ROWS; ++row)
                if (ids[row] == distinct[d])
#pragma unroll
                    for (int e = 0; e < VEC; ++e) sums[row] = fmaf(u[row * pitch + r + e], w[e], sums[row]);
        }
#pragma unroll
        for (int row = 0; row < ROWS; ++row)
            if (row < rows && ids[row] == distinct[d]) {
                float* y = reinterpret_cast<float*>(s.y) + (int64_t)(row0 + row) * s.ldy + column;
                *y += sums[row];
            }
    }
}

// ------------------------------------------------------------------ host side
constexpr int FEW_ROWS = 128;                   // rows up to which a CTA has 16 rows and one adapter

int ceil_div(int a, int b) { return (a + b - 1) / b; }

// pieces of k, so that the grid fills the GPU about twice and a warp keeps a few blocks of 32
int shrink_splits(int m, int k, int rank, int f32) {
    const int blocks = ceil_div(k, 32);
    if (f32) return max(1, min(min(8, k / 512), ceil_div(1184, m * ceil_div(rank, 16))));
    if (m <= FEW_ROWS) return max(1, min(16, blocks / 8));
    return max(1, min(min(8, blocks / 16), ceil_div(444, ceil_div(m, 64) * ceil_div(rank, 64))));
}

template <typename K, typename S> int launch(K kernel, dim3 grid, size_t shared, int pdl, cudaStream_t stream, const S& s) {
    if (shared > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * 64 * (MAX_RANK + 8) * 2);
        if (e != cudaSuccess) return (int)e;
    }
    TvbLaunch at(grid, dim3(THREADS), shared, stream, pdl);
    const cudaError_t e = cudaLaunchKernelEx(&at.config, kernel, s);
    return e == cudaSuccess ? tvb_last_error() : (int)e;
}

}  // namespace

extern "C" int tvb_adapters_max_rank() { return MAX_RANK; }

// float32 of scratch: the pieces of u
extern "C" long long tvb_adapters_scratch(int m, int k, int rank, int dtype) {
    return m <= 0 ? 0 : (long long)shrink_splits(m, k, rank, dtype == TVB_F32) * m * rank;
}

extern "C" int tvb_adapters_shrink(const void* x, long long ldx, const void* down, const int* ids, float* part, int m, int k, int rank,
                                   int adapters, int dtype, int pdl, void* stream) {
    if (m <= 0 || adapters <= 0) return 0;
    if (k <= 0 || rank <= 0 || rank > MAX_RANK) return TVB_BAD_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    const int splits = shrink_splits(m, k, rank, dtype == TVB_F32);
    if (dtype == TVB_F32) {
        const bool wide = k % 4 == 0 && ldx % 4 == 0 && !(((uintptr_t)x | (uintptr_t)down) & 15);
        const int per = ceil_div(ceil_div(k, splits), 4) * 4;
        const Shrink32 a{(const float*)x, ldx, (const float*)down, ids, part, m, k, rank, adapters, splits, per};
        const long long ctas = (long long)m * splits * ceil_div(rank, 4 * WARPS);
        if (ctas > 0x7fffffffLL) return TVB_BAD_ARGUMENT;
        const dim3 grid((unsigned)ctas);
        return wide ? launch(shrink_f32_kernel<4>, grid, 0, pdl, s, a) : launch(shrink_f32_kernel<1>, grid, 0, pdl, s, a);
    }
    if (dtype != TVB_BF16) return TVB_BAD_ARGUMENT;
    const bool wide = k % 8 == 0 && ldx % 8 == 0 && !(((uintptr_t)x | (uintptr_t)down) & 15);
    const Shrink a{(const bf16*)x, ldx, (const bf16*)down, ids, part, m, k, rank, adapters, splits, ceil_div(ceil_div(k, 32), splits)};
    if (m <= FEW_ROWS) {
        const dim3 grid(splits * ceil_div(rank, 16), ceil_div(m, 16), min(min(16, m), adapters));
        return wide ? launch(shrink_kernel<2, false, true>, grid, 0, pdl, s, a) : launch(shrink_kernel<2, false, false>, grid, 0, pdl, s, a);
    }
    if (ceil_div(m, 64) > 65535) return TVB_BAD_ARGUMENT;
    if (rank <= 16) {
        const dim3 grid(splits, ceil_div(m, 64));
        return wide ? launch(shrink_kernel<2, true, true>, grid, 0, pdl, s, a) : launch(shrink_kernel<2, true, false>, grid, 0, pdl, s, a);
    }
    const dim3 grid(splits * ceil_div(rank, 64), ceil_div(m, 64));
    return wide ? launch(shrink_kernel<8, true, true>, grid, 0, pdl, s, a) : launch(shrink_kernel<8, true, false>, grid, 0, pdl, s, a);
}

// dtype: of x, A and B; y_dtype: of y (float32 with either, bfloat16 with bfloat16)
extern "C" int tvb_adapters_expand(const float* part, const void* up, const int* ids, const float* scales, void* y, long long ldy, int m,
                                   int n, int k, int rank, int adapters, int dtype, int y_dtype, int pdl, void* stream) {
    if (m <= 0 || n <= 0 || adapters <= 0) return 0;
    if (rank <= 0 || rank > MAX_RANK) return TVB_BAD_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    const Expand a{part, up, ids, scales, y, ldy, m, n, rank, adapters, shrink_splits(m, k, rank, dtype == TVB_F32)};
    if (ceil_div(m, 16) > 65535) return TVB_BAD_ARGUMENT;
    if (dtype == TVB_F32) {
        if (y_dtype != TVB_F32) return TVB_BAD_ARGUMENT;
        const dim3 grid(ceil_div(n, THREADS), ceil_div(m, 16));
        const size_t shared = 16 * (size_t)((rank + 3) / 4 * 4) * 4;
        return rank % 4 == 0 && !((uintptr_t)up & 15) ? launch(expand_f32_kernel<4>, grid, shared, pdl, s, a)
                                                     : launch(expand_f32_kernel<1>, grid, shared, pdl, s, a);
    }
    if (dtype != TVB_BF16) return TVB_BAD_ARGUMENT;
    const int size = y_dtype == TVB_F32 ? 4 : 2;
    const bool wide = rank % 4 == 0 && !((uintptr_t)up & 7) && !((uintptr_t)y & 15) && ldy * size % 16 == 0;
    const bool few = m <= FEW_ROWS;
    const int rows = few ? 16 : 64;
    const dim3 grid(ceil_div(n, 128), ceil_div(m, rows));
    const size_t shared = 2 * (size_t)rows * ((rank + 15) / 16 * 16 + 8) * 2;
    if (y_dtype == TVB_F32) {
        if (few) return wide ? launch(expand_kernel<1, float, true>, grid, shared, pdl, s, a) : launch(expand_kernel<1, float, false>, grid, shared, pdl, s, a);
        return wide ? launch(expand_kernel<4, float, true>, grid, shared, pdl, s, a) : launch(expand_kernel<4, float, false>, grid, shared, pdl, s, a);
    }
    if (y_dtype != TVB_BF16) return TVB_BAD_ARGUMENT;
    if (few) return wide ? launch(expand_kernel<1, bf16, true>, grid, shared, pdl, s, a) : launch(expand_kernel<1, bf16, false>, grid, shared, pdl, s, a);
    return wide ? launch(expand_kernel<4, bf16, true>, grid, shared, pdl, s, a) : launch(expand_kernel<4, bf16, false>, grid, shared, pdl, s, a);
}
