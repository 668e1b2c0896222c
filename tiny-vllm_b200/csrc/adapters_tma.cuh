// The adapters' two products for many rows as they lie (included by adapters.cu): bfloat16, ranks of up to 64, x and A on 16 bytes for
// `shrink`, y and B (a rank that is a multiple of 8) for `expand`.  Tiles come in by tensor-map copies in the 128-byte swizzle that a warp of its own issues,
// four warps multiply them with mma.sync; full and empty mbarriers between them, every wait bounded (tc5.cuh).
//
//   shrink  64 rows and up to 64 ranks a CTA, stages of 64 k; the CTAs of a cluster have a piece of k each and add up through
//           distributed shared memory.
//   expand  64 rows a CTA, which walks over tiles of 64 columns: the tile of y comes in, the products with the B of every adapter of the
//           rows are made in float32 and added in place, each to its own adapter's rows, and every warp copies its 16 rows out again.
//           (Rows without an adapter go out as they came in.)
//
// Bound by the instructions between the copies as much as by the traffic of x and y through L2: 4099 rows, 4096 -> 4096, rank 64
// take 17 us for shrink and 24 us for expand (1 of it the look at whether every sum is finite, mend_sums), where 101 MB pass, 15 us at the speed of HBM (the kernels of adapters.cu: 27 and
// 33 us).  Without the rests of u, which bfloat16 accuracy of the sum would allow and float32 accuracy of u does not, expand
// would save 5 us.  Measured and not taken: 4, 8 and 11 tiles of y a CTA (rows without an adapter leave their SM idle: 1 to 5 us
// more), longer rings and fewer CTAs an SM (1 to 3 us more), more pieces of k (3 us more).
#pragma once

#include "tc5.cuh"

__device__ int tvb_adapters_status_word = 0;

constexpr int TMA_ROWS = 64, TMA_THREADS = THREADS + 32;

// 16-byte word `word` of row `row` in a tile whose rows are 128 swizzled bytes
__device__ __forceinline__ uint32_t swizzled(uint32_t tile, int row, int word) { return tile + row * 128 + ((word ^ (row & 7)) << 4); }
__device__ __forceinline__ void ldmatrix_x4_at(uint32_t* r, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(src) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;\n" ::"n"(N) : "memory"); }
template <int N> __device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group %0;\n" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t load_shared_32(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void store_shared_32(uint32_t at, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(at), "r"(v) : "memory"); }

// ------------------------------------------------------------------ u = s x A^T
template <int RANKS> struct ShrinkTma {
    static constexpr int RING = 4, X_BYTES = TMA_ROWS * 128, STAGE = X_BYTES + RANKS * 128, SUM_PITCH = RANKS + 4;
    static constexpr int RING_BYTES = RING * STAGE, SUM_BYTES = TMA_ROWS * SUM_PITCH * 4;
    static constexpr int AREA = RING_BYTES > SUM_BYTES ? RING_BYTES : SUM_BYTES;
    static constexpr int BYTES = 1024 + AREA + 2 * RING * 8 + 16;
};
template <int RANKS>
__global__ void __launch_bounds__(TMA_THREADS) shrink_tma_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a,
                                                                 Shrink s) {
    using S = ShrinkTma<RANKS>;
    extern __shared__ uint8_t raw_tma[];
    __shared__ int ids[TMA_ROWS], distinct[TMA_ROWS];
    const uint32_t base = (smem_address(raw_tma) + 1023u) & ~1023u;
    uint8_t* area = raw_tma + (base - smem_address(raw_tma));
    float* sums_s = reinterpret_cast<float*>(area);                             // [TMA_ROWS][SUM_PITCH], over the ring
    auto full = [&](int i) { return base + S::AREA + 8u * i; };
    auto empty = [&](int i) { return base + S::AREA + 8u * (S::RING + i); };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(area + S::AREA + 2 * S::RING * 8);
    int* status = &tvb_adapters_status_word;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % s.splits, row0 = blockIdx.y * TMA_ROWS, padded = padded_rank(s.rank);
    const int first = split * s.per_split, stages = max(0, min((s.k + STAGE_K - 1) / STAGE_K, first + s.per_split) - first);
    if (tid == 0) {
        for (int i = 0; i < S::RING; ++i) {
            mbar_init(full(i), 1);
            mbar_init(empty(i), WARPS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        prefetch_tensormap(&map_x);
        prefetch_tensormap(&map_a);
    }
    pdl_wait();
    pdl_launch_dependents();
    const int count = find_adapters<TMA_ROWS>(s.ids, s.m, s.adapters, row0, ids, distinct);       // (its barriers: ours are set up)
    uint32_t used = 0;                          // stages so far, of all adapters
    for (int d = blockIdx.z; d < count; d += gridDim.z, used += stages) {       // the same for the whole cluster
        const int adapter = distinct[d];
        if (warp == WARPS) {
            if (lane == 0)
                for (int i = 0; i < stages; ++i) {
                    const uint32_t n = used + i, slot = n % S::RING;
                    if (n >= S::RING && !mbar_wait(empty(slot), (n / S::RING - 1) & 1u, abort_flag, status, 1)) break;
                    mbar_arrive_expect(full(slot), S::STAGE);
                    tma_load_2d(base + slot * S::STAGE, &map_x, (first + i) * STAGE_K, row0, full(slot));
                    tma_load_2d(base + slot * S::STAGE + S::X_BYTES, &map_a, (first + i) * STAGE_K, adapter * s.rank, full(slot));
                }
            __syncwarp();
        }
        float sums[RANKS / 8][4] = {};
        if (warp < WARPS)
            for (int i = 0; i < stages; ++i) {
                const uint32_t n = used + i, slot = n % S::RING, x_s = base + slot * S::STAGE, a_s = x_s + S::X_BYTES;
                if (!__all_sync(0xffffffffu, mbar_wait(full(slot), (n / S::RING) & 1u, abort_flag, status, 2))) break;
#pragma unroll
                for (int kk = 0; kk < STAGE_K / 16; ++kk) {
                    uint32_t a[4];
                    ldmatrix_x4_at(a, swizzled(x_s, warp * 16 + (lane & 15), kk * 2 + (lane >> 4)));
#pragma unroll
                    for (int j = 0; j < RANKS / 16; ++j) {
                        uint32_t b[4];
                        const int matrix = lane >> 3;
                        ldmatrix_x4_at(b, swizzled(a_s, j * 16 + (matrix >> 1) * 8 + (lane & 7), kk * 2 + (matrix & 1)));
                        mma_16816(sums[2 * j], a[0], a[1], a[2], a[3], b[0], b[1]);
                        mma_16816(sums[2 * j + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty(slot));
            }
        __syncthreads();                        // every stage is read
        if (warp < WARPS)
#pragma unroll
            for (int j = 0; j < RANKS / 8; ++j)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    *reinterpret_cast<float2*>(sums_s + (warp * 16 + g + 8 * half) * S::SUM_PITCH + 8 * j + 2 * t) =
                        make_float2(sums[j][2 * half], sums[j][2 * half + 1]);
        cluster_arrive();
        cluster_wait();
        // a CTA adds the pieces of its share of the rows
        const float scale = s.scales ? s.scales[adapter] : 1.0f;
        const int share = TMA_ROWS / s.splits;
        for (int i = tid; i < share * RANKS; i += TMA_THREADS) {
            const int row = split * share + i / RANKS, rank = i % RANKS;
            if (ids[row] != adapter || rank >= padded) continue;
            float piece[MAX_SPLITS];
#pragma unroll
            for (int p = 0; p < MAX_SPLITS; ++p)
                piece[p] = p < s.splits ? cluster.map_shared_rank(sums_s, p)[row * S::SUM_PITCH + rank] : 0.0f;
            float sum = piece[0];
#pragma unroll
            for (int p = 1; p < MAX_SPLITS; ++p) sum += piece[p];
            store_u(s.u, row0 + row, rank, padded, rank < s.rank ? sum * scale : 0.0f);
        }
        fence_async_shared();                   // the next adapter's copies come over what was read here
        cluster_arrive();
        cluster_wait();
    }
    if (*abort_flag) {
        // copies may still be in flight towards this CTA's memory: give them time
        const long long started = clock64();
        while (clock64() - started < 400000) __nanosleep(1000);
    }
}

// ------------------------------------------------------------------- y += u B^T
struct ExpandTma {
    static constexpr int COLUMNS = 64, Y_RING = 4, B_RING = 2, TILE = TMA_ROWS * 128;
    static constexpr int BYTES = 1024 + (Y_RING + B_RING) * TILE + 2 * (Y_RING + B_RING) * 8 + 16;
};
__global__ void __launch_bounds__(TMA_THREADS, 4) expand_tma_kernel(const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_out,
                                                                    const __grid_constant__ CUtensorMap map_b, Expand s, int tiles_each) {
    using S = ExpandTma;
    extern __shared__ uint8_t raw_tma[];
    __shared__ int ids[TMA_ROWS], distinct[TMA_ROWS];
    const uint32_t base = (smem_address(raw_tma) + 1023u) & ~1023u, b_base = base + S::Y_RING * S::TILE, bars = b_base + S::B_RING * S::TILE;
    auto y_full = [&](int i) { return bars + 8u * i; };
    auto y_empty = [&](int i) { return bars + 8u * (S::Y_RING + i); };
    auto b_full = [&](int i) { return bars + 8u * (2 * S::Y_RING + i); };
    auto b_empty = [&](int i) { return bars + 8u * (2 * S::Y_RING + S::B_RING + i); };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(raw_tma + (bars - smem_address(raw_tma)) + 2 * (S::Y_RING + S::B_RING) * 8);
    int* status = &tvb_adapters_status_word;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int row0 = blockIdx.y * TMA_ROWS, padded = padded_rank(s.rank);
    const int tile0 = blockIdx.x * tiles_each, tiles = min((s.n + S::COLUMNS - 1) / S::COLUMNS, tile0 + tiles_each) - tile0;
    if (tid == 0) {
        for (int i = 0; i < S::Y_RING; ++i) {
            mbar_init(y_full(i), 1);
            mbar_init(y_empty(i), WARPS);
        }
        for (int i = 0; i < S::B_RING; ++i) {
            mbar_init(b_full(i), 1);
            mbar_init(b_empty(i), WARPS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        prefetch_tensormap(&map_y);
        prefetch_tensormap(&map_out);
        prefetch_tensormap(&map_b);
    }
    // (before `shrink` is through, see expand_rows: the adapters here, the first tiles of y and B below)
    const int count = find_adapters<TMA_ROWS>(s.ids, s.m, s.adapters, row0, ids, distinct);       // (its barriers: ours are set up)
    if (warp < WARPS || count == 0) {
        pdl_wait();
        pdl_launch_dependents();
    }
    if (count == 0) return;                     // the whole CTA
    if (warp == WARPS) {
        if (lane == 0) {
            bool alive = true;
            uint32_t n = 0;                     // tiles of B so far
            for (int i = 0; i < tiles && alive; ++i) {
                const int slot = i % S::Y_RING, column = (tile0 + i) * S::COLUMNS;
                if (i >= S::Y_RING && !mbar_wait(y_empty(slot), (i / S::Y_RING - 1) & 1u, abort_flag, status, 3)) break;
                mbar_arrive_expect(y_full(slot), S::TILE);
                tma_load_2d(base + slot * S::TILE, &map_y, column, row0, y_full(slot));
                for (int d = 0; d < count; ++d, ++n) {
                    const uint32_t at = n % S::B_RING;
                    if (n >= S::B_RING && !mbar_wait(b_empty(at), (n / S::B_RING - 1) & 1u, abort_flag, status, 4)) { alive = false; break; }
                    mbar_arrive_expect(b_full(at), S::TILE);
                    tma_load_2d(b_base + at * S::TILE, &map_b, 0, distinct[d] * s.n + column, b_full(at));
                }
            }
        }
        __syncwarp();
    } else {
        // u of rows g and g + 8 of the warp's: heads, then rests
        uint32_t u[2][4][4];
        const int rows[2] = {warp * 16 + g, warp * 16 + g + 8};
        const bool has[2] = {ids[rows[0]] >= 0, ids[rows[1]] >= 0};             // (a row without an adapter has no u)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = 16 * k + (e >> 1) * 8 + 2 * t;
                    u[q][k][e] = has[e & 1] && at < padded ? *reinterpret_cast<const uint32_t*>(reinterpret_cast<const bf16*>(s.u) +
                                                                 ((int64_t)(row0 + rows[e & 1]) * 2 + q) * padded + at) : 0u;
                }
        const bool stores = __any_sync(0xffffffffu, has[0] || has[1]);
        uint32_t n = 0;
        bool alive = true;
        for (int i = 0; i < tiles && alive; ++i) {
            const int slot = i % S::Y_RING;
            const uint32_t y_s = base + slot * S::TILE;
            if (!__all_sync(0xffffffffu, mbar_wait(y_full(slot), (i / S::Y_RING) & 1u, abort_flag, status, 5))) break;
            for (int d = 0; d < count; ++d, ++n) {
                const uint32_t at = n % S::B_RING, b_s = b_base + at * S::TILE;
                if (!__all_sync(0xffffffffu, mbar_wait(b_full(at), (n / S::B_RING) & 1u, abort_flag, status, 6))) { alive = false; break; }
                const bool mine[2] = {ids[rows[0]] == distinct[d], ids[rows[1]] == distinct[d]};
                if (__any_sync(0xffffffffu, mine[0] || mine[1])) {
                    float sums[8][4] = {};                                      // columns 8 j + 2 t and the next of rows g and g + 8
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (16 * k >= padded) break;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t b[4];
                            const int matrix = lane >> 3;
                            ldmatrix_x4_at(b, swizzled(b_s, j * 16 + (matrix >> 1) * 8 + (lane & 7), 2 * k + (matrix & 1)));
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                mma_16816(sums[2 * j], u[q][k][0], u[q][k][1], u[q][k][2], u[q][k][3], b[0], b[1]);
                                mma_16816(sums[2 * j + 1], u[q][k][0], u[q][k][1], u[q][k][2], u[q][k][3], b[2], b[3]);
                            }
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (mine[h]) {
                            float add[16];
#pragma unroll
                            for (int j = 0; j < 8; ++j) { add[2 * j] = sums[j][2 * h]; add[2 * j + 1] = sums[j][2 * h + 1]; }
                            mend_sums(add, reinterpret_cast<const bf16*>(s.u) + (int64_t)(row0 + rows[h]) * 2 * padded, padded,
                                      reinterpret_cast<const bf16*>(s.up) + (int64_t)distinct[d] * s.n * s.rank, s.rank, s.n,
                                      [&](int c) { return (tile0 + i) * S::COLUMNS + c / 2 * 8 + 2 * t + c % 2; });
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const uint32_t to = swizzled(y_s, rows[h], j) + 4 * t, v = load_shared_32(to);
                                store_shared_32(to, pack_bf16x2(__uint_as_float(v << 16) + add[2 * j],
                                                                __uint_as_float(v & 0xffff0000u) + add[2 * j + 1]));
                            }
                        }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(b_empty(at));
            }
            if (stores) {
                fence_async_shared();
                __syncwarp();
                if (lane == 0) {
                    if (row0 + warp * 16 < s.m) tma_store_2d(&map_out, y_s + warp * 2048, (tile0 + i) * S::COLUMNS, row0 + warp * 16);
                    bulk_commit();
                    bulk_wait_read<1>();        // the tile before this one has gone
                }
            }
            if (lane == 0 && i > 0) mbar_arrive(y_empty((i - 1) % S::Y_RING));
        }
        if (lane == 0) bulk_wait<0>();          // written, before what follows this kernel may read it
    }
    __syncthreads();
    if (*abort_flag) {
        const long long started = clock64();
        while (clock64() - started < 400000) __nanosleep(1000);
    }
}

inline bool shrink_tma_takes(const void* x, long long ldx, const void* down, int k, int rank, int adapters) {
    return rank <= 64 && k % 8 == 0 && ldx >= k && ldx % 8 == 0 && !(((uintptr_t)x | (uintptr_t)down) & 15) && (long long)adapters * rank < 0x7fffffffLL;
}
inline bool expand_tma_takes(const void* up, const void* y, long long ldy, int n, int rank, int adapters, int y_dtype) {
    return rank <= 64 && rank % 8 == 0 && n >= 8 && ldy >= n && ldy % 8 == 0 && y_dtype == TVB_BF16 && !(((uintptr_t)up | (uintptr_t)y) & 15) &&
           (long long)adapters * n < 0x7fffffffLL;
}
inline bool matrix_map(CUtensorMap* map, const void* p, long long rows, long long columns, long long ld, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    return tvb_make_map(map, p, 2, dims, strides, box);
}
template <typename K, typename... A> int launch_tma(K kernel, dim3 grid, int shared, int cluster, int pdl, cudaStream_t stream, const A&... arguments) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
    if (e != cudaSuccess) return (int)e;
    TvbLaunch at(grid, dim3(TMA_THREADS), shared, stream, pdl, cluster);
    const cudaError_t launched = cudaLaunchKernelEx(&at.config, kernel, arguments...);
    return launched == cudaSuccess ? tvb_last_error() : (int)launched;
}
inline int shrink_tma(Shrink a, int pdl, cudaStream_t s) {
    // pieces of k while the CTAs still have one round on the GPU (three an SM)
    const int stages = (a.k + STAGE_K - 1) / STAGE_K, rows = (a.m + TMA_ROWS - 1) / TMA_ROWS;
    while (a.splits < MAX_SPLITS && a.splits * 4 <= stages && (long long)rows * a.splits * 2 <= 3 * 148) a.splits *= 2;
    a.per_split = (stages + a.splits - 1) / a.splits;
    CUtensorMap map_x, map_a;
    if (!matrix_map(&map_x, a.x, a.m, a.k, a.ldx, TMA_ROWS) || !matrix_map(&map_a, a.down, (long long)a.adapters * a.rank, a.k, a.k, a.rank <= 16 ? 16 : 64))
        return (int)cudaErrorNotSupported;
    const dim3 grid(a.splits, rows, a.adapters < 2 ? 1 : 2);
    return a.rank <= 16 ? launch_tma(shrink_tma_kernel<16>, grid, ShrinkTma<16>::BYTES, a.splits, pdl, s, map_x, map_a, a)
                        : launch_tma(shrink_tma_kernel<64>, grid, ShrinkTma<64>::BYTES, a.splits, pdl, s, map_x, map_a, a);
}
inline int expand_tma(const Expand& a, int pdl, cudaStream_t s) {
    CUtensorMap map_y, map_out, map_b;
    if (!matrix_map(&map_y, a.y, a.m, a.n, a.ldy, TMA_ROWS) || !matrix_map(&map_out, a.y, a.m, a.n, a.ldy, 16) ||
        !matrix_map(&map_b, a.up, (long long)a.adapters * a.n, a.rank, a.rank, ExpandTma::COLUMNS))
        return (int)cudaErrorNotSupported;
    const int rows = (a.m + TMA_ROWS - 1) / TMA_ROWS, tiles = (a.n + ExpandTma::COLUMNS - 1) / ExpandTma::COLUMNS;
    // up to three tiles a CTA: rows without an adapter leave at once, and what is left has to even out
    const int across = max(1, min(tiles, 4 * 148 / rows)), each = min(3, (tiles + across - 1) / across);
    const dim3 grid((tiles + each - 1) / each, rows);
    return launch_tma(expand_tma_kernel, grid, ExpandTma::BYTES, 0, pdl, s, map_y, map_out, map_b, a, each);
}
