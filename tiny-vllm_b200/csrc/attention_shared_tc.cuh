// The pieces of the shared keys on the fifth-generation tensor cores (included by attention_shared.cu): bfloat16, head sizes
// 64 and 128, pages of 8 to 128 tokens (a power of two).
//
// A CTA has up to 128 query rows (the q heads of one kv head of as many tokens as fit) and a piece of the keys in blocks of 128.
// S = Q K^T and O += P V are tcgen05.mma with the accumulators in tensor memory; Q comes in one copy (a box of heads x tokens),
// K and V page by page, in the 128-byte swizzle.  The blocks go alternately to two groups of 128 softmax threads, a thread a
// query row; each group has its own S and O, so that one group's exponentials run under the other's products.  P (two bfloat16 a
// column) lies over the columns of S it was made from and is the second product's a operand there.  O is scaled only when a row's
// maximum has grown by more than 2^8 since the reference that its exponentials use was set.  No key of a piece is hidden from
// one row and seen by another, so the only masks are the end of the keys and pages that are none.
//
// Roles: warps 0 and 11 issue the copies of keys and of values (lane p the page p of a block), a thread of warp 1 the products Q K^T, warps 2 to 5 and 6 to 9
// are the softmax groups, warp 10 issues P V (and zeroes rows of V behind the last shared key: what a page holds there is of no
// account).  Every wait is bounded (tc5.cuh).
//
// Bound by a block's chain (a tile's arrival, S, the softmax, P V) of 1.2 us, of which two run side by side: 16 tiles of 120 rows over
// 6,144 keys on 64 SMs take 21 us beside attend_own's reading; whole calls, us with this kernel / with
// attend_shared_bf16_kernel: 60 tokens behind 6,144 keys, 32 / 8 heads of size 128, 28.2 / 68.6; three groups of 13 behind 2,896, 64 / 8
// heads, 31.3 / 59.9.
#pragma once

#include "tc5.cuh"

constexpr int TC_THREADS = 384, TC_ROWS = 128, TC_KEYS = 128, TC_GROUP_WARPS = 4;
constexpr int TC_HALF = 128 * 64 * 2;           // [128 rows, 64 values] bfloat16: one swizzled sub-tile
constexpr float TC_RESCALE = 8.0f;              // log2 of the growth of a row's maximum that moves its reference
constexpr uint32_t TC_COLUMNS = 512;

template <int HD> struct TcShared {
    static constexpr int TILE = HD / 64 * TC_HALF;                              // a Q, K or V tile
    // A tile takes 2,500 cycles to come in beside what else the GPU reads, a block's products and softmax 2,000.
    static constexpr int K_RING = 3, V_RING = 3;
    static constexpr int Q_FULL = 0, K_FULL = 1, K_EMPTY = K_FULL + K_RING, V_FULL = K_EMPTY + K_RING, V_EMPTY = V_FULL + V_RING,
                         S_FULL = V_EMPTY + V_RING, P_FULL = S_FULL + 2,
                         P_READ = P_FULL + 2, O_LAST = P_READ + 2, SECOND_DONE = O_LAST + 2, BARRIERS = SECOND_DONE + 1;
    static constexpr int BYTES = TILE * (1 + K_RING + V_RING) + BARRIERS * 8 + 16 + 1024;
};

__device__ int tvb_attention_shared_status_word = 0;

template <int HD>
__global__ void __launch_bounds__(TC_THREADS, 1)
attend_shared_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, Attend a, int tile_tokens) {
    using T = TcShared<HD>;
    extern __shared__ uint8_t raw_tc[];
    const int heads = a.num_q / a.num_kv;
    const uint32_t base = (smem_address(raw_tc) + 1023u) & ~1023u;
    uint8_t* aligned = raw_tc + (base - smem_address(raw_tc));
    const uint32_t q_at = base, kv_at = base + T::TILE;
    // over the first Q tile, when it has been multiplied for the last time: [row][reference, denominator] of the second group, then
    // [row] place of the result
    float* exchange = reinterpret_cast<float*>(aligned);
    const uint32_t bars = base + T::TILE * (1 + T::K_RING + T::V_RING);
    auto bar = [&](int i) { return bars + 8u * i; };
    uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(aligned + T::TILE * (1 + T::K_RING + T::V_RING) + T::BARRIERS * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);
    int* status = &tvb_attention_shared_status_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // what needs nothing of the kernel before, while that ends
    if (threadIdx.x == 0) {
        for (int i = 0; i < T::BARRIERS; ++i)
            mbar_init(bar(i), (i >= T::P_FULL && i < T::P_FULL + 2) || i == T::SECOND_DONE ? TC_GROUP_WARPS : 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        prefetch_tensormap(&map_q);
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
    }
    if (warp == 1) tmem_alloc(smem_address(tmem_base_slot), TC_COLUMNS);
    pdl_wait();
    pdl_launch_dependents();
    Piece p;
    const int tile_rows = tile_tokens * heads;
    const bool found = find_shared_piece(a, tile_rows, p);                      // the same for the whole CTA
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_base_slot;
    if (!found) {
        if (warp == 1) tmem_free(tmem_base, TC_COLUMNS);
        return;
    }
    const int blocks = (p.range.end - p.range.first + TC_KEYS - 1) / TC_KEYS, pages_per_block = TC_KEYS / a.page_size;
    // Two rings, of keys and of values: block j is in slot j % its length.
    // page of this lane in block j as it stands in the table, -1 past the keys; whether it is one is asked where it is used, since the
    // warp would wait for the load there and then
    auto page_of = [&](int j) -> int {
        const int index = p.range.first / a.page_size + j * pages_per_block + lane;
        return lane < pages_per_block && j < blocks && (int64_t)index * a.page_size < p.range.end ? __ldcg(p.table + index) : -1;
    };
    const uint32_t k_at = kv_at, v_at = kv_at + T::K_RING * T::TILE;

    if (warp == 0 || warp == 11) {
        // ---- copies
        const bool of_k = warp == 0;
        const int ring = of_k ? T::K_RING : T::V_RING, first_full = of_k ? T::K_FULL : T::V_FULL, first_empty = of_k ? T::K_EMPTY : T::V_EMPTY;
        const CUtensorMap* map = of_k ? &map_k : &map_v;
        int page = page_of(0), next_page = page_of(1);
        if (of_k && lane == 0) {
            mbar_arrive_expect(bar(T::Q_FULL), (uint32_t)(tile_rows * HD * 2));
#pragma unroll
            for (int h = 0; h < HD / 64; ++h)
                tma_load_3d(q_at + h * TC_HALF, &map_q, 64 * h, p.kv_head * heads, p.token0 + p.row0 / heads, bar(T::Q_FULL));
        }
        __syncwarp();
        for (int j = 0; j < blocks; ++j) {
            const int slot = j % ring, after = page_of(j + 2);
            if (j >= ring) {
                const int ready = lane == 0 ? (int)mbar_wait(bar(first_empty + slot), (j / ring - 1) & 1u, abort_flag, status, 1) : 1;
                if (__shfl_sync(0xffffffffu, ready, 0) == 0) break;
            }
            if (lane == 0) mbar_arrive_expect(bar(first_full + slot), T::TILE);
            __syncwarp();
            if (lane < pages_per_block)         // a page that is none: a coordinate that reads zeros
#pragma unroll
                for (int h = 0; h < HD / 64; ++h)
                    tma_load_4d((of_k ? k_at : v_at) + slot * T::TILE + h * TC_HALF + (uint32_t)(lane * a.page_size * 128), map, 64 * h, 0,
                                p.kv_head, (unsigned)page < (unsigned)a.pages ? page : -1, bar(first_full + slot));
            page = next_page;
            next_page = after;
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- S = Q K^T of every block
        if (lane == 0 && mbar_wait(bar(T::Q_FULL), 0, abort_flag, status, 8)) {
            constexpr uint32_t idesc = instruction_descriptor_bf16(TC_ROWS, TC_KEYS, false);
            for (int j = 0; j < blocks; ++j) {
                const uint32_t b = j & 1u, n = j / 2, slot = j % T::K_RING;
                if (!mbar_wait(bar(T::K_FULL + slot), (j / T::K_RING) & 1u, abort_flag, status, 3)) break;
                // S of the group is also where its P lies: the product that read P of the block before must have finished
                if (n > 0 && !mbar_wait(bar(T::P_READ + b), (n - 1) & 1u, abort_flag, status, 4)) break;
                tc_fence_after_sync();
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint32_t half = (kk / 4) * TC_HALF, step = 2u * (kk % 4);
                    tc_mma(tmem_base + b * TC_KEYS, tile_descriptor(q_at + half) + step,
                           tile_descriptor(k_at + slot * T::TILE + half) + step, idesc, kk != 0);
                }
                tc_commit(bar(T::K_EMPTY + slot));
                tc_commit(bar(T::S_FULL + b));
            }
        }
        __syncwarp();
    } else if (warp == 10) {
        // ---- O += P V
        constexpr uint32_t idesc = instruction_descriptor_bf16(TC_ROWS, HD, true);
        auto all_wait = [&](int barrier, uint32_t parity, int code) -> bool {
            return __all_sync(0xffffffffu, mbar_wait(bar(barrier), parity, abort_flag, status, code));
        };
        for (int j = 0; j < blocks; ++j) {
            const uint32_t b = j & 1u, n = j / 2, slot = j % T::V_RING;
            if (!all_wait(T::V_FULL + slot, (j / T::V_RING) & 1u, 5)) break;
            const uint32_t v_tile = v_at + slot * T::TILE;
            const int have = p.range.end - p.range.first - j * TC_KEYS;         // keys of this block that are shared
            if (have < TC_KEYS) {
                const int end = min(TC_KEYS, (have + a.page_size - 1) / a.page_size * a.page_size);
                constexpr int WORDS = HD / 8;
                for (int i = have * WORDS + lane; i < end * WORDS; i += 32) {
                    const int row = i / WORDS, word = i % WORDS;
                    *reinterpret_cast<uint4*>(aligned + (v_tile - base) + word / 8 * TC_HALF + row * 128 + word % 8 * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_async_shared();
                __syncwarp();
            }
            if (!all_wait(T::P_FULL + b, n & 1u, 6)) break;
            if (lane == 0) {
                tc_fence_after_sync();
#pragma unroll
                for (int kk = 0; kk < TC_KEYS / 16; ++kk)
                    // 16 keys: 8 columns of P (two bfloat16 a column), two 1024-byte atoms of V
                    tc_mma_a_in_tmem(tmem_base + 2 * TC_KEYS + b * HD, tmem_base + b * TC_KEYS + kk * 8,
                                     tile_descriptor_mn_major(v_tile + kk * 2048, TC_HALF), idesc, !(n == 0 && kk == 0));
                tc_commit(bar(T::V_EMPTY + slot));
                tc_commit(bar(T::P_READ + b));
                if (j + 2 >= blocks) tc_commit(bar(T::O_LAST + b));
            }
            __syncwarp();
        }
    } else {
        // ---- softmax rows: group 0 = warps 2..5 takes the even blocks, group 1 = warps 6..9 the odd ones; a warp's number modulo 4
        // names the 32 lanes of tensor memory it may read
        const int quarter = warp & 3, group = (warp - 2) >> 2, row = quarter * 32 + lane;
        const uint32_t lane_address = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const uint32_t s_address = lane_address + group * TC_KEYS, o_address = lane_address + 2 * TC_KEYS + group * HD;
        auto warp_wait = [&](int barrier, uint32_t parity, int code) -> bool {
            return __all_sync(0xffffffffu, mbar_wait(bar(barrier), parity, abort_flag, status, code));
        };
        auto warp_arrive = [&](int barrier) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(barrier));
        };
        // where the row's result goes (-1: nowhere); asked for here, while the first tiles come in
        int place = -1;
        if (group == 0 && row < p.rows) {
            int head;
            const int token = token_of(a, p, row, head);
            if (takes_part(a, p, token)) place = (int)part_of(a, token, head, p.slot);
        }
        float reference = -INFINITY, l = 0.0f;  // what the exponentials of this row subtract (log2); the group's denominator
        bool alive = true;
        int next_page = page_of(group);
        for (int j = group; j < blocks && alive; j += 2) {
            const int have = p.range.end - p.range.first - j * TC_KEYS;
            const uint32_t pages = __ballot_sync(0xffffffffu, (unsigned)next_page < (unsigned)a.pages);
            next_page = page_of(j + 2);
            const bool full = have >= TC_KEYS && __popc(pages) == pages_per_block;
            // which of the 32 keys from c on are there
            auto seen_of = [&](int c) -> uint32_t {
                uint32_t bits = 0;
                if (a.page_size >= 32) bits = pages >> (c / a.page_size) & 1u ? ~0u : 0u;
                else
                    for (int i = 0; i < 32; i += a.page_size)
                        if (pages >> ((c + i) / a.page_size) & 1u) bits |= ((1u << a.page_size) - 1u) << i;
                const int n = have - c;
                return bits & (n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u);
            };
            if (!warp_wait(T::S_FULL + group, (j / 2) & 1u, 10)) { alive = false; break; }
            tc_fence_after_sync();
            // the row's 128 scores, once: the maximum, then the exponentials
            uint32_t v[TC_KEYS];
#pragma unroll
            for (int c = 0; c < TC_KEYS; c += 32) tmem_load_32(s_address + c, v + c);
            tmem_load_wait();
            if (!full)
#pragma unroll
                for (int c = 0; c < TC_KEYS; c += 32) {
                    const uint32_t seen = seen_of(c);
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(seen >> e & 1u)) v[c + e] = 0xff800000u;          // -inf: its exponential is 0
                }
            float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < TC_KEYS; ++e) part[e & 3] = fmaxf(part[e & 3], __uint_as_float(v[e]));
            // (the scale is positive)
            const float block_max = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) * a.scale_log2;
            const bool moves = block_max > reference + TC_RESCALE || (reference == -INFINITY && block_max > -INFINITY);
            float factor = 1.0f;
            if (moves) {
                factor = exp2_unit(reference - block_max);                      // 0 for a row that had seen no key
                reference = block_max;
                l *= factor;
            }
            const float subtract = reference == -INFINITY ? 0.0f : reference;
            float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < TC_KEYS; c += 32) {
                uint32_t packed[16];
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float w0 = exp2_unit(fmaf(__uint_as_float(v[c + e]), a.scale_log2, -subtract));
                    const float w1 = exp2_unit(fmaf(__uint_as_float(v[c + e + 1]), a.scale_log2, -subtract));
                    sums[e & 3] += w0;
                    sums[(e & 3) + 1] += w1;
                    packed[e / 2] = pack_bf16x2(w0, w1);
                }
                tmem_store_16(s_address + c / 2, packed);                       // P over the columns of S
            }
            l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
            // S of this block is there, so the product into this group's O before it has finished: O may be scaled
            if (j >= 2 && __any_sync(0xffffffffu, moves)) {
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t o[32];
                    tmem_load_32(o_address + c, o);
                    tmem_load_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
                    tmem_store_32(o_address + c, o);
                }
            }
            tmem_store_wait();
            tc_fence_before_sync();
            warp_arrive(T::P_FULL + group);
        }
        // ---- the rows' results.  O goes out through shared memory (that of the keys and values, of which all are consumed), so that a
        // warp stores whole rows; 16-byte word w of row r lies in place w ^ (r % 32, or % 16 for 64 values).
        constexpr int WORDS = HD / 4;
        const bool second = blocks > 1;         // else the second group had no block, and its O holds nothing
        int* places = reinterpret_cast<int*>(exchange + TC_ROWS * 2);
        uint4* staged = reinterpret_cast<uint4*>(aligned + T::TILE);
        static_assert(TC_ROWS * HD * 4 <= (T::K_RING + T::V_RING) * T::TILE, "room for the results");
        if (alive) alive = warp_wait(T::O_LAST, 0, 13);
        if (alive && second) alive = warp_wait(T::O_LAST + 1, 0, 13);
        if (group == 1) {
            exchange[row * 2] = reference;
            exchange[row * 2 + 1] = l;
            tc_fence_before_sync();
            if (alive) warp_arrive(T::SECOND_DONE);
        } else {
            if (alive) alive = warp_wait(T::SECOND_DONE, 0, 17);
            tc_fence_after_sync();
            const float other = alive ? exchange[row * 2] : -INFINITY, other_l = alive ? exchange[row * 2 + 1] : 0.0f;
            const float top = fmaxf(reference, other);
            const float mine = reference == -INFINITY ? 0.0f : exp2_unit(reference - top);
            const float theirs = other == -INFINITY ? 0.0f : exp2_unit(other - top);
            places[row] = alive ? place : -1;
            if (alive && place >= 0) *reinterpret_cast<float2*>(a.part_ml + (int64_t)place * 2) = make_float2(top, l * mine + other_l * theirs);
            if (alive)
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t x[32], y[32];
                    tmem_load_32(o_address + c, x);
                    if (second) tmem_load_32(o_address + HD + c, y);
                    tmem_load_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        float f = __uint_as_float(x[e]) * mine;
                        if (second) f = fmaf(__uint_as_float(y[e]), theirs, f);
                        x[e] = __float_as_uint(f);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        staged[row * WORDS + (((c + e) / 4) ^ (row % WORDS))] = make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                }
        }
        asm volatile("bar.sync 1, 256;\n" ::: "memory");                        // the softmax warps
        for (int r = warp - 2; r < TC_ROWS; r += 8) {
            const int64_t at = places[r];
            if (at >= 0 && lane < WORDS) *reinterpret_cast<uint4*>(a.part_o + at * HD + lane * 4) = staged[r * WORDS + (lane ^ (r % WORDS))];
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        // copies or products may still be in flight towards this CTA's memory: give them time
        const long long started = clock64();
        while (clock64() - started < 400000) __nanosleep(1000);
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_free(tmem_base, TC_COLUMNS);
    }
}

inline bool tc_takes(int head_dim, int heads, int page_size) {
    return (head_dim == 64 || head_dim == 128) && heads <= TC_ROWS && page_size >= 8 && page_size <= TC_KEYS && (page_size & (page_size - 1)) == 0;
}

template <int HD> int launch_shared_tc(const Attend& a, long long items, int tile_tokens, int pdl, cudaStream_t stream) {
    CUtensorMap map_q, map_k, map_v;
    {
        const int heads = a.num_q / a.num_kv;
        const cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)a.num_q, (cuuint64_t)a.tokens};
        const cuuint64_t strides[2] = {HD * 2, (cuuint64_t)a.q_stride * 2};
        const cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tile_tokens};
        if (!tvb_make_map(&map_q, a.q, 3, dims, strides, box)) return (int)cudaErrorNotSupported;
    }
    const cuuint64_t dims[4] = {(cuuint64_t)HD, (cuuint64_t)a.page_size, (cuuint64_t)a.num_kv, (cuuint64_t)a.pages};
    const cuuint64_t strides[3] = {HD * 2, (cuuint64_t)a.page_size * HD * 2, (cuuint64_t)a.num_kv * a.page_size * HD * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)a.page_size, 1, 1};
    if (!tvb_make_map(&map_k, a.keys, 4, dims, strides, box) || !tvb_make_map(&map_v, a.values, 4, dims, strides, box))
        return (int)cudaErrorNotSupported;
    auto kernel = attend_shared_tc_kernel<HD>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShared<HD>::BYTES);
    if (e != cudaSuccess) return (int)e;
    TvbLaunch at(dim3((unsigned)items), dim3(TC_THREADS), TcShared<HD>::BYTES, stream, pdl);
    const cudaError_t launched = cudaLaunchKernelEx(&at.config, kernel, map_q, map_k, map_v, a, tile_tokens);
    return launched == cudaSuccess ? tvb_last_error() : (int)launched;
}
