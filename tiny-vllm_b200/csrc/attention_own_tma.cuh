// A token's own keys for bfloat16 and pages of 8 to 128 tokens (a power of two), included by attention_shared.cu: as
// attend_own_bf16_kernel, with K and V brought in by tensor-map copies.  A page's keys of one kv head lie together, so a tile of
// 32 keys is a handful of copies that the lanes of a warp of their own issue, where cp.async took a dozen instructions of every thread
// for them; the warps follow one another by mbarriers alone (a full and an empty one a tile), not by barriers of the CTA.
//
// Tiles are those of the positions (32 from 0 on), so that boxes lie on the 1024 bytes of the 128-byte swizzle; keys of a tile that
// are not the piece's get no weight, and their values are zeroed in the fragments (what lies there is of no account).
//
// Bound by reading keys and values, and by the tiles of the longest piece, one after another.  Whole calls, us with this kernel / with
// attend_own_bf16_kernel: 60 tokens with up to 431 keys behind 6,144, 32 / 8 heads of size 128, 28.2 / 33.0; three groups of 13 with up
// to 777 behind 2,896, 64 / 8 heads, 31.3 / 38.9; 2 tokens with 231 keys, 16 / 8 heads, alone 6.9 / 9.8, which is the chain of
// position, page number, eight tiles and the meeting of the warps.  Rings of four and six tiles in as many CTAs as then fit: 28.7, 33.0.
#pragma once

template <int D> struct OwnTma {
    static constexpr int KEYS = 32, RING = 3;
    static constexpr int HALF = KEYS * 128, TILE = D / 64 * HALF;               // bytes of a K or V tile
    static constexpr int Q_PITCH = D + 8, Q_BYTES = 16 * Q_PITCH * 2;
    static constexpr int RING_BYTES = 2 * RING * TILE, END_BYTES = Ends<D, 16>::FLOATS * 4;
    static constexpr int BYTES = 1024 + (RING_BYTES > END_BYTES ? RING_BYTES : END_BYTES) + Q_BYTES + 2 * RING * 8 + 16;
    static constexpr int CTAS = D == 64 ? 4 : D == 128 ? 3 : 1;                 // on an SM (one more: 1 us slower, with fewer registers)
    static constexpr bool Q_HELD = D <= 128;                                    // q fragments in registers (else read again a tile)
    static constexpr int THREADS_ALL = THREADS + 32;                            // four warps of products, one of copies
};

// SHARED: a piece of a group's shared keys instead, for 16 of the group's query rows.
template <int D, bool SHARED>
__global__ void __launch_bounds__(OwnTma<D>::THREADS_ALL, OwnTma<D>::CTAS)
attend_own_tma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Attend a) {
    using S = OwnTma<D>;
    extern __shared__ uint8_t raw_own[];
    const uint32_t base = (smem_address(raw_own) + 1023u) & ~1023u;
    uint8_t* ring = raw_own + (base - smem_address(raw_own));                   // [RING][K, V][D / 64][KEYS][128 bytes]
    constexpr int RING_AREA = S::RING_BYTES > S::END_BYTES ? S::RING_BYTES : S::END_BYTES;
    bf16* q_s = reinterpret_cast<bf16*>(ring + RING_AREA);
    const uint32_t bars = base + RING_AREA + S::Q_BYTES;
    auto full = [&](int slot) { return bars + 8u * slot; };
    auto empty = [&](int slot) { return bars + 8u * (S::RING + slot); };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(ring + RING_AREA + S::Q_BYTES + 2 * S::RING * 8);
    int* status = &tvb_attention_shared_status_word;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    if (tid == 0) {
        for (int i = 0; i < S::RING; ++i) {
            mbar_init(full(i), 1);
            mbar_init(empty(i), WARPS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
    }
    Piece p;
    uint32_t rows = ~0u;
    if constexpr (SHARED) {
        pdl_wait();
        pdl_launch_dependents();
        if (!find_shared_piece(a, 16, p)) return;
        int head;
        rows = __ballot_sync(0xffffffffu, lane < p.rows && takes_part(a, p, token_of(a, p, min(lane, p.rows - 1), head)));
    } else {
        start_own(a);
        if (!find_own_piece(a, 16, p)) {
            store_zeros<bf16, D>(a, p);
            end_own(a);
            return;
        }
    }
    const int key0 = p.range.first / S::KEYS * S::KEYS;                          // of the first tile
    const int tiles = (p.range.end - key0 + S::KEYS - 1) / S::KEYS;
    const int box = min(a.page_size, S::KEYS), boxes = S::KEYS / box;            // keys of a copy; copies of a tile of 64 values
    const int shift = 31 - __clz(a.page_size);
    // a page's number as it stands in the table (-1 past the piece); whether it is one is asked where it is used, since the warp
    // would wait for the load there and then
    auto page_at = [&](int key) -> int { return key < p.range.end ? __ldcg(p.table + (key >> shift)) : -1; };
    if (warp == WARPS) {
        // ---- copies: the one that this lane makes of every tile is keys' or values', which 64 values, which keys
        const int half = (lane >> 1) % (D / 64), part = lane / (2 * (D / 64));
        const bool copies = part < boxes;
        const uint32_t to = base + (lane & 1) * S::TILE + half * S::HALF + part * box * 128;
        const CUtensorMap* map = lane & 1 ? &map_v : &map_k;
        int key = key0 + part * box, page = copies ? page_at(key) : -1, next_page = copies ? page_at(key + S::KEYS) : -1;
        __syncthreads();                        // (the others' q)
        for (int tile = 0; tile < tiles; ++tile, key += S::KEYS) {
            const int slot = tile % S::RING, after = copies ? page_at(key + 2 * S::KEYS) : -1;
            if (tile >= S::RING && !__all_sync(0xffffffffu, mbar_wait(empty(slot), (tile / S::RING - 1) & 1u, abort_flag, status, 21))) break;
            if (lane == 0) mbar_arrive_expect(full(slot), 2 * S::TILE);
            __syncwarp();
            if (copies)                         // a page that is none: a coordinate that reads zeros
                tma_load_4d(to + 2 * slot * S::TILE, map, 64 * half, key & (a.page_size - 1), p.kv_head,
                            (unsigned)page < (unsigned)a.pages ? page : -1, full(slot));
            page = next_page;
            next_page = after;
        }
    }
    // the page of this warp's eight keys of the next tile
    int my_page = warp < WARPS ? page_at(key0 + warp * 8) : -1;
    if (warp < WARPS) {
        for (int i = tid; i < 16 * (D / 8); i += THREADS) {
            const int r = i / (D / 8), word = i % (D / 8);
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < p.rows) {
                int head;
                const int token = token_of(a, p, r, head);
                v = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.q) + token * a.q_stride + head * D + word * 8));
            }
            *reinterpret_cast<uint4*>(q_s + r * S::Q_PITCH + word * 8) = v;
        }
        __syncthreads();                        // the barriers are set up, q is there
    }
    const bf16* q_rows = q_s + (lane & 15) * S::Q_PITCH + (lane >> 4) * 8;
    uint32_t q_frag[S::Q_HELD ? D / 16 : 1][4];
    if constexpr (S::Q_HELD)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) ldmatrix_x4(q_frag[ks], q_rows + ks * 16);
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    // where this lane reads the eight rows of its warp: row lane % 8, 16-byte words in pairs of 32 values, swizzled by the row
    const uint32_t row_at = (uint32_t)(warp * 8 + (lane & 7)) * 128, word = lane >> 3, swizzle = lane & 7;
    bool alive = true;

    for (int tile = 0; warp < WARPS && tile < tiles; ++tile) {
        const int slot = tile % S::RING, at = key0 + tile * S::KEYS + warp * 8;
        // which of the warp's keys are the piece's
        uint32_t there = 0;
        if ((unsigned)my_page < (unsigned)a.pages) {
            const int lo = max(p.range.first - at, 0), hi = min(p.range.end - at, 8);
            there = lo < hi ? ((1u << hi) - 1u) & ~((1u << lo) - 1u) : 0u;
        }
        my_page = page_at(at + S::KEYS);
        alive = __all_sync(0xffffffffu, mbar_wait(full(slot), (tile / S::RING) & 1u, abort_flag, status, 20));
        if (!alive) break;
        const uint32_t k_at = base + 2 * slot * S::TILE + row_at, v_at = k_at + S::TILE;
        float s[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
            uint32_t b[4];
            ldmatrix_x4_at(b, k_at + ks / 2 * S::HALF + ((((ks & 1) * 4 + word) ^ swizzle) << 4));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t q_now[4];
                if constexpr (!S::Q_HELD) ldmatrix_x4(q_now, q_rows + (2 * ks + h) * 16);
                const uint32_t (&q4)[4] = S::Q_HELD ? q_frag[S::Q_HELD ? 2 * ks + h : 0] : q_now;
                mma_16816(s[h], q4, b[2 * h], b[2 * h + 1]);
            }
        }
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
        // values of keys that are not seen: zeros, so that no 0 * NaN comes in
        const uint32_t keep = (there >> (2 * t4) & 1 ? 0xffffu : 0u) | (there >> (2 * t4 + 1) & 1 ? 0xffff0000u : 0u);
#pragma unroll
        for (int dp = 0; dp < D / 32; ++dp) {
            uint32_t b[4];
            ldmatrix_x4_trans_at(b, v_at + dp / 2 * S::HALF + ((((dp & 1) * 4 + word) ^ swizzle) << 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) mma_1688(o[4 * dp + j], w_lo, w_hi, b[j] & keep);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(slot));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    __syncthreads();
    if (*abort_flag) {
        // copies may still be in flight towards this CTA's memory: give them time
        const long long started = clock64();
        while (clock64() - started < 400000) __nanosleep(1000);
    }
    const Ends<D, 16> ends(reinterpret_cast<float*>(ring));                     // over the tiles
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h, row = warp * 16 + r;
        if (r >= p.rows || warp >= WARPS) continue;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(ends.o + row * Ends<D, 16>::PITCH + n * 8 + 2 * t4) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        if (t4 == 0) *reinterpret_cast<float2*>(ends.ml + 2 * row) = make_float2(m[h], l[h]);
    }
    finish_own<bf16, D, 16>(a, p, ends, rows);
    if constexpr (!SHARED) end_own(a);
}

inline bool own_tma_takes(int page_size) { return page_size >= 8 && page_size <= 128 && (page_size & (page_size - 1)) == 0; }

template <int D, bool SHARED> int launch_own_tma(const Attend& a, long long items, int pdl, cudaStream_t stream) {
    CUtensorMap map_k, map_v;
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)a.page_size, (cuuint64_t)a.num_kv, (cuuint64_t)a.pages};
    const cuuint64_t strides[3] = {D * 2, (cuuint64_t)a.page_size * D * 2, (cuuint64_t)a.num_kv * a.page_size * D * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)(a.page_size < OwnTma<D>::KEYS ? a.page_size : OwnTma<D>::KEYS), 1, 1};
    if (!tvb_make_map(&map_k, a.keys, 4, dims, strides, box) || !tvb_make_map(&map_v, a.values, 4, dims, strides, box))
        return (int)cudaErrorNotSupported;
    auto kernel = attend_own_tma_kernel<D, SHARED>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, OwnTma<D>::BYTES);
    if (e != cudaSuccess) return (int)e;
    TvbLaunch at(dim3((unsigned)items), dim3(OwnTma<D>::THREADS_ALL), OwnTma<D>::BYTES, stream, pdl);
    const cudaError_t launched = cudaLaunchKernelEx(&at.config, kernel, map_k, map_v, a);
    return launched == cudaSuccess ? tvb_last_error() : (int)launched;
}
