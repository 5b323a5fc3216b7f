// ff_attend_rows.hip - attention of many query rows (a tree or a chunk of new tokens, times the heads of a kv head) over the paged
// cache, for 16-bit T.
//
// With more than 128 rows the products, not the cache's bytes, are what costs, so keys and values are made ready ONCE for all
// waves of a workgroup: 64 keys at a time are loaded, turned into T (codes) and laid in shared memory row by row; two buffers, the
// next 64 keys in flight in registers meanwhile (and the page numbers of those behind them), one barrier a step.  A wave owns 32
// rows: S^T = K Q^T leaves a lane with 16 of 32 keys of ONE row (its other half in lane + 32), which is also what O^T = V^T P^T
// wants, so the weights never leave the registers; V^T comes out of shared memory by the transposing reads (ds_read_b64_tr_b16:
// 16 lanes that point at 4 rows of 16 channels get one channel of 4 rows each).  At 32 rows a wave a product is fed by one
// read of 16 bytes a lane, which shared memory keeps up with; what a step costs is its products, its softmax (an exponential a score, at
// a quarter of the rate) and the barrier, which the two waves of a SIMD overlap only in part.  28 / 4 heads of 128, 4 sequences, 61 new
// tokens in bf16, 1 to 52 steps of 64 keys a workgroup: 15 us (the way to the first keys and out: lengths, pages, Q, partial rows) and 2.35 us
// a step, of which the products are 1.5 at the rate of a large one; the join takes 8.  Over up to 13 474 keys: 47 us + 8.  A higher priority
// for one wave of each SIMD changed nothing (50 to 56 us with and without).
#include <atomic>

#include "ff_attend.h"

namespace ff {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kRowsKeys = 64;                 // keys of a step

template <int DT> __device__ inline f32x16 mma32(const uint4& a, const uint4& b, f32x16 c) {
    if constexpr (DT == FF_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Rows lie in shared memory without padding; the 16-byte pieces of a row are exchanged by this mask (piece ^ turn) so that 16 rows at
// one piece (the reads of K), 4 rows at 4 neighbouring pieces (the transposing reads of V, the writes) meet 64 different banks: the
// row's number within the rows that share a bank line, its bits reversed.
template <int DH> __device__ inline uint32_t turn(uint32_t row) {
    constexpr uint32_t kPieces = DH / 8 < 16 ? DH / 8 : 16, kBits = kPieces == 4 ? 2 : kPieces == 8 ? 3 : 4;
    return __builtin_bitreverse32((row / (16 / kPieces)) & (kPieces - 1)) >> (32 - kBits);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// 16 channels x 4 rows: lane i of 16 points at channels 4 (i % 4) of row i / 4 and gets channel i of the rows
__device__ inline uint2 read_turned(const char* p) { return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p))); }

template <int DT, int STORE, int DH, int NW>
__global__ __launch_bounds__(64 * NW, DH == 256 ? 1 : 2) void k_cache_attention_rows(const ff_cache_attention_t a, const AttPlan p) {
    constexpr int kThreads = 64 * NW, kSteps = DH / 16, kTiles = DH / 32;
    constexpr int kStride = DH * 2;                                                  // bytes of a row in shared memory
    constexpr int kBuf = 2 * kRowsKeys * kStride;                                    // keys, then values
    // a unit of the loading: 32 channels of one key or value
    constexpr int kUnits = 4 * DH, kMine = (kUnits + kThreads - 1) / kThreads, kWords = STORE == kStoreSame ? 16 : STORE == FF_STORE_E4M3 ? 8 : 4;
    constexpr int kRow = STORE == FF_STORE_E4M3 ? DH : STORE == FF_STORE_E2M1 ? DH / 2 : 2 * DH;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int s_odd;                     // a value of the keys from the new tokens on is NaN or infinite
    __shared__ int s_have[2][4];              // which 16 keys of a buffer have a place
    __shared__ uint64_t s_bits[2][32 * NW];   // which keys of a buffer a new token sees, from the first one on that not all see
    const ff_cache_t& c = a.cache;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5, col = lane & 31;
    const int n = (int)c.n, kv = (int)c.kv_heads;
    // workgroups that read the same keys for other rows are 8 apart: on the same XCD (they go round the eight), at the same time
    const int order = blockIdx.x >> 3, group = order % p.groups, which = (order / p.groups) * 8 + (blockIdx.x & 7);
    const int across = p.slots == 1 ? (int)c.B : p.slots, head = which / across, slot = which - head * across;
    if (head >= kv) return;
    const bool plain = plain_share(c, p);
    Share share = {p.slots == 1 ? slot : 0, p.slots == 1 ? 0 : slot, 1, 0};
    if (!plain && !share_of(c, p, slot, share)) return;
    const int b = share.b, split = share.split;
    const int32_t* table = c.table + (int64_t)b * c.table_width;
    int64_t base = (int64_t)split * kRowsKeys;
    if (tid == 0) s_odd = 0;

    // ---- unit u = tid + i kThreads: block x of key (u mod 2 DH) / (DH / 32), of the keys for u < 2 DH, else of the values
    uint32_t w[kMine][kWords], sc[kMine];
    int page[kMine], page_next[kMine];
    auto key_of = [&](int i) { return ((tid + i * kThreads) % (2 * DH)) / (DH / 32); };
    auto slot_of = [&](uint32_t at) {
        uint32_t slot = __umulhi(at >> 4, p.magic);
        return slot + ((at >> 4) - slot * p.page16 >= (uint32_t)p.page16);
    };
    auto look_up = [&](int64_t base) {           // the pages of a step, a step before its rows are loaded
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int64_t at = base + key_of(i);
            page_next[i] = at < c.table_width * c.page_size ? table[slot_of((uint32_t)at)] : -1;       // (looked at only when the rows are loaded)
        }
    };
    look_up(base);
    const int64_t start = c.start[b], end = keys_of(c, start);
    if (plain && p.slots > 1) share.used = max(1, min(p.want, blocks_of(c, p, b)));
    if (split >= share.used) return;
    if (p.slots > 1 && split == 0 && head == 0 && group == 0 && tid == 0) p.shares[b] = make_int2(share.first, share.used);

    // the wave's 32 rows of Q; a wave behind the group's last tile only loads
    const int tile = group * p.tiles + wave, row = tile * 32 + col;
    const bool works = wave < p.tiles && tile * 32 < p.R;
    const int token = row / p.G;
    // (up to 128 channels in shared memory, in the order of the products: 64 pieces a step, one a lane)
    constexpr bool kShared = DH <= 128;
    uint4 qf[kSteps];
    uint4* const qs = (uint4*)(lds + 2 * kBuf) + wave * kSteps * 64 + lane;
    {
        const char* src = (const char*)a.q + ((int64_t)b * a.q_batch + (int64_t)(head * p.G + row - token * p.G) * a.q_head + (int64_t)token * a.q_token) * 2;
#pragma unroll
        for (int x = 0; x < kSteps; ++x) qf[x] = make_uint4(0, 0, 0, 0);
        if (works && row < p.R) {
#pragma unroll
            for (int x = 0; x < kSteps; ++x) qf[x] = *(const uint4*)(src + (x * 16 + h * 8) * 2);
        }
    }
    f32x16 o[kTiles];
#pragma unroll
    for (int y = 0; y < kTiles; ++y)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[y][e] = 0.f;
    float m = kNone, l = 0.f;

    auto fetch = [&](int64_t base) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const uint32_t at = (uint32_t)(base + key_of(i));
            page[i] = base + key_of(i) < end && page_next[i] < c.n_pages ? page_next[i] : -1;
            const int u = tid + i * kThreads;
            if (kUnits % kThreads && u >= kUnits) continue;
            const int64_t row = page[i] < 0 ? 0 : ((int64_t)page[i] * kv + head) * c.page_size + (at - slot_of(at) * (uint32_t)c.page_size);   // (no place: any row, left out below)
            const int x = u % (DH / 32);
            const bool is_v = u >= 2 * DH;
            const char* src = (const char*)(is_v ? c.values : c.keys) + row * kRow;
            if constexpr (STORE == kStoreSame) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint4 v = ((const uint4*)src)[k * (DH / 32) + x];          // (16 bytes of neighbours side by side)
                    w[i][4 * k] = v.x; w[i][4 * k + 1] = v.y; w[i][4 * k + 2] = v.z; w[i][4 * k + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int k = 0; k < kWords / 4; ++k) {
                    const uint4 v = ((const uint4*)src)[x * (kWords / 4) + k];
                    w[i][4 * k] = v.x; w[i][4 * k + 1] = v.y; w[i][4 * k + 2] = v.z; w[i][4 * k + 3] = v.w;
                }
                sc[i] = (is_v ? c.value_scales : c.key_scales)[row * (DH / 32) + x];
            }
        }
    };
    auto deliver = [&](int buf, int64_t base) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int u = tid + i * kThreads;
            if (kUnits % kThreads && u >= kUnits) continue;
            const int key = key_of(i), x = u % (DH / 32);
            const bool is_v = u >= 2 * DH, in = page[i] >= 0;
            char* dst = lds + buf * kBuf + (is_v ? kRowsKeys * kStride : 0) + key * kStride;
            bool odd = false;
            constexpr uint32_t kExp = DT == FF_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t t[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (STORE == kStoreSame) t[e] = w[i][4 * k + e];
                    else t[e] = codes2<DT, STORE>(w[i][(4 * k + e) / (STORE == FF_STORE_E4M3 ? 2 : 4)], __uint_as_float(sc[i] << 23), (4 * k + e) % (STORE == FF_STORE_E4M3 ? 2 : 4));
                    t[e] = in ? t[e] : 0;                            // (what nobody sees may be anything: zeros stand in)
                    if (is_v && base + kRowsKeys > start) {
                        // new tokens do not all see each other, and 0 x NaN is NaN: a NaN or infinity among these keys' values stays
                        // out of the products and is added at the end to the rows that see it
                        if ((t[e] & kExp) == kExp) t[e] &= 0xffff0000u, odd = true;
                        if ((t[e] & (kExp << 16)) == (kExp << 16)) t[e] &= 0xffffu, odd = true;
                    }
                }
                *(uint4*)(dst + ((uint32_t)(STORE == kStoreSame ? k * (DH / 32) + x : 4 * x + k) ^ turn<DH>(key)) * 16) = make_uint4(t[0], t[1], t[2], t[3]);
            }
            if (odd) s_odd = 1;
            if (!is_v && x == 0 && (key & 15) == 0) s_have[buf][key >> 4] = in;       // (a page holds whole sixteens)
        }
    };
    // ---- what the new tokens of this workgroup see of a step that not all of them see whole: a bit a key, a lane of a wave asks
    const int token0 = group * p.tiles * 32 / p.G, tokens = min((min((group + 1) * p.tiles * 32, p.R) - 1) / p.G, n - 1) - token0 + 1;
    const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.mask_batch : nullptr;
    auto look_at = [&](int buf, int64_t base) {
        if (base + kRowsKeys <= start) return;
        const int64_t fresh = base + lane - start;
        const int fresh_in = (int)min(max(fresh, (int64_t)0), (int64_t)n - 1);
        for (int t = wave; t < tokens; t += 4 * NW) {
            bool sees[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int own = token0 + min(t + k * NW, tokens - 1);
                sees[k] = mask ? mask[(int64_t)own * n + fresh_in] != 0 : fresh_in <= own;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint64_t bits = __ballot(fresh < 0 || (sees[k] && base + lane < end));
                if (lane == 0 && t + k * NW < tokens) s_bits[buf][t + k * NW] = bits;
            }
        }
    };

    // where this lane's pieces lie in a row (bytes, before the step's own are exchanged in): keys `col`, values 4 h + i and 8 behind
    const uint32_t key_piece = ((uint32_t)h ^ turn<DH>(col)) * 16;
    const uint32_t value_at = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1), value_row = 4 * h + ((lane & 15) >> 2);
    const uint32_t value_piece0 = (value_at ^ turn<DH>(value_row)) * 16, value_piece1 = (value_at ^ turn<DH>(value_row + 8)) * 16;
    const int64_t stride = (int64_t)share.used * kRowsKeys;
    if (base < end) {
        fetch(base);
        look_up(base + stride);
    }
    if constexpr (kShared) {
#pragma unroll
        for (int x = 0; x < kSteps; ++x) qs[x * 64] = make_uint4(qf[x].x ^ p.flip, qf[x].y ^ p.flip, qf[x].z ^ p.flip, qf[x].w ^ p.flip);      // (read by the same lane alone)
    } else {
#pragma unroll
        for (int x = 0; x < kSteps; ++x) qf[x] = make_uint4(qf[x].x ^ p.flip, qf[x].y ^ p.flip, qf[x].z ^ p.flip, qf[x].w ^ p.flip);
    }
    __syncthreads();                           // (s_odd is clear)
    if (base < end) {
        deliver(0, base);
        look_at(0, base);
    }
    __syncthreads();
    for (int buf = 0; base < end; buf ^= 1, base += stride) {
        const bool more = base + stride < end;
        if (more) {
            fetch(base + stride);
            look_up(base + 2 * stride);
        }
        const uint32_t have = uniform(s_have[buf][0] | s_have[buf][1] << 1 | s_have[buf][2] << 2 | s_have[buf][3] << 3);
        if (works) {
            const char* keys = lds + buf * kBuf + col * kStride;
            const char* values = lds + buf * kBuf + (kRowsKeys + 4 * h + ((lane & 15) >> 2)) * kStride + (lane & 1) * 8;
            uint2 vf[2][kTiles][2];
            f32x16 s[2];
            auto load_values = [&](int sub) {                     // of 16 keys: 4 h + 0..3 and 8 behind
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int y = 0; y < kTiles; ++y)
#pragma unroll
                        for (int z = 0; z < 2; ++z)
                            vf[k][y][z] = read_turned(values + (sub * 32 + 16 * k + 8 * z) * kStride + ((uint32_t)(y * 64) ^ (z ? value_piece1 : value_piece0)));
            };
            // both halves of the step at once: two independent chains of products, Q read once for them
            auto score = [&]() {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[0][e] = s[1][e] = 0.f;
#pragma unroll
                for (int x = 0; x < kSteps; ++x) {
                    const char* at = keys + ((uint32_t)(x * 32) ^ key_piece);
                    const uint4 k0 = *(const uint4*)at, k1 = *(const uint4*)(at + 32 * kStride), qx = kShared ? qs[x * 64] : qf[x];
                    s[0] = mma32<DT>(k0, qx, s[0]);
                    s[1] = mma32<DT>(k1, qx, s[1]);
                }
            };
            uint4 pf[2];
            auto weigh = [&](int sub) {
                f32x16& w = s[sub];
                if (((have >> (2 * sub)) & 3u) != 3u || base + sub * 32 + 32 > start) {               // not every row sees every key
                    uint32_t sees = base + kRowsKeys > start ? (uint32_t)(s_bits[buf][min(token, n - 1) - token0] >> (sub * 32)) : ~0u;
                    if (!((have >> (2 * sub)) & 1u)) sees &= 0xffff0000u;
                    if (!((have >> (2 * sub)) & 2u)) sees &= 0x0000ffffu;
                    sees >>= 4 * h;
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (!((sees >> (8 * (e >> 2) + (e & 3))) & 1u)) w[e] = kNone;
                }
                float top = kNone;
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, w[e]);
                top *= p.scale2;
                const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                top = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
                // (the maximum moves only when a row passes it by 2^8, as in ff_attend.hip)
                if (__any(top > m + 8.f)) {
                    const float up = fmaxf(m, top), down = __builtin_amdgcn_exp2f(m - (up == kNone ? 0.f : up));
                    m = up;
                    l *= down;
#pragma unroll
                    for (int y = 0; y < kTiles; ++y) o[y] *= down;
                }
                const float zero = (m == kNone ? 0.f : m) - kLift<DT>;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(fmaf(w[e], p.scale2, -zero));
                    sum += w[e];
                }
                l += sum;
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    pf[k] = make_uint4(pack2<DT>(w[8 * k], w[8 * k + 1]), pack2<DT>(w[8 * k + 2], w[8 * k + 3]),
                                       pack2<DT>(w[8 * k + 4], w[8 * k + 5]), pack2<DT>(w[8 * k + 6], w[8 * k + 7]));
            };
            auto gather = [&]() {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int y = 0; y < kTiles; ++y)
                        o[y] = mma32<DT>(make_uint4(vf[k][y][0].x, vf[k][y][0].y, vf[k][y][1].x, vf[k][y][1].y), pf[k], o[y]);
            };
            // values are read while the weights that meet them are made, and the first half's products run under the second half's
            // softmax; the barriers keep the compiler from undoing that.  (256 channels: the outputs and Q leave no registers for it - 64 new
            // tokens of 28 / 4 heads over 8 x 20 000 keys 920 us spilling, 700 us with the values read behind the weights)
            score();
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kShared) load_values(0);
            __builtin_amdgcn_sched_barrier(0);
            weigh(0);
            if constexpr (!kShared) load_values(0);
            gather();
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kShared) load_values(1);
            __builtin_amdgcn_sched_barrier(0);
            weigh(1);
            if constexpr (!kShared) load_values(1);
            gather();
        }
        if (more) {
            deliver(buf ^ 1, base + stride);
            look_at(buf ^ 1, base + stride);
        }
        __syncthreads();
    }

    if (!works) return;
    if (s_odd && row < p.R) {
        // rare: the values left out above, to the rows that see them (their weight is positive: infinities and NaN stay what they are)
        for (int64_t first = ((int64_t)split + max((int64_t)0, start / kRowsKeys - split + share.used - 1) / share.used * share.used) * kRowsKeys; first < end; first += stride) {
#pragma unroll 1
            for (int k = 0; k < kRowsKeys; ++k) {
                const int64_t r = row_of_16(c, p, table, head, first + (k & 48), end);
                const int64_t fresh = first + k - start;
                if (r < 0 || first + k >= end) continue;
                if (fresh >= 0 && !(mask ? mask[(int64_t)token * n + fresh] != 0 : fresh <= token)) continue;
#pragma unroll
                for (int g = 0; g < DH / 8; ++g) {
                    float f[4];
                    fetch4<DT, STORE>(c.values, c.value_scales, r + (k & 15), DH, 2 * g + h, f);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = Act<DT>::rnd(f[e]);
                        if (!(fabsf(v) < __builtin_inff())) o[g >> 2][4 * (g & 3) + e] += v;
                    }
                }
            }
        }
    }
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    const float sum = __uint_as_float(both[0]) + __uint_as_float(both[1]);
    // channel of o[y][e]: 32 y + 8 (e / 4) + 4 h + e % 4
    if (p.slots > 1) {
        // through the wave's share of the shared memory (nobody reads it any more), pieces of 16 bytes exchanged by the row as above, so
        // that the partial rows go out whole: 16 bytes of 32 rows at a time took 9 us of 50 for 27 MB
        f32x4* mine = (f32x4*)lds + wave * 8 * DH;
#pragma unroll
        for (int y = 0; y < kTiles; ++y)
#pragma unroll
            for (int g = 0; g < 4; ++g) mine[col * (DH / 4) + ((8 * y + 2 * g + h) ^ (col % (DH / 4)))] = f32x4{o[y][4 * g], o[y][4 * g + 1], o[y][4 * g + 2], o[y][4 * g + 3]};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 4
        for (int x = 0; x < DH / 8; ++x) {
            const int i = x * 64 + lane, r = i / (DH / 4), piece = i % (DH / 4), to = tile * 32 + r;
            if (to < p.R) *(f32x4*)(p.part + (((int64_t)head * p.R + to) * p.slots + slot) * DH + piece * 4) = mine[r * (DH / 4) + (piece ^ (r % (DH / 4)))];
        }
        if (row < p.R && h == 0) ((float2*)(p.part + p.part_rows * DH))[((int64_t)head * p.R + row) * p.slots + slot] = make_float2(m, sum);
    } else if (row < p.R) {
        char* out = (char*)a.out + ((int64_t)b * a.o_batch + (int64_t)(head * p.G + row - token * p.G) * a.o_head + (int64_t)token * a.o_token) * 2;
#pragma unroll
        for (int y = 0; y < kTiles; ++y)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                write_out4<DT>(out, 32 * y + 8 * g + 4 * h, f32x4{o[y][4 * g], o[y][4 * g + 1], o[y][4 * g + 2], o[y][4 * g + 3]}, sum);
    }
}

template <int DT, int STORE, int DH, int NW>
static int launch_rows_of(const ff_cache_attention_t* a, const AttPlan& p) {
    constexpr int kBytes = 4 * kRowsKeys * DH * 2 + (DH <= 128 ? NW * 64 * DH : 0);           // two buffers, and Q
    static_assert(kBytes + 2 * 32 * NW * 8 + 64 <= 160 * 1024, "two buffers, Q and the rest fit the shared memory of a CU");
    static std::atomic<bool> ready[kMaxDevices];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) dev = -1;
    if (dev < 0 || !ready[dev].load(std::memory_order_acquire)) {
        const hipError_t e = hipFuncSetAttribute((const void*)k_cache_attention_rows<DT, STORE, DH, NW>, hipFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        if (e != hipSuccess) return (int)e;
        if (dev >= 0) ready[dev].store(true, std::memory_order_release);
    }
    const ff_cache_t& c = a->cache;
    const int64_t across = c.kv_heads * (p.slots == 1 ? c.B : p.slots);
    if ((across + 7) / 8 * 8 * p.groups > 0x7fffffff) return FF_ERR_UNSUPPORTED;
    const dim3 grid((uint32_t)((across + 7) / 8 * 8 * p.groups));
    k_cache_attention_rows<DT, STORE, DH, NW><<<grid, 64 * NW, kBytes, (hipStream_t)a->stream>>>(*a, p);
    return (int)hipGetLastError();
}
template <int DT, int STORE>
static int launch_rows_store(const ff_cache_attention_t* a, const AttPlan& p) {
    switch (a->cache.dh) {
        case 32: return launch_rows_of<DT, STORE, 32, 8>(a, p);
        case 64: return launch_rows_of<DT, STORE, 64, 8>(a, p);
        case 128: return launch_rows_of<DT, STORE, 128, 8>(a, p);
        default: return launch_rows_of<DT, STORE, 256, 4>(a, p);
    }
}
template <int DT> int launch_attention_rows(const ff_cache_attention_t* a, const AttPlan& p) {
    if (a->cache.store == FF_STORE_E4M3) return launch_rows_store<DT, FF_STORE_E4M3>(a, p);
    if (a->cache.store == FF_STORE_E2M1) return launch_rows_store<DT, FF_STORE_E2M1>(a, p);
    return launch_rows_store<DT, kStoreSame>(a, p);
}
template int launch_attention_rows<FF_BF16>(const ff_cache_attention_t*, const AttPlan&);
template int launch_attention_rows<FF_F16>(const ff_cache_attention_t*, const AttPlan&);

}  // namespace ff
