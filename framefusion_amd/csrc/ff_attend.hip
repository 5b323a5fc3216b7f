// ff_attend.hip - attention of the new tokens of each sequence (one, a chunk, or a tree of drafted ones) over the paged cache.
//
// All query rows that share a kv head - n tokens times G heads - are one matrix of R = n G rows, so the cache is read once for
// all of them.  A wave works on 32 keys at a time, alone, with nothing in shared memory:
//   S^T = K Q^T   keys are the rows of the first operand, channels its contraction.  A lane owns a key (lane & 15) and a quarter
//                 of its channels (lane >> 4); WHICH channels is free as long as Q agrees, so they are whole 16-byte loads.
//   softmax       S^T leaves a lane with 8 scores of ONE query row: maximum and sum need two cross-lane steps each.
//   O^T = V^T P^T the second operand wants, in each lane, 8 keys of one query row - which is what the lane has.  The first wants
//                 8 keys of one channel: a lane loads dh / 16 consecutive channels of each of its 8 keys and turns that block
//                 over in registers (v_perm), the channels of a tile being every (dh / 16)-th one.
// Codes become T by the scaled conversions of gfx950, one scale a block, exact (a code times a power of two fits T's mantissa).
// The four waves of a workgroup take every fourth tile of 32 keys and are summed through shared memory; long caches are split over
// workgroups, whose partial rows (maximum, sum, unscaled output, all fp32) a second launch joins in fixed order.
#include "ff_attend.h"

namespace ff {

constexpr int kAttWaves = 4;
constexpr int kAttTile = 32;                       // keys of one step of a wave

// ---- 8 elements of a lane in the operands of a product over 8 x 4 of them ------------------------------------------------
template <int DT> struct Frag { uint32_t w[4]; };
template <> struct Frag<FF_F32> { float w[8]; };

template <int DT> __device__ inline f32x4 mma(const Frag<DT>& a, const Frag<DT>& b, f32x4 c) {
    if constexpr (DT == FF_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else if constexpr (DT == FF_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.w[e], b.w[e], c, 0, 0, 0);
        return c;
    }
}

template <int STORE> __device__ inline f32x2 codes2_f32(uint32_t w, float scale, int i) {
    f32x2 f;
    if constexpr (STORE == FF_STORE_E4M3) {
        f = i ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    } else {
        f = i == 0 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0) : i == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1)
          : i == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    }
    f.x *= scale;
    f.y *= scale;
    return f;
}

// N bytes (a power of two) from p into words
template <int N> __device__ inline void load_words(const char* p, uint32_t* w) {
    if constexpr (N == 1) {
        w[0] = *(const uint8_t*)p;
    } else if constexpr (N == 2) {
        w[0] = *(const uint16_t*)p;
    } else if constexpr (N == 4) {
        w[0] = *(const uint32_t*)p;
    } else if constexpr (N == 8) {
        const uint2 v = *(const uint2*)p;
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int k = 0; k < N / 16; ++k) {
            const uint4 v = ((const uint4*)p)[k];
            w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
        }
    }
}

__device__ inline float max_over_quarters(float x) {       // over the four lanes that hold one query row
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float sum_over_quarters(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// How a row of DH channels is loaded: as the key operand (a quarter of the channels a lane, kKC loads of kKE) and as the value
// operand (kVE consecutive channels of 8 keys).
template <int DT, int STORE, int DH> struct Geo {
    static constexpr bool kCodes = STORE != kStoreSame;
    static constexpr int kBits = STORE == FF_STORE_E4M3 ? 8 : STORE == FF_STORE_E2M1 ? 4 : 8 * Act<DT>::kBytes;
    static constexpr int kRow = DH * kBits / 8;
    static constexpr int kKE = DH / 4 < 128 / kBits ? DH / 4 : 128 / kBits;
    static constexpr int kKC = DH / 4 / kKE;
    static constexpr int kKB = kKE * kBits / 8;
    static constexpr int kKW = DH / 4 * kBits / 32;                    // words of a quarter row
    static constexpr int kVE = DH / 16;
    static constexpr int kVB = kVE * kBits / 8;
    static constexpr int kVW = kVB < 4 ? 1 : kVB / 4;
    static constexpr int kBlocks = DH / 32;                            // scale bytes of a row
    static constexpr int kKSW = kBlocks < 4 ? 1 : kBlocks / 4;         // words of one row's scales
    static constexpr int kVSW = kBlocks;                               // words of four rows' scales
};

// What a lane has loaded of 32 keys: quarter rows of keys (lane & 15) and 16 + (lane & 15); channels kVE (lane & 15) .. of keys
// 4 q .. 4 q + 3 and 16 + 4 q .., q = lane >> 4; the scales of the same.
template <int DT, int STORE, int DH> struct Raw {
    using G = Geo<DT, STORE, DH>;
    uint32_t k[2][G::kKW];
    uint32_t v[8][G::kVW];
    uint32_t ks[2][G::kCodes ? G::kKSW : 1];
    uint32_t vs[2][G::kCodes ? G::kVSW : 1];
};

template <int DT, int STORE, int DH>
__device__ inline void load_half(Raw<DT, STORE, DH>& raw, int sub, const ff_cache_t& c, int64_t row, int lane) {
    using G = Geo<DT, STORE, DH>;
    const int key = lane & 15, q = lane >> 4;
    const char* k = (const char*)c.keys + row * G::kRow;
    const char* v = (const char*)c.values + row * G::kRow;
    const uint32_t ko = key * G::kRow + q * G::kKB, vo = 4 * q * G::kRow + key * G::kVB;
#pragma unroll
    for (int x = 0; x < G::kKC; ++x) load_words<G::kKB>(k + (ko + x * 4 * G::kKB), raw.k[sub] + x * (G::kKB / 4));
#pragma unroll
    for (int r = 0; r < 4; ++r) load_words<G::kVB>(v + (vo + r * G::kRow), raw.v[4 * sub + r]);
    if constexpr (G::kCodes) {
        load_words<G::kBlocks>((const char*)c.key_scales + row * G::kBlocks + key * G::kBlocks, raw.ks[sub]);
        load_words<4 * G::kBlocks>((const char*)c.value_scales + row * G::kBlocks + 4 * q * G::kBlocks, raw.vs[sub]);
    }
}

// 8 channels `step` of the quarter row
template <int DT, int STORE, int DH> __device__ inline Frag<DT> key_frag(const Raw<DT, STORE, DH>& raw, int sub, int step, int lane) {
    using G = Geo<DT, STORE, DH>;
    Frag<DT> f;
    if constexpr (!G::kCodes) {
        if constexpr (DT == FF_F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f.w[e] = __uint_as_float(raw.k[sub][step * 8 + e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) f.w[e] = raw.k[sub][step * 4 + e];
        }
    } else {
        // block of the load this step belongs to: loads of 32 channels are blocks, of 16 halves, of 8 quarters of one
        const int x = step * 8 / G::kKE, block = (x * 4 * G::kKE) / 32 + (lane >> 4) * G::kKE / 32;
        const uint32_t word = G::kKSW == 1 ? raw.ks[sub][0] : (block >> 2 ? raw.ks[sub][G::kKSW - 1] : raw.ks[sub][0]);
        const float scale = __uint_as_float(((word >> (8 * (block & 3))) & 255u) << 23);
        constexpr int kPer = STORE == FF_STORE_E4M3 ? 2 : 4;          // pairs of a word
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t w = raw.k[sub][(step * 4 + e) / kPer];
            if constexpr (DT == FF_F32) {
                const f32x2 p = codes2_f32<STORE>(w, block_scale((word >> (8 * (block & 3))) & 255u), (step * 4 + e) % kPer);
                f.w[2 * e] = p.x;
                f.w[2 * e + 1] = p.y;
            } else {
                f.w[e] = codes2<DT, STORE>(w, scale, (step * 4 + e) % kPer);
            }
        }
    }
    return f;
}
// scale byte of key slot j for this lane's channels
template <int DT, int STORE, int DH> __device__ inline uint32_t value_scale(const Raw<DT, STORE, DH>& raw, int j, int lane) {
    using G = Geo<DT, STORE, DH>;
    const int block = (lane & 15) * G::kVE / 32, r = j & 3, sub = j >> 2;
    if constexpr (G::kBlocks == 8) {
        const uint32_t w = block >> 2 ? raw.vs[sub][2 * r + 1] : raw.vs[sub][2 * r];
        return (w >> (8 * (block & 3))) & 255u;
    } else if constexpr (G::kBlocks == 4) {
        return (raw.vs[sub][r] >> (8 * block)) & 255u;
    } else if constexpr (G::kBlocks == 2) {
        return (raw.vs[sub][r >> 1] >> (16 * (r & 1) + 8 * block)) & 255u;
    } else {
        return (raw.vs[sub][0] >> (8 * r)) & 255u;
    }
}

template <int DT, int STORE, int DH> __device__ inline void clear_value(Raw<DT, STORE, DH>& raw, int j) {
    using G = Geo<DT, STORE, DH>;
#pragma unroll
    for (int y = 0; y < G::kVW; ++y) raw.v[j][y] = 0;
    if constexpr (G::kCodes) {
        if constexpr (G::kBlocks == 8) raw.vs[j >> 2][2 * (j & 3)] = raw.vs[j >> 2][2 * (j & 3) + 1] = 0;
        else if constexpr (G::kBlocks == 4) raw.vs[j >> 2][j & 3] = 0;
        else if constexpr (G::kBlocks == 2) raw.vs[j >> 2][(j & 3) >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
        else raw.vs[j >> 2][0] &= ~(255u << (8 * (j & 3)));
    }
}
// takes the NaN and infinities out of a lane's values; whether there were any
template <int DT, int STORE, int DH> __device__ inline bool take_out_odd(Raw<DT, STORE, DH>& raw, int lane) {
    using G = Geo<DT, STORE, DH>;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        bool block = false;
        if constexpr (G::kCodes) block = value_scale<DT, STORE, DH>(raw, j, lane) == 255u;
        odd |= block;
        if (block) clear_value<DT, STORE, DH>(raw, j);
#pragma unroll
        for (int y = 0; y < G::kVW; ++y) {
            uint32_t& w = raw.v[j][y];
            if constexpr (G::kCodes && DT == FF_F16) {              // (values written as another type may pass fp16's range)
                constexpr int kPer = STORE == FF_STORE_E4M3 ? 2 : 4, kWidth = 16 / kPer;
                const float scale = __uint_as_float(value_scale<DT, STORE, DH>(raw, j, lane) << 23);
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    const uint32_t pair = codes2<DT, STORE>(w, scale, k);
                    if ((pair & 0x7c00u) == 0x7c00u) w &= ~(((1u << kWidth) - 1) << (2 * k * kWidth)), odd = true;
                    if ((pair & 0x7c000000u) == 0x7c000000u) w &= ~(((1u << kWidth) - 1) << ((2 * k + 1) * kWidth)), odd = true;
                }
            } else if constexpr (STORE == FF_STORE_E4M3) {                 // the code of all ones is NaN
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (((w >> (8 * k)) & 0x7fu) == 0x7fu) w &= ~(255u << (8 * k)), odd = true;
            } else if constexpr (!G::kCodes) {
                constexpr uint32_t kExp = DT == FF_F32 ? 0x7f800000u : DT == FF_BF16 ? 0x7f80u : 0x7c00u;
                if ((w & kExp) == kExp) w = DT == FF_F32 ? 0u : w & 0xffff0000u, odd = true;
                if (DT != FF_F32 && (w & (kExp << 16)) == (kExp << 16)) w &= 0xffffu, odd = true;
            }
        }
    }
    return odd;
}

// Registers: keys and values of two steps (one in use, one on its way), Q and the outputs.  Where they pass 256 the kernel runs one wave a
// SIMD with 512 (one token of 28 / 4 fp32 heads of 128 over 8 x 20 000 keys: 257 us spilling, 140 us so); fp32 rows of 256 channels
// pass 512 too and are loaded when they are needed (587 us spilling, 267 us so): 64 KB a wave in flight are enough for the memory.
// bf16 and fp16 rows of 128 channels in two tiles are 3 and 5 registers too many for 256, which go to memory and back: 35 rows a kv head over
// 4 x 13 474 keys take 49 us so and 63 us with one wave a SIMD.
constexpr int waves_a_simd(int dt, int store, int dh, int nt) {
    const int bytes = store == kStoreSame && dt == FF_F32 ? 4 : 2;
    return dh * nt * bytes > 512 || dh == 256 || (bytes == 4 && dh == 128) ? 1 : 2;
}
template <int DT, int STORE, int DH, int NT>
__global__ __launch_bounds__(64 * kAttWaves, waves_a_simd(DT, STORE, DH, NT)) void k_cache_attention(const ff_cache_attention_t a, const AttPlan p) {
    using G = Geo<DT, STORE, DH>;
    constexpr int kSteps = DH / 32, kTiles = DH / 16, kPad = 4;
    constexpr bool kAhead = !(DT == FF_F32 && STORE == kStoreSame && DH == 256);
    // Two tiles of 256 channels pass 512 registers by far.  What the compiler then spills it splits between accumulation registers and
    // memory, and in the 8-bit form it brought the first fragment of the first tile's Q back without its third word: wrong scores.
    static_assert(NT == 1 || DH <= (DT == FF_F32 ? 64 : 128), "two tiles of rows must leave the registers room");
    __shared__ float s_o[kAttWaves][16][DH + kPad];
    __shared__ float s_m[kAttWaves][16], s_l[kAttWaves][16];
    const ff_cache_t& c = a.cache;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), q = lane >> 4, col = lane & 15;
    const int n = (int)c.n;
    const int head = blockIdx.y / p.groups, group = blockIdx.y - head * p.groups;
    const bool plain = plain_share(c, p);
    Share share = {p.slots == 1 ? (int)blockIdx.x : 0, p.slots == 1 ? 0 : (int)blockIdx.x, 1, 0};
    if (!plain && !share_of(c, p, blockIdx.x, share)) return;
    const int b = share.b, split = share.split;
    const int32_t* table = c.table + (int64_t)b * c.table_width;
    int page0, page1, off0, off1;
    auto look_up = [&](int64_t key) {             // the pages of a tile, a tile before its rows are loaded
        page0 = page_of_16(c, p, table, key, off0);
        page1 = page_of_16(c, p, table, key + 16, off1);
    };
    const int64_t begin = ((int64_t)split * kAttWaves + wave) * kAttTile;
    look_up(begin);
    const int64_t start = c.start[b], end = keys_of(c, start);

    // the wave's rows of Q, NT tiles of 16; rows past R are zeros
    Frag<DT> qf[NT][kSteps];
    int token[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = (group * NT + t) * 16 + col;
        token[t] = r / p.G;
        const char* src = (const char*)a.q + ((int64_t)b * a.q_batch + (int64_t)(head * p.G + r - token[t] * p.G) * a.q_head + (int64_t)token[t] * a.q_token) * Act<DT>::kBytes;
        // channels in the order of the keys' loads
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            constexpr int kQE = G::kKE < 8 ? G::kKE : 8;              // consecutive channels of a piece (fp32 keys: 4)
#pragma unroll
            for (int x = 0; x < 8 / kQE; ++x) {
                const int at = s * 8 + x * kQE, load = at / G::kKE, d = load * 4 * G::kKE + q * G::kKE + at % G::kKE;
                if constexpr (DT == FF_F32) {
                    uint32_t w[kQE];
                    if (r < p.R) {
                        load_words<kQE * 4>(src + d * 4, w);
                    } else {
#pragma unroll
                        for (int e = 0; e < kQE; ++e) w[e] = 0;
                    }
#pragma unroll
                    for (int e = 0; e < kQE; ++e) qf[t][s].w[x * kQE + e] = __uint_as_float(w[e] ^ p.flip);
                } else {
                    if (r < p.R) {
                        load_words<16>(src + d * 2, qf[t][s].w);
#pragma unroll
                        for (int e = 0; e < 4; ++e) qf[t][s].w[e] ^= p.flip;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) qf[t][s].w[e] = 0;
                    }
                }
            }
        }
    }

    f32x4 o[NT][kTiles];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = kNone;
        l[t] = 0.f;
#pragma unroll
        for (int x = 0; x < kTiles; ++x) o[t][x] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    Raw<DT, STORE, DH> next;
    int64_t next0 = -1, next1 = -1;
    auto fetch = [&](int64_t key) {
        next0 = key < end ? row_on_page(c, head, page0, off0) : -1;
        next1 = key + 16 < end ? row_on_page(c, head, page1, off1) : -1;
        load_half<DT, STORE, DH>(next, 0, c, next0 < 0 ? 0 : next0, lane);      // (what has no place: any row, left out below)
        load_half<DT, STORE, DH>(next, 1, c, next1 < 0 ? 0 : next1, lane);
    };
    const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.mask_batch : nullptr;
    bool odd = false;
    if (plain && p.slots > 1) share.used = max(1, min(p.want, blocks_of(c, p, b)));
    if (split >= share.used) return;
    const int64_t stride = (int64_t)share.used * kAttWaves * kAttTile;
    if (kAhead && begin < end) {
        fetch(begin);
        look_up(begin + stride);
    }
    for (int64_t base = begin; base < end; base += stride) {
        if constexpr (!kAhead) {
            fetch(base);
            look_up(base + stride);
        }
        Raw<DT, STORE, DH> raw = next;
        const int64_t row0 = next0, row1 = next1;
        const bool have0 = row0 >= 0, have1 = row1 >= 0;
        if (kAhead && base + stride < end) {
            fetch(base + stride);
            look_up(base + 2 * stride);
        }
        const bool whole = have0 && have1 && base + kAttTile <= start;    // every row sees every key of the tile

        f32x4 s[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
            for (int x = 0; x < kSteps; ++x) {
                const Frag<DT> kf = key_frag<DT, STORE, DH>(raw, sub, x, lane);
#pragma unroll
                for (int t = 0; t < NT; ++t) s[t][sub] = mma<DT>(kf, qf[t][x], s[t][sub]);
            }
        if (!whole) {
            // values nobody sees may be anything: zeros stand in
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!((j >> 2 ? have1 : have0) && base + (j >> 2) * 16 + 4 * q + (j & 3) < end)) clear_value<DT, STORE, DH>(raw, j);
            // new tokens do not all see each other, and 0 x NaN is NaN: a NaN or infinity among these keys' values stays out of the
            // products and is added at the end to the rows that see it
            if (base + kAttTile > start && take_out_odd<DT, STORE, DH>(raw, lane)) odd = true;
        }
        Frag<DT> pf[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = s[t][j >> 2][j & 3];
            if (!whole) {
                const int fresh0 = (int)(base - start) + 4 * q, left = (int)(end - base) - 4 * q, own = min(token[t], n - 1);
                uint32_t sees = 0;
                if (mask) {
                    uint32_t byte[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) byte[j] = mask[(int64_t)own * n + min(max(fresh0 + (j >> 2) * 16 + (j & 3), 0), n - 1)];
#pragma unroll
                    for (int j = 0; j < 8; ++j) sees |= byte[j] || fresh0 + (j >> 2) * 16 + (j & 3) < 0 ? 1u << j : 0u;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) sees |= fresh0 + (j >> 2) * 16 + (j & 3) <= own ? 1u << j : 0u;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!((sees >> j) & 1u) || !(j >> 2 ? have1 : have0) || (j >> 2) * 16 + (j & 3) >= left) x[j] = kNone;
            }
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            top = max_over_quarters(top) * p.scale2;
            // the running maximum moves only when a row passes it by 2^8: until then the weights stay below 256, nothing is lost
            // and no output is rescaled
            if (__any(top > m[t] + 8.f)) {
                const float up = fmaxf(m[t], top), down = __builtin_amdgcn_exp2f(m[t] - (up == kNone ? 0.f : up));
                m[t] = up;
                l[t] *= down;
#pragma unroll
                for (int y = 0; y < kTiles; ++y) o[t][y] *= down;
            }
            const float zero = (m[t] == kNone ? 0.f : m[t]) - kLift<DT>;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], p.scale2, -zero));
                sum += x[j];
            }
            l[t] += sum;
            if constexpr (DT == FF_F32) {
#pragma unroll
                for (int j = 0; j < 8; ++j) pf[t].w[j] = x[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) pf[t].w[j] = pack2<DT>(x[2 * j], x[2 * j + 1]);
            }
        }
        if constexpr (DT == FF_F32) {
            Frag<DT> vf[kTiles];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (G::kCodes) {
                    const float scale = block_scale(value_scale<DT, STORE, DH>(raw, j, lane));
                    constexpr int kPer = STORE == FF_STORE_E4M3 ? 2 : 4;
#pragma unroll
                    for (int y = 0; y < kTiles / 2; ++y) {
                        const f32x2 v = codes2_f32<STORE>(raw.v[j][y / kPer], scale, y % kPer);
                        vf[2 * y].w[j] = v.x;
                        vf[2 * y + 1].w[j] = v.y;
                    }
                } else {
#pragma unroll
                    for (int y = 0; y < kTiles; ++y) vf[y].w[j] = __uint_as_float(raw.v[j][y]);
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int y = 0; y < kTiles; ++y) o[t][y] = mma<DT>(vf[y], pf[t], o[t][y]);
        } else {
            float scale[8];
            if constexpr (G::kCodes) {
#pragma unroll
                for (int j = 0; j < 8; ++j) scale[j] = __uint_as_float(value_scale<DT, STORE, DH>(raw, j, lane) << 23);
            }
            constexpr int kPer = STORE == FF_STORE_E4M3 ? 2 : 4;
#pragma unroll
            for (int y = 0; y < kTiles / 2; ++y) {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if constexpr (G::kCodes) w[j] = codes2<DT, STORE>(raw.v[j][y / kPer], scale[j], y % kPer);
                    else w[j] = raw.v[j][y];
                }
                Frag<DT> even, odd;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    even.w[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x05040100u);
                    odd.w[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x07060302u);
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    o[t][2 * y] = mma<DT>(even, pf[t], o[t][2 * y]);
                    o[t][2 * y + 1] = mma<DT>(odd, pf[t], o[t][2 * y + 1]);
                }
            }
        }
    }

    if (__any(odd)) {
        // rare: the values left out above, to the rows that see them (their weight is positive: infinities and NaN stay what they are)
        for (int64_t base = begin; base < end; base += stride) {
            if (base + kAttTile <= start) continue;
#pragma unroll 1
            for (int k = 0; k < kAttTile; ++k) {
                const int64_t r = row_of_16(c, p, table, head, base + (k & 16), end), fresh = base + k - start;
                if (r < 0 || base + k >= end) continue;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int own = min(token[t], n - 1);
                    if (fresh >= 0 && !(mask ? mask[(int64_t)own * n + fresh] != 0 : fresh <= own)) continue;
#pragma unroll
                    for (int u = 0; u < DH / 32; ++u) {
                        float f[8];
                        __builtin_amdgcn_sched_barrier(0);             // (one load at a time: registers are for the usual path)
                        fetch8<DT, STORE>(c.values, c.value_scales, r + (k & 15), DH, q * (DH / 32) + u, f);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float v = Act<DT>::rnd(f[e]);
                            if (!(fabsf(v) < __builtin_inff())) o[t][(u * 8 + e) % kTiles][(u * 8 + e) / kTiles] += v;
                        }
                    }
                }
            }
        }
    }

    // (stores stand behind the loop: in front of it the page table could no longer be read as a constant, by scalar loads - 358 us
    // became 490)
    if (p.slots > 1 && split == 0 && blockIdx.y == 0 && threadIdx.x == 0) p.shares[b] = make_int2(share.first, share.used);
    // the four waves' rows, joined: channel (4 q + r) kVE + x of row `col` is o[x][r]
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (t) __syncthreads();
        l[t] = sum_over_quarters(l[t]);
        if (q == 0) {
            s_m[wave][col] = m[t];
            s_l[wave][col] = l[t];
        }
        __syncthreads();
        float top = kNone;
#pragma unroll
        for (int w = 0; w < kAttWaves; ++w) top = fmaxf(top, s_m[w][col]);
        const float down = __builtin_amdgcn_exp2f(m[t] - (top == kNone ? 0.f : top));
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int x = 0; x < kTiles; ++x) s_o[wave][col][(4 * q + r) * kTiles + x] = o[t][x][r] * down;
        __syncthreads();
        constexpr int kUnits = DH / 4;                                 // float4s of a row
        for (int u = threadIdx.x; u < 16 * kUnits; u += 64 * kAttWaves) {
            const int row = u / kUnits, d = (u - row * kUnits) * 4, r = (group * NT + t) * 16 + row;
            if (r >= p.R) continue;
            float most = kNone, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kAttWaves; ++w) most = fmaxf(most, s_m[w][row]);
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kAttWaves; ++w) {
                sum += s_l[w][row] * __builtin_amdgcn_exp2f(s_m[w][row] - (most == kNone ? 0.f : most));
                acc += *(const f32x4*)&s_o[w][row][d];
            }
            if (p.slots > 1) {
                const int64_t at = ((int64_t)head * p.R + r) * p.slots + blockIdx.x;
                *(f32x4*)(p.part + at * DH + d) = acc;
                if (d == 0) ((float2*)(p.part + p.part_rows * DH))[at] = make_float2(most, sum);
            } else {
                const int i = r / p.G;
                char* out = (char*)a.out + ((int64_t)b * a.o_batch + (int64_t)(head * p.G + r - i * p.G) * a.o_head + (int64_t)i * a.o_token) * Act<DT>::kBytes;
                write_out4<DT>(out, d, acc, sum);
            }
        }
    }
}

// Joins the splits of query rows: kLanes lanes take 4 channels each of a row (or a piece of it), kGroup such groups share its splits.
// Rows enough: a group for the whole row.  The few rows and many splits of single tokens: 32 channels a workgroup and 32 groups over
// the splits, so that 28 rows of 256 splits are 112 workgroups of 8 loads a thread.  The sums meet in fixed order.
constexpr int kJoinThreads = 256;
template <int DT, int DH, int kLanes, int kGroup>
__global__ __launch_bounds__(kJoinThreads) void k_cache_attention_join(const ff_cache_attention_t a, const AttPlan p) {
    constexpr int kPieces = DH / 4 / kLanes, kRows = kJoinThreads / kLanes / kGroup;
    __shared__ f32x4 s_o[kRows * kGroup][kLanes];
    __shared__ float s_l[kRows * kGroup], s_m[kRows * kGroup];
    const int lane = threadIdx.x % kLanes, g = threadIdx.x / kLanes, y = g % kGroup, head = blockIdx.y, b = blockIdx.z;
    const int u = blockIdx.x % kPieces * kLanes + lane, r = blockIdx.x / kPieces * kRows + g / kGroup;
    const int2 share = p.shares[b];
    const int used = r < p.R ? share.y : 0;
    const int64_t at = ((int64_t)head * p.R + (r < p.R ? r : 0)) * p.slots + share.x;
    const float2* ml = (const float2*)(p.part + p.part_rows * DH) + at;
    const float* part = p.part + at * DH + u * 4;
    float top = kNone;
    for (int s = y; s < used; s += kGroup) top = fmaxf(top, ml[s].x);
    const float zero = top == kNone ? 0.f : top;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll 4
    for (int s = y; s < used; s += kGroup) {
        const float2 x = ml[s];
        const float w = __builtin_amdgcn_exp2f(x.x - zero);
        acc += *(const f32x4*)(part + (int64_t)s * DH) * w;
        sum += x.y * w;
    }
    if constexpr (kGroup > 1) {
        s_o[g][lane] = acc;
        if (lane == 0) s_l[g] = sum, s_m[g] = top;
        __syncthreads();
        if (y) return;
        float most = kNone;
#pragma unroll
        for (int k = 0; k < kGroup; ++k) most = fmaxf(most, s_m[g + k]);
        const float base = most == kNone ? 0.f : most;
        acc = f32x4{0.f, 0.f, 0.f, 0.f};
        sum = 0.f;
#pragma unroll
        for (int k = 0; k < kGroup; ++k) {
            const float w = __builtin_amdgcn_exp2f(s_m[g + k] - base);
            acc += s_o[g + k][lane] * w;
            sum += s_l[g + k] * w;
        }
    }
    if (r >= p.R) return;
    const int i = r / p.G;
    char* out = (char*)a.out + ((int64_t)b * a.o_batch + (int64_t)(head * p.G + r - i * p.G) * a.o_head + (int64_t)i * a.o_token) * Act<DT>::kBytes;
    write_out4<DT>(out, u * 4, acc, sum);
}

static int attention_check(const ff_cache_attention_t* a) {
    if (!a) return FF_ERR_ARG;
    const int rc = cache_check(&a->cache);
    if (rc) return rc;
    if ((a->cache.B && a->cache.n && (!a->q || !a->out)) || a->H < 1 || a->H % a->cache.kv_heads || a->mask_batch < 0 || !(fabs(a->scale) <= 1e30)) return FF_ERR_ARG;
    if (a->cache.dh != 32 && a->cache.dh != 64 && a->cache.dh != 128 && a->cache.dh != 256) return FF_ERR_UNSUPPORTED;
    if (a->H > 65535 || a->cache.B > 65535 || a->cache.n * a->H > 61439 * 16) return FF_ERR_UNSUPPORTED;      // (grids: kv heads x groups of 16 rows)
    const int64_t per = a->cache.dtype == FF_F32 ? 4 : 8;
    if (!cache_aligned(a->q) || !cache_aligned(a->out)) return FF_ERR_ALIGN;
    const int64_t strides[6] = {a->q_batch, a->q_head, a->q_token, a->o_batch, a->o_head, a->o_token};
    for (int64_t s : strides)
        if (s % per) return FF_ERR_ALIGN;
    return FF_OK;
}

// Which kernel serves R query rows, and how many waves share a block of keys there.  Up to 128 rows (and fp32, whose products are
// slow anyway): 0, ff_attend.hip, whose waves hold 16 or 32 rows and read the cache again for the rows of the next workgroup; more:
// ff_attend_rows.hip, tiles of 32 rows, a wave each.  A call over 4 sequences of 13 474, 28 / 4 heads of 128, here / there in us:
//   rows       35         63         84         126        168        252
//   bf16   49 / 38    55 / 41    69 / 38    57 / 40    90 / 50    84 / 53
//   8 bits 39 / 39    46 / 42    53 / 39    53 / 41    67 / 51    78 / 54
//   4 bits 34 / 39    39 / 42    45 / 40    46 / 42    60 / 50    70 / 53
// Heads of 64 and 256 and a single sequence cross at the same place: at about 32 rows for a cache in T, 64 for codes.  From there to 128
// the kernel there is ahead, by up to 1.8 (2.2 at 256 channels): the border was set before that kernel fed its products as it does now.
static int row_waves(int dtype, int64_t R, int64_t dh) { return dtype == FF_F32 || R <= 128 ? 0 : dh == 256 ? 4 : 8; }

static AttPlan attention_plan(const ff_cache_attention_t* a) {
    const ff_cache_t& c = a->cache;
    AttPlan p;
    p.G = (int)(a->H / c.kv_heads);
    p.R = (int)(p.G * c.n);
    const int waves = row_waves((int)c.dtype, p.R, c.dh);
    if (waves) {
        const int tiles = (p.R + 31) / 32;
        p.groups = (tiles + waves - 1) / waves;
        p.tiles = (tiles + p.groups - 1) / p.groups;
        p.block = 64;
    } else {
        // two tiles of 16 rows a wave where their registers fit beside the keys' (16-bit T up to 128 channels, fp32 up to 64)
        p.tiles = p.R <= 16 || c.dh > (c.dtype == FF_F32 ? 64 : 128) ? 1 : 2;
        p.groups = (p.R + 16 * p.tiles - 1) / (16 * p.tiles);
        p.block = kAttWaves * kAttTile;
    }
    p.page16 = (int)(c.page_size / 16);
    p.magic = p.page16 == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / p.page16);
    const double scale2 = a->scale * 1.4426950408889634;
    p.scale2 = fmaxf(fabsf((float)scale2), 1.17549435e-38f);
    p.flip = scale2 < 0 ? (c.dtype == FF_F32 ? 0x80000000u : 0x80008000u) : 0u;
    // workgroups over the keys: enough to fill 256 CUs several times over, no more than there can be blocks; none where every
    // sequence is one block at most, or where the sequences alone make twice as many workgroups
    const int64_t base = c.kv_heads * p.groups, blocks = (c.table_width * c.page_size + p.block - 1) / p.block;
    // (many rows: one workgroup a CU; few rows: two at a time, in two rounds - half or twice as many cost a fifth more)
    const int64_t fill = waves ? 256 : 1024, want = fill / base > 0 ? fill / base : 1;
    p.exact = waves != 0;
    const bool whole = blocks <= 1 || c.B >= 2 * want;
    p.want = (int)(want < c.B * blocks ? want : c.B * blocks);
    p.slots = whole ? 1 : (int)(p.want + (c.B > 1 ? c.B : 0));
    p.part_rows = p.slots > 1 ? c.kv_heads * p.R * p.slots : 0;
    p.part = (float*)a->ws;
    p.shares = p.part ? (int2*)(p.part + p.part_rows * (c.dh + 2)) : nullptr;
    return p;
}

template <int DT, int STORE, int DH>
static int launch_attention(const ff_cache_attention_t* a, const AttPlan& p) {
    const ff_cache_t& c = a->cache;
    const dim3 grid((uint32_t)(p.slots == 1 ? c.B : p.slots), (uint32_t)(c.kv_heads * p.groups));
    hipStream_t st = (hipStream_t)a->stream;
    if constexpr (DH <= (DT == FF_F32 ? 64 : 128))
        if (p.tiles == 2) k_cache_attention<DT, STORE, DH, 2><<<grid, 64 * kAttWaves, 0, st>>>(*a, p);
    if (p.tiles == 1) k_cache_attention<DT, STORE, DH, 1><<<grid, 64 * kAttWaves, 0, st>>>(*a, p);
    return (int)hipGetLastError();
}
template <int DT, int STORE>
static int launch_attention_dh(const ff_cache_attention_t* a, const AttPlan& p) {
    switch (a->cache.dh) {
        case 32: return launch_attention<DT, STORE, 32>(a, p);
        case 64: return launch_attention<DT, STORE, 64>(a, p);
        case 128: return launch_attention<DT, STORE, 128>(a, p);
        default: return launch_attention<DT, STORE, 256>(a, p);
    }
}
template <int DT, int DH, int kLanes, int kGroup>
static int launch_join_groups(const ff_cache_attention_t* a, const AttPlan& p) {
    constexpr int kRows = kJoinThreads / kLanes / kGroup;
    const dim3 grid((uint32_t)((p.R + kRows - 1) / kRows * (DH / 4 / kLanes)), (uint32_t)a->cache.kv_heads, (uint32_t)a->cache.B);
    k_cache_attention_join<DT, DH, kLanes, kGroup><<<grid, kJoinThreads, 0, (hipStream_t)a->stream>>>(*a, p);
    return (int)hipGetLastError();
}
template <int DT, int DH>
static int launch_join(const ff_cache_attention_t* a, const AttPlan& p) {
    // (6 832 rows of 32 slots: 8.2 us with four groups a row, 8.3 us with one)
    if (a->cache.B * a->cache.kv_heads * p.R >= 1024) return launch_join_groups<DT, DH, DH / 4, DH == 256 ? 2 : 4>(a, p);
    // (28 rows: 256 slots 12.3 us with the rows whole, 7.1 us in pieces; 33 slots 3.9 and 4.5; 56 rows of 258 slots 7.0 and 6.2)
    return p.slots > 64 ? launch_join_groups<DT, DH, 8, 32>(a, p) : launch_join_groups<DT, DH, DH / 4, kJoinThreads / (DH / 4)>(a, p);
}
template <int DT>
static int launch_attention_t(const ff_cache_attention_t* a, const AttPlan& p) {
    const int waves = row_waves(DT, p.R, a->cache.dh);
    int rc = FF_OK;
    if constexpr (DT != FF_F32) rc = waves ? launch_attention_rows<DT>(a, p) : FF_OK;
    if (!waves) {
        if (a->cache.store == FF_STORE_E4M3) rc = launch_attention_dh<DT, FF_STORE_E4M3>(a, p);
        else if (a->cache.store == FF_STORE_E2M1) rc = launch_attention_dh<DT, FF_STORE_E2M1>(a, p);
        else rc = launch_attention_dh<DT, kStoreSame>(a, p);
    }
    if (rc || p.slots == 1) return rc;
    switch (a->cache.dh) {
        case 32: return launch_join<DT, 32>(a, p);
        case 64: return launch_join<DT, 64>(a, p);
        case 128: return launch_join<DT, 128>(a, p);
        default: return launch_join<DT, 256>(a, p);
    }
}

}  // namespace ff

extern "C" size_t ff_cache_attention_workspace_bytes(const ff_cache_attention_t* a) {
    if (ff::attention_check(a) || a->cache.B == 0 || a->cache.n == 0) return 0;
    const ff::AttPlan p = ff::attention_plan(a);
    return p.slots > 1 ? (size_t)p.part_rows * (size_t)(a->cache.dh + 2) * sizeof(float) + (size_t)a->cache.B * sizeof(int2) : 0;
}

extern "C" int ff_cache_attention(const ff_cache_attention_t* a) {
    const int rc = ff::attention_check(a);
    if (rc) return rc;
    if (a->cache.B == 0 || a->cache.n == 0) return FF_OK;
    const size_t need = ff_cache_attention_workspace_bytes(a);
    if (a->ws_bytes < need || (need && (!a->ws || !ff::cache_aligned(a->ws)))) return FF_ERR_WORKSPACE;
    const ff::AttPlan p = ff::attention_plan(a);
    if (a->cache.dtype == FF_F32) return ff::launch_attention_t<FF_F32>(a, p);
    if (a->cache.dtype == FF_BF16) return ff::launch_attention_t<FF_BF16>(a, p);
    return ff::launch_attention_t<FF_F16>(a, p);
}
