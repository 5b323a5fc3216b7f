// Shared by the two attention kernels over the paged cache: ff_attend.hip (few query rows) and ff_attend_rows.hip (many).
#pragma once

#include "ff_cache.h"

namespace ff {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kNone = -__builtin_inff();

template <int DT> __device__ inline uint32_t pack2(float a, float b) {      // two floats rounded to T (16 bits)
    if constexpr (DT == FF_BF16) {
        bf16x2_t p;
        p.x = (__bf16)a;
        p.y = (__bf16)b;
        return __builtin_bit_cast(uint32_t, p);
    } else {
        half2_t p;
        p.x = (_Float16)a;
        p.y = (_Float16)b;
        return __builtin_bit_cast(uint32_t, p);
    }
}
// two codes of a stored word as T: 8 bits - pair `i` of 2, 4 bits - pair `i` of 4
template <int DT, int STORE> __device__ inline uint32_t codes2(uint32_t w, float scale, int i) {
    if constexpr (STORE == FF_STORE_E4M3) {
        if constexpr (DT == FF_BF16)
            return i ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))
                     : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
        else
            return i ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true))
                     : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
    } else {
        if constexpr (DT == FF_BF16) {
            return i == 0 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0))
                 : i == 1 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1))
                 : i == 2 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2))
                          : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
        } else {
            return i == 0 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0))
                 : i == 1 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1))
                 : i == 2 ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2))
                          : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
        }
    }
}
struct AttPlan {                    // what the host derives once a call
    int G, R, groups;               // heads a kv head, query rows of one (n G), workgroups over the rows
    int want, slots, block;         // workgroups over the keys of all sequences: about `want`, at most `slots` = want + B (1: each
                                    // sequence whole); they take blocks of so many keys
    int exact;                      // no more than `want`: they fill the chip once, and a second round would cost as much again
    int tiles;                      // many rows: tiles of 32 rows a workgroup
    int page16;                     // page_size / 16 ...
    uint32_t magic;                 // ... and floor(2^32 / page16) (2^32 - 1 for 1)
    float scale2;                   // |scale| log2(e), at least the smallest normal number (0 times a masked score would be NaN)
    uint32_t flip;                  // scale < 0: sign bits of two elements of 16-bit Q, taken up there (fp32: of one)
    float* part;                    // slots > 1: [kv heads, R, slots] x DH sums, then as many (maximum, sum) pairs, then
    int2* shares;                   // (first slot, splits) of each sequence, written by its split 0 for the join
    int64_t part_rows;
};

// Weights are 2^(score - maximum + lift), which leaves sums and outputs scaled alike.  fp16 keeps numbers from 2^-14 whole: with the maximum
// allowed to lag by 2^8, a lift of 2^7 still fits (2^15), and weights down to 2^-21 of the largest lose nothing (2^-32: are not lost).
template <int DT> constexpr float kLift = DT == FF_F16 ? 7.f : 0.f;

// keys of a sequence that the new tokens may see: everything before them and themselves, as far as the table reaches
__device__ inline int64_t keys_of(const ff_cache_t& c, int64_t start) {
    const int64_t room = c.n_pages > 0 ? c.table_width * c.page_size : 0;
    return start < 0 ? 0 : min(start + c.n, room);
}
// Which part of the work workgroup `w` over the keys has: split `split` of the `used` ones of sequence `b`, blocks split, split +
// used, ..; `first` = the slot of the sequence's split 0.  The lengths are on the device alone, so the shares are made there: every
// wave adds up the blocks of all sequences and deals them out so that each split has about as many (a long sequence gets more
// splits, an empty one the one that writes its zeros).  All lanes of the wave call it.
struct Share { int b, split, used, first; };
// one sequence, or none split: known at once but for `used`, so a kernel's first loads need not wait for the lengths
__device__ inline bool plain_share(const ff_cache_t& c, const AttPlan& p) { return c.B == 1 || p.slots == 1; }
__device__ inline int blocks_of(const ff_cache_t& c, const AttPlan& p, int b) { return (int)((keys_of(c, c.start[b]) + p.block - 1) / p.block); }
__device__ inline bool share_of(const ff_cache_t& c, const AttPlan& p, int w, Share& s) {
    const int B = (int)c.B, lane = threadIdx.x & 63;
    auto sum = [&](int each) {                    // blocks of all sequences, or with each > 0 their splits of so many
        uint32_t low = 0, high = 0;               // (2^16 sequences of 2^25 blocks pass 32 bits)
        for (int b = lane; b < B; b += 64) {
            const uint32_t n = blocks_of(c, p, b), x = each ? max(1u, (n + each - 1) / each) : n;
            low += x & 0xffffu;
            high += x >> 16;
        }
        // on the DPP network: a sum by shuffles through the LDS crossbar costs 0.5 us, and there are several
        return (int64_t)(uint32_t)__builtin_amdgcn_readlane(wave_incl_scan_dpp((int)low), 63) +
               ((int64_t)(uint32_t)__builtin_amdgcn_readlane(wave_incl_scan_dpp((int)high), 63) << 16);
    };
    const int64_t total = sum(0);
    int each = (int)max((int64_t)1, (total + p.want - 1) / p.want);
    if (p.exact && B < p.want) {                  // (shares are rounded up sequence by sequence: where that makes too many, they grow a little)
        for (int k = 0; k < 6 && sum(each) > p.want; ++k) each += each / 16 + 1;
    }
    int before = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int b = b0 + lane, used = b < B ? max(1, (blocks_of(c, p, b) + each - 1) / each) : 0;
        const int incl = wave_incl_scan_dpp(used);
        const uint64_t found = __ballot(b < B && before + incl > w);
        if (found) {
            const int l = __ffsll((long long)found) - 1;
            s.b = b0 + l;
            s.used = __builtin_amdgcn_readlane(used, l);
            s.first = before + __builtin_amdgcn_readlane(incl, l) - s.used;
            s.split = w - s.first;
            return true;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
}

// the page number (any value) of the 16 keys from `key` on, a multiple of 16, and their first row on it; -1 past the table
__device__ inline int page_of_16(const ff_cache_t& c, const AttPlan& p, const int32_t* table, int64_t key, int& off) {
    const uint32_t x = (uint32_t)(key >> 4);
    uint32_t slot = __umulhi(x, p.magic);                                      // (one too small at most)
    off = x - slot * p.page16;
    if (off >= p.page16) {
        ++slot;
        off -= p.page16;
    }
    off *= 16;
    return key < c.table_width * c.page_size ? table[slot] : -1;
}
// row of the cache behind it for one kv head; -1: the keys have no place
__device__ inline int64_t row_on_page(const ff_cache_t& c, int head, int page, int off) {
    return page < 0 || page >= c.n_pages ? -1 : ((int64_t)page * (int)c.kv_heads + head) * c.page_size + off;
}
__device__ inline int64_t row_of_16(const ff_cache_t& c, const AttPlan& p, const int32_t* table, int head, int64_t key, int64_t end) {
    int off;
    const int page = page_of_16(c, p, table, key, off);
    return key < end ? row_on_page(c, head, page, off) : -1;
}

// four consecutive channels of one output row, sums divided by the weights' total (0: the row saw nothing)
template <int DT> __device__ inline void write_out4(char* out, int d, f32x4 acc, float sum) {
    const float over = sum == 0.f ? 0.f : 1.f / sum;
    if constexpr (DT == FF_F32) *(f32x4*)(out + d * 4) = acc * over;
    else *(uint2*)(out + d * 2) = make_uint2(pack2<DT>(acc[0] * over, acc[1] * over), pack2<DT>(acc[2] * over, acc[3] * over));
}

// csrc/ff_attend_rows.hip
template <int DT> int launch_attention_rows(const ff_cache_attention_t* a, const AttPlan& p);

}  // namespace ff
