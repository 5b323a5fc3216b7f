// ff_cache.hip - the paged cache of decoded tokens: writing (with quantisation), reading back, moving accepted drafts.
//
// All three are copies: what bounds them is the bytes of the rows (and, for one token, the launch).  A row's `dh` channels are
// handled 8 to a lane, so that a block of 32 channels - the unit of a scale - is four neighbouring lanes and its maximum two
// cross-lane steps, with nothing in shared memory.
#include "ff_cache.h"

namespace ff {

constexpr int kRowThreads = 256;

int cache_check(const ff_cache_t* c) {
    // (an empty tensor may have no address: a pool of no pages, a table of no width, a batch of nothing)
    if ((c->n_pages && (!c->keys || !c->values)) || (c->table_width && c->B && !c->table) || (c->B && !c->start)) return FF_ERR_ARG;
    if (c->dtype != FF_F32 && c->dtype != FF_BF16 && c->dtype != FF_F16) return FF_ERR_ARG;
    const bool codes = c->store == FF_STORE_E4M3 || c->store == FF_STORE_E2M1;
    if (!codes && c->store != c->dtype) return FF_ERR_ARG;
    if (codes && c->n_pages && (!c->key_scales || !c->value_scales)) return FF_ERR_ARG;
    if (c->n_pages < 0 || c->kv_heads < 1 || c->page_size < 1 || c->dh < 1 || c->table_width < 0 || c->B < 0 || c->n < 0) return FF_ERR_ARG;
    if (!cache_aligned(c->keys) || !cache_aligned(c->values) || !cache_aligned(c->key_scales) || !cache_aligned(c->value_scales)) return FF_ERR_ALIGN;
    if (c->dh % 32 || c->dh > 256 || c->page_size % 16 || c->page_size > 65536 || c->n_pages > 0x7fffffff || c->kv_heads > 4096) return FF_ERR_UNSUPPORTED;
    if (c->table_width > 0x7fff0000 / c->page_size) return FF_ERR_UNSUPPORTED;
    if (c->B > 0x7fffffff / 64 || c->n > 0x7fffffff / 64 || (c->n && c->B > 0x7fffffff / 64 / c->n)) return FF_ERR_UNSUPPORTED;
    return FF_OK;
}

// x as four lanes' 8 channels of one block: returns the scale byte, x becomes x * 2^-e (limited, and zeros for a block that
// holds a NaN or an infinity).  In fp32 every step is exact: the limit and 2^-e are powers of two times small integers.
template <int DT, int STORE>
__device__ inline uint32_t block_prepare(float* x) {
    constexpr float kCap = (STORE == FF_STORE_E4M3 ? 1.875f : 1.5f) * (DT == FF_F16 ? 0x1p15f : 0x1p127f);
    constexpr uint32_t kTopMantissa = STORE == FF_STORE_E4M3 ? 0x600000u : 0x400000u;    // 448 = 1.75 * 2^8, 6 = 1.5 * 2^2
    constexpr int kTopExponent = STORE == FF_STORE_E4M3 ? 8 : 2;
    uint32_t big = 0;                                             // (magnitudes order as their bits do; NaN above infinity)
#pragma unroll
    for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(x[e]) & 0x7fffffffu);
    big = max(big, (uint32_t)__shfl_xor((int)big, 1, 4));
    big = max(big, (uint32_t)__shfl_xor((int)big, 2, 4));
    if (big >= 0x7f800000u) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
        return 255u;
    }
    big = min(big, __float_as_uint(kCap));
    // the smallest e with big <= top * 2^e, from the bits of `big` (a subnormal fp32 has field 0: far below the lower limit)
    const int e = max((int)(big >> 23) - 127 - kTopExponent + ((big & 0x7fffffu) > kTopMantissa ? 1 : 0), -100);
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -kCap), kCap) * down;
    return (uint32_t)(e + 127);
}

// Unit threadIdx.x (8 channels) of a row, a key or value of one kv head of one token.
// kChunk = 0, few tokens: a token to a workgroup, its rows threadIdx.y, + blockDim.y, ..; the page is looked up once for all of them.
// kChunk > 0: kChunk times blockDim.y consecutive tokens of ONE row (blockIdx.y) to a workgroup, kChunk in flight a thread: then what a
// workgroup writes is whole lines, also of the scales (4 bytes a token at 128 channels), which otherwise go out in pieces from the
// L2s of different XCDs.
template <int DT, int STORE, int kChunk, bool kWrite>
__global__ __launch_bounds__(kRowThreads) void k_cache_rows(const ff_cache_rows_t a) {
    constexpr int kTokens = kChunk ? kChunk : 1;
    const ff_cache_t& c = a.cache;
    const uint32_t n = (uint32_t)c.n, step = kChunk ? blockDim.y : 1, per = (n + kTokens * step - 1) / (kTokens * step);
    const uint32_t b = blockIdx.x / per, t0 = (blockIdx.x - b * per) * kTokens * step + (kChunk ? threadIdx.y : 0);
    const int start = c.start[b];
    if (kWrite && start < 0) return;
    const int kv = (int)c.kv_heads, dh = (int)c.dh, u = threadIdx.x;
    int64_t row0[kTokens];
#pragma unroll
    for (int k = 0; k < kTokens; ++k)
        row0[k] = start < 0 || t0 + k * step >= n ? -1 : cache_row(c.table + (int64_t)b * c.table_width, c.table_width, c.n_pages, (int)c.page_size, kv, 0,
                                                                  (int64_t)start + t0 + k * step);
    for (int r = kChunk ? blockIdx.y : threadIdx.y; r < 2 * kv; r += kChunk ? 2 * kv : blockDim.y) {
        const bool is_v = r >= kv;
        const int h = is_v ? r - kv : r;
        const int64_t token = (is_v ? a.v_token : a.k_token) * step;
        char* mine = (char*)(is_v ? a.v : a.k) +
            ((is_v ? (int64_t)b * a.v_batch + h * a.v_head : (int64_t)b * a.k_batch + h * a.k_head) + t0 * (is_v ? a.v_token : a.k_token) + u * 8) * Act<DT>::kBytes;
        void* codes = is_v ? c.values : c.keys;
        uint8_t* scales = is_v ? c.value_scales : c.key_scales;
        float x[kTokens][8];
#pragma unroll
        for (int k = 0; k < kTokens; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[k][e] = 0.f;
            if (row0[k] < 0) continue;
            if constexpr (kWrite) load8<DT>(mine + k * token * Act<DT>::kBytes, x[k]);
            else fetch8<DT, STORE>(codes, scales, row0[k] + (int64_t)h * c.page_size, dh, u, x[k]);
        }
#pragma unroll
        for (int k = 0; k < kTokens; ++k) {
            if constexpr (!kWrite) {
                if (t0 + k * step < n) store8<DT>(mine + k * token * Act<DT>::kBytes, x[k]);
                continue;
            }
            if (row0[k] < 0) continue;                       // (the same for all lanes of a block of 32 channels)
            const int64_t row = row0[k] + (int64_t)h * c.page_size;
            char* dst = (char*)codes + row * row_bytes<DT, STORE>(dh);
            if constexpr (STORE == kStoreSame) {
                store8<DT>(dst + u * 8 * Act<DT>::kBytes, x[k]);
            } else {
                const uint32_t byte = block_prepare<DT, STORE>(x[k]);
                if constexpr (STORE == FF_STORE_E4M3) {
                    int lo = 0, hi = 0;
                    lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[k][0], x[k][1], lo, false);
                    lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[k][2], x[k][3], lo, true);
                    hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[k][4], x[k][5], hi, false);
                    hi = __builtin_amdgcn_cvt_pk_fp8_f32(x[k][6], x[k][7], hi, true);
                    ((uint2*)dst)[u] = make_uint2((uint32_t)lo, (uint32_t)hi);
                } else {
                    uint32_t w = 0;
                    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[k][0], x[k][1], 1.0f, 0);
                    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[k][2], x[k][3], 1.0f, 1);
                    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[k][4], x[k][5], 1.0f, 2);
                    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[k][6], x[k][7], 1.0f, 3);
                    ((uint32_t*)dst)[u] = w;
                }
                if ((u & 3) == 0) scales[row * (dh / 32) + u / 4] = (uint8_t)byte;
            }
        }
    }
}

// One workgroup for the keys or the values of one head of one sequence.  Row i comes from row accepted[i] >= i, so rows are moved
// in chunks, ascending, each read whole before it is written: a chunk's sources lie at or behind its own first row, which no
// earlier chunk has written.  A row is moved as 16-byte pieces (dh is a multiple of 32: at least one), its scale bytes by the
// lanes of its first pieces (never more of them than pieces).
__global__ __launch_bounds__(kRowThreads) void k_cache_keep(const ff_cache_t c, const int32_t* __restrict__ accepted, int m, int bytes, int scale_bytes) {
    __shared__ int s_count;
    const uint32_t b = blockIdx.x;
    const int h = blockIdx.y, tid = threadIdx.x;
    const int start = c.start[b];
    if (start < 0) return;
    const int32_t* list = accepted + (int64_t)b * m;
    const int32_t* table = c.table + (int64_t)b * c.table_width;
    if (tid == 0) s_count = m;
    __syncthreads();
    for (int i = tid; i < m; i += kRowThreads) {
        const int x = list[i], before = i ? list[i - 1] : -1;
        if (x <= before || x < 0 || cache_row(table, c.table_width, c.n_pages, (int)c.page_size, 1, 0, (int64_t)start + x) < 0) atomicMin(&s_count, i);
    }
    __syncthreads();
    const int count = s_count;
    char* rows = (char*)(blockIdx.z ? c.values : c.keys);
    uint8_t* scales = blockIdx.z ? c.value_scales : c.key_scales;
    const int pieces = bytes / 16, per = kRowThreads / pieces, mine = tid / pieces, piece = tid - mine * pieces;
    for (int i0 = 0; i0 < count; i0 += per) {
        const int i = i0 + mine;
        int64_t dst = -1;
        uint4 x;
        uint8_t sc = 0;
        if (mine < per && i < count && list[i] != i) {
            const int64_t src = cache_row(table, c.table_width, c.n_pages, (int)c.page_size, (int)c.kv_heads, h, (int64_t)start + list[i]);
            dst = cache_row(table, c.table_width, c.n_pages, (int)c.page_size, (int)c.kv_heads, h, (int64_t)start + i);
            if (src < 0) dst = -1;
            if (dst >= 0) {
                x = *(const uint4*)(rows + src * bytes + piece * 16);
                if (piece < scale_bytes) sc = scales[src * scale_bytes + piece];
            }
        }
        __syncthreads();
        if (dst >= 0) {
            *(uint4*)(rows + dst * bytes + piece * 16) = x;
            if (piece < scale_bytes) scales[dst * scale_bytes + piece] = sc;
        }
        __syncthreads();
    }
}

static int rows_check(const ff_cache_rows_t* a) {
    if (!a) return FF_ERR_ARG;
    const int rc = cache_check(&a->cache);
    if (rc) return rc;
    if (!a->k || !a->v) return FF_ERR_ARG;
    const int64_t per = a->cache.dtype == FF_F32 ? 4 : 8;
    if (!cache_aligned(a->k) || !cache_aligned(a->v)) return FF_ERR_ALIGN;
    const int64_t strides[6] = {a->k_batch, a->k_head, a->k_token, a->v_batch, a->v_head, a->v_token};
    for (int64_t s : strides)
        if (s % per) return FF_ERR_ALIGN;
    return FF_OK;
}

template <int DT, int STORE>
static int launch_rows(const ff_cache_rows_t* a, bool write) {
    const ff_cache_t& c = a->cache;
    const int units = (int)c.dh / 8, most = kRowThreads / units;
    hipStream_t st = (hipStream_t)a->stream;
    if (c.n >= most) {
        constexpr int kChunk = 2;
        const dim3 block(units, most), grid((uint32_t)(c.B * ((c.n + kChunk * most - 1) / (kChunk * most))), (uint32_t)(2 * c.kv_heads));
        if (write) k_cache_rows<DT, STORE, kChunk, true><<<grid, block, 0, st>>>(*a);
        else k_cache_rows<DT, STORE, kChunk, false><<<grid, block, 0, st>>>(*a);
    } else {
        const dim3 block(units, min(most, (int)(2 * c.kv_heads))), grid((uint32_t)(c.B * c.n));
        if (write) k_cache_rows<DT, STORE, 0, true><<<grid, block, 0, st>>>(*a);
        else k_cache_rows<DT, STORE, 0, false><<<grid, block, 0, st>>>(*a);
    }
    return (int)hipGetLastError();
}
template <int DT>
static int launch_rows_t(const ff_cache_rows_t* a, bool write) {
    if (a->cache.store == FF_STORE_E4M3) return launch_rows<DT, FF_STORE_E4M3>(a, write);
    if (a->cache.store == FF_STORE_E2M1) return launch_rows<DT, FF_STORE_E2M1>(a, write);
    return launch_rows<DT, kStoreSame>(a, write);
}
static int launch_rows_any(const ff_cache_rows_t* a, bool write) {
    const int rc = rows_check(a);
    if (rc) return rc;
    if (a->cache.B == 0 || a->cache.n == 0) return FF_OK;
    if (a->cache.dtype == FF_F32) return launch_rows_t<FF_F32>(a, write);
    if (a->cache.dtype == FF_BF16) return launch_rows_t<FF_BF16>(a, write);
    return launch_rows_t<FF_F16>(a, write);
}

}  // namespace ff

extern "C" int ff_cache_write(const ff_cache_rows_t* args) { return ff::launch_rows_any(args, true); }
extern "C" int ff_cache_read(const ff_cache_rows_t* args) { return ff::launch_rows_any(args, false); }

extern "C" int ff_cache_keep(const ff_cache_t* c, const int32_t* accepted, int64_t m, ff_stream_t stream) {
    if (!c || m < 0 || (m && !accepted)) return FF_ERR_ARG;
    const int rc = ff::cache_check(c);
    if (rc) return rc;
    if (m > 0x7fffffff / 2) return FF_ERR_UNSUPPORTED;
    if (c->B == 0 || m == 0) return FF_OK;
    const bool codes = c->store == FF_STORE_E4M3 || c->store == FF_STORE_E2M1;
    const int bytes = (int)(c->store == FF_STORE_E4M3 ? c->dh : c->store == FF_STORE_E2M1 ? c->dh / 2 : c->dh * (c->dtype == FF_F32 ? 4 : 2));
    const dim3 grid((uint32_t)c->B, (uint32_t)c->kv_heads, 2);
    ff::k_cache_keep<<<grid, ff::kRowThreads, 0, (hipStream_t)stream>>>(*c, accepted, (int)m, bytes, codes ? (int)(c->dh / 32) : 0);
    return (int)hipGetLastError();
}
