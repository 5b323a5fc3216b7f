// ff_attend.hip - attention of the new tokens of each sequence (one, a chunk, or a tree of drafted ones) over the paged cache.
#include "ff_cache.h"

namespace ff {

// One wave to a query row.  Lanes take keys for the scores (64 at a time, running maximum and sum in fp32), channels for the
// values.
template <int DT, int STORE>
__global__ __launch_bounds__(64) void k_cache_attention(const ff_cache_attention_t a) {
    __shared__ float s_q[256];
    const ff_cache_t& c = a.cache;
    const int lane = threadIdx.x, dh = (int)c.dh, kv = (int)c.kv_heads, n = (int)c.n;
    const uint32_t h = blockIdx.y, b = blockIdx.x / (uint32_t)n, i = blockIdx.x - b * (uint32_t)n;
    const int head = (int)(h / (uint32_t)(a.H / kv));
    const int32_t* table = c.table + (int64_t)b * c.table_width;
    const int64_t start = c.start[b];
    char* out = (char*)a.out + ((int64_t)b * a.o_batch + h * a.o_head + i * a.o_token) * Act<DT>::kBytes;
    for (int e = lane; e < dh; e += 64) s_q[e] = Act<DT>::load1(a.q, (int64_t)b * a.q_batch + h * a.q_head + i * a.q_token + e);
    __syncthreads();
    const int64_t end = start < 0 ? 0 : min(start + n, c.table_width * c.page_size);
    float m = -__builtin_inff(), l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t j0 = 0; j0 < end; j0 += 64) {
        const int64_t j = j0 + lane;
        const int64_t row = j < end ? cache_row(table, c.table_width, c.n_pages, (int)c.page_size, kv, head, j) : -1;
        bool seen = row >= 0;
        if (seen && j >= start) seen = a.mask ? a.mask[(int64_t)b * a.mask_batch + (int64_t)i * n + (j - start)] != 0 : j - start <= i;
        float s = -__builtin_inff();
        if (seen) {
            s = 0.f;
            for (int u = 0; u < dh / 8; ++u) {
                float f[8];
                fetch8<DT, STORE>(c.keys, c.key_scales, row, dh, u, f);
                for (int e = 0; e < 8; ++e) s = fmaf(s_q[u * 8 + e], f[e], s);
            }
            s *= (float)a.scale;
        }
        float top = s;
        for (int k = 32; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor(top, k, 64));
        const float m_new = fmaxf(m, top), base = m_new == -__builtin_inff() ? 0.f : m_new;
        const float down = __expf(m - base), p = seen ? __expf(s - base) : 0.f;
        l = l * down + wave_sum(p);
        m = m_new;
        for (int k = 0; k < 4; ++k) o[k] *= down;
        for (int k = 0; k < 64; ++k) {
            const int64_t r = __shfl(row, k, 64);
            const float w = __shfl(p, k, 64);
            if (!__shfl((int)seen, k, 64)) continue;
            if (lane * 4 >= dh) continue;
            float f[8];
            fetch8<DT, STORE>(c.values, c.value_scales, r, dh, lane / 2, f);
            for (int e = 0; e < 4; ++e) o[e] = fmaf(w, f[(lane & 1) * 4 + e], o[e]);
        }
    }
    if (lane * 4 < dh)
        for (int e = 0; e < 4; ++e) Act<DT>::store1(out, lane * 4 + e, l > 0.f || l != l ? o[e] / l : 0.f);
}

static int attention_check(const ff_cache_attention_t* a) {
    if (!a) return FF_ERR_ARG;
    const int rc = cache_check(&a->cache);
    if (rc) return rc;
    if (!a->q || !a->out || a->H < 1 || a->H % a->cache.kv_heads || a->mask_batch < 0) return FF_ERR_ARG;
    if (a->cache.dh != 32 && a->cache.dh != 64 && a->cache.dh != 128 && a->cache.dh != 256) return FF_ERR_UNSUPPORTED;
    if (a->H > 65535) return FF_ERR_UNSUPPORTED;
    const int64_t per = a->cache.dtype == FF_F32 ? 4 : 8;
    if (!cache_aligned(a->q) || !cache_aligned(a->out)) return FF_ERR_ALIGN;
    const int64_t strides[6] = {a->q_batch, a->q_head, a->q_token, a->o_batch, a->o_head, a->o_token};
    for (int64_t s : strides)
        if (s % per) return FF_ERR_ALIGN;
    return FF_OK;
}

template <int DT, int STORE>
static int launch_attention(const ff_cache_attention_t* a) {
    k_cache_attention<DT, STORE><<<dim3((uint32_t)(a->cache.B * a->cache.n), (uint32_t)a->H), 64, 0, (hipStream_t)a->stream>>>(*a);
    return (int)hipGetLastError();
}
template <int DT>
static int launch_attention_t(const ff_cache_attention_t* a) {
    if (a->cache.store == FF_STORE_E4M3) return launch_attention<DT, FF_STORE_E4M3>(a);
    if (a->cache.store == FF_STORE_E2M1) return launch_attention<DT, FF_STORE_E2M1>(a);
    return launch_attention<DT, kStoreSame>(a);
}

}  // namespace ff

extern "C" size_t ff_cache_attention_workspace_bytes(const ff_cache_attention_t* a) {
    (void)a;
    return 0;
}

extern "C" int ff_cache_attention(const ff_cache_attention_t* a) {
    const int rc = ff::attention_check(a);
    if (rc) return rc;
    if (a->cache.B == 0 || a->cache.n == 0) return FF_OK;
    if (a->ws_bytes < ff_cache_attention_workspace_bytes(a)) return FF_ERR_WORKSPACE;
    if (a->cache.dtype == FF_F32) return ff::launch_attention_t<FF_F32>(a);
    if (a->cache.dtype == FF_BF16) return ff::launch_attention_t<FF_BF16>(a);
    return ff::launch_attention_t<FF_F16>(a);
}
