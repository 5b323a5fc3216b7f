// ff_rotary.hip - rotary positions: the tables, and q and k turned by them.
#include "ff_common.h"

namespace ff {

// kVec consecutive channels as floats
template <int DT, int kVec> __device__ inline void get(const void* p, int64_t at, float* f) {
    if constexpr (kVec == 1) {
        f[0] = Act<DT>::load1(p, at);
    } else {
        const uint4* w = (const uint4*)((const char*)p + at * Act<DT>::kBytes);
        constexpr int kWords = kVec / Act<DT>::kPer16;
#pragma unroll
        for (int k = 0; k < kWords; ++k) Act<DT>::unpack(w[k], f + k * Act<DT>::kPer16);
    }
}
template <int DT, int kVec> __device__ inline void put(void* p, int64_t at, float* f) {
    if constexpr (kVec == 1) {
        Act<DT>::store1(p, at, f[0]);
    } else {
        uint4* w = (uint4*)((char*)p + at * Act<DT>::kBytes);
        constexpr int kWords = kVec / Act<DT>::kPer16;
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
            float* x = f + k * Act<DT>::kPer16;
            if constexpr (DT == FF_BF16) w[k] = Act<DT>::pack_rne(x);
            else w[k] = Act<DT>::pack(x);
        }
    }
}

// kVec consecutive angles of one position to a thread, blockDim.x threads to a position.  position * inv_freq is formed in turns in
// fp64 (2^-52 of up to 2^31 turns: 2^-21 of a turn at the far end, 2^-31 at a million), its whole turns are taken off there, and only
// the rest goes to fp32.  The tables are written in 16-byte pieces (one element at a time where half a row does not allow it): with
// two bytes a thread and a 64-bit division to find the position the stores and the division cost as much again as the bytes.
template <int DT, int kVec>
__global__ __launch_bounds__(256) void k_rotary_tables(const int64_t* __restrict__ positions, int64_t n, const double* __restrict__ inv_freq,
                                                       int half, float factor, int interleaved, void* __restrict__ cos_out, void* __restrict__ sin_out) {
    const int64_t p = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (p >= n) return;
    const double position = (double)positions[p];
    for (int i = threadIdx.x * kVec; i < half; i += blockDim.x * kVec) {
        float c[kVec], s[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const double turns = position * (inv_freq[i + e] * 0.15915494309189533577);
            sincospif(2.f * (float)(turns - rint(turns)), &s[e], &c[e]);
            c[e] *= factor;
            s[e] *= factor;
        }
        const int64_t row = p * 2 * half;
        if (interleaved) {
            float cc[2 * kVec], ss[2 * kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                cc[2 * e] = cc[2 * e + 1] = c[e];
                ss[2 * e] = ss[2 * e + 1] = s[e];
            }
            put<DT, kVec>(cos_out, row + 2 * i, cc);
            put<DT, kVec>(cos_out, row + 2 * i + kVec, cc + kVec);
            put<DT, kVec>(sin_out, row + 2 * i, ss);
            put<DT, kVec>(sin_out, row + 2 * i + kVec, ss + kVec);
        } else {
            put<DT, kVec>(cos_out, row + i, c);
            put<DT, kVec>(cos_out, row + half + i, c);
            put<DT, kVec>(sin_out, row + i, s);
            put<DT, kVec>(sin_out, row + half + i, s);
        }
    }
}

// One token (blockIdx.x) of blockDim.y heads: thread (u, y) turns one piece of one head.  Piece u of the half layout is channels
// [u kVec, + kVec) of both halves; of the interleaved one, 2 kVec consecutive channels.  Pieces past rot / 2 are copied.  Every
// byte of q and k is read and written once; the tables of a token are read once by a workgroup and again by its heads from L1.
template <int DT, int TDT, int kVec>
__global__ __launch_bounds__(256) void k_rotary_apply(const ff_rotary_t a) {
    const uint32_t tok = blockIdx.x, b = tok / (uint32_t)a.L, t = tok - b * (uint32_t)a.L;
    const int head = blockIdx.y * blockDim.y + threadIdx.y, H = (int)a.H;
    if (head >= H + (int)a.H_kv) return;
    const bool is_k = head >= H;
    const int h = is_k ? head - H : head;
    const void* src = is_k ? a.k : a.q;
    void* dst = is_k ? a.k_out : a.q_out;
    const int64_t from = is_k ? (int64_t)b * a.k_batch + h * a.k_head + t * a.k_token : (int64_t)b * a.q_batch + h * a.q_head + t * a.q_token;
    const int64_t to = is_k ? (int64_t)b * a.ko_batch + h * a.ko_head + t * a.ko_token : (int64_t)b * a.qo_batch + h * a.qo_head + t * a.qo_token;
    const int half = (int)(a.rot / 2), pairs = half / kVec, units = pairs + (int)(a.dh - a.rot) / kVec;
    const float flip = a.transpose ? -1.f : 1.f;
    const int64_t tab = (int64_t)b * a.t_batch + t * a.t_token;
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
        if (u >= pairs) {
            float x[kVec];
            const int64_t at = a.rot + (int64_t)(u - pairs) * kVec;
            get<DT, kVec>(src, from + at, x);
            put<DT, kVec>(dst, to + at, x);
            continue;
        }
        float x[2 * kVec], c[2 * kVec], s[2 * kVec], y[2 * kVec];
        const int one = a.interleaved ? 2 * u * kVec : u * kVec, two = a.interleaved ? one + kVec : one + half;
        get<DT, kVec>(src, from + one, x);
        get<DT, kVec>(src, from + two, x + kVec);
        const int i0 = u * kVec, i1 = i0 + kVec - 1, sec1 = (int)(a.sec0 + a.sec1);
        if (sec1 > 0 && ((i0 < a.sec0) != (i1 < a.sec0) || (i0 < sec1) != (i1 < sec1))) {
            // a section ends inside the piece: each pair from its own axis
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                const int64_t at = tab + (i0 + e < a.sec0 ? 0 : i0 + e < sec1 ? 1 : 2) * a.t_axis + i0 + e;
                c[e] = Act<TDT>::load1(a.cos, at);
                c[kVec + e] = Act<TDT>::load1(a.cos, at + half);
                s[e] = Act<TDT>::load1(a.sin, at);
                s[kVec + e] = Act<TDT>::load1(a.sin, at + half);
            }
        } else {
            const int64_t at = tab + (sec1 == 0 || i0 < a.sec0 ? 0 : i0 < sec1 ? 1 : 2) * a.t_axis;
            get<TDT, kVec>(a.cos, at + one, c);
            get<TDT, kVec>(a.cos, at + two, c + kVec);
            get<TDT, kVec>(a.sin, at + one, s);
            get<TDT, kVec>(a.sin, at + two, s + kVec);
        }
        // partner of register r: half layout r <-> r + kVec, interleaved r <-> r ^ 1 (one pair when kVec == 1: the same thing);
        // forwards a channel's sine multiplies its partner's x, in the gradient the partner's sine does
        if (a.interleaved) {
#pragma unroll
            for (int e = 0; e < 2 * kVec; e += 2) {
                const float s1 = a.transpose ? s[e + 1] : s[e], s2 = a.transpose ? s[e] : s[e + 1];
                y[e] = fmaf(x[e], c[e], -flip * (x[e + 1] * s1));
                y[e + 1] = fmaf(x[e + 1], c[e + 1], flip * (x[e] * s2));
            }
        } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                const float s1 = a.transpose ? s[kVec + e] : s[e], s2 = a.transpose ? s[e] : s[kVec + e];
                y[e] = fmaf(x[e], c[e], -flip * (x[kVec + e] * s1));
                y[kVec + e] = fmaf(x[kVec + e], c[kVec + e], flip * (x[e] * s2));
            }
        }
        put<DT, kVec>(dst, to + one, y);
        put<DT, kVec>(dst, to + two, y + kVec);
    }
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int DT>
static int launch_tables(const int64_t* positions, int64_t n, const double* inv_freq, int half, float factor, int interleaved, void* cos, void* sin,
                         hipStream_t st) {
    constexpr int kVec = Act<DT>::kPer16;
    const bool wide = half % kVec == 0 && aligned16(cos) && aligned16(sin);
    const int units = wide ? half / kVec : half, x = min(units, 256), y = 256 / x;
    const dim3 block(x, y), grid((uint32_t)((n + y - 1) / y));
    if (wide) k_rotary_tables<DT, kVec><<<grid, block, 0, st>>>(positions, n, inv_freq, half, factor, interleaved, cos, sin);
    else k_rotary_tables<DT, 1><<<grid, block, 0, st>>>(positions, n, inv_freq, half, factor, interleaved, cos, sin);
    return (int)hipGetLastError();
}

template <int DT, int TDT, int kVec>
static int launch_apply(const ff_rotary_t* a) {
    const int units = (int)(a->rot / 2 / kVec + (a->dh - a->rot) / kVec), x = min(units, 256);
    const int heads = (int)(a->H + a->H_kv), y = max(1, min(256 / x, heads));
    const dim3 block(x, y), grid((uint32_t)(a->B * a->L), (heads + y - 1) / y);
    k_rotary_apply<DT, TDT, kVec><<<grid, block, 0, (hipStream_t)a->stream>>>(*a);
    return (int)hipGetLastError();
}
template <int DT, int TDT>
static int launch_apply_any(const ff_rotary_t* a) {
    // 16-byte pieces of the activations when every row, half and tail starts on one (tables: the same channels, 32 bytes of
    // fp32 beside 16 of T), else one element a thread
    constexpr int kVec = 8 > Act<DT>::kPer16 ? Act<DT>::kPer16 : 8;
    constexpr int kTab = Act<TDT>::kPer16;
    constexpr int kStep = kVec > kTab ? kVec : kTab;
    const int64_t st[12] = {a->q_batch, a->q_head, a->q_token, a->k_batch, a->k_head, a->k_token,
                            a->qo_batch, a->qo_head, a->qo_token, a->ko_batch, a->ko_head, a->ko_token};
    bool wide = aligned16(a->q) && aligned16(a->q_out) && aligned16(a->k) && aligned16(a->k_out) && aligned16(a->cos) && aligned16(a->sin);
    wide = wide && (a->rot / 2) % kStep == 0 && (a->dh - a->rot) % kStep == 0 && a->t_axis % kTab == 0 && a->t_batch % kTab == 0 && a->t_token % kTab == 0;
    for (int64_t s : st) wide = wide && s % Act<DT>::kPer16 == 0;
    return wide ? launch_apply<DT, TDT, kStep>(a) : launch_apply<DT, TDT, 1>(a);
}
template <int DT>
static int launch_apply_t(const ff_rotary_t* a) {
    return a->table_dtype == FF_F32 ? launch_apply_any<DT, FF_F32>(a) : launch_apply_any<DT, DT>(a);
}

}  // namespace ff

extern "C" int ff_rotary_tables(const int64_t* positions, int64_t n, const double* inv_freq, int64_t half, double factor, int interleaved,
                                int dtype, void* cos, void* sin, ff_stream_t stream) {
    if (n < 0 || half < 1 || !positions || !inv_freq || !cos || !sin) return FF_ERR_ARG;
    if (dtype != FF_F32 && dtype != FF_BF16 && dtype != FF_F16) return FF_ERR_ARG;
    if (half > 4096 || n > 0x7fffffff) return FF_ERR_UNSUPPORTED;
    if (n == 0) return FF_OK;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == FF_F32) return ff::launch_tables<FF_F32>(positions, n, inv_freq, (int)half, (float)factor, interleaved, cos, sin, st);
    if (dtype == FF_BF16) return ff::launch_tables<FF_BF16>(positions, n, inv_freq, (int)half, (float)factor, interleaved, cos, sin, st);
    return ff::launch_tables<FF_F16>(positions, n, inv_freq, (int)half, (float)factor, interleaved, cos, sin, st);
}

extern "C" int ff_rotary_apply(const ff_rotary_t* a) {
    if (!a || !a->cos || !a->sin || a->B < 0 || a->L < 0 || a->H < 0 || a->H_kv < 0 || a->dh < 2 || a->rot < 2) return FF_ERR_ARG;
    if ((a->H && (!a->q || !a->q_out)) || (a->H_kv && (!a->k || !a->k_out))) return FF_ERR_ARG;
    if (a->dtype != FF_F32 && a->dtype != FF_BF16 && a->dtype != FF_F16) return FF_ERR_ARG;
    if (a->table_dtype != a->dtype && a->table_dtype != FF_F32) return FF_ERR_ARG;
    if (a->rot % 2 || a->rot > a->dh || a->sec0 < 0 || a->sec1 < 0 || a->sec0 + a->sec1 > a->rot / 2) return FF_ERR_ARG;
    if (a->interleaved && a->sec0 + a->sec1 > 0) return FF_ERR_ARG;
    if (a->dh > 4096 || a->H + a->H_kv > 65535 || (a->L && a->B > 0x7fffffff / a->L)) return FF_ERR_UNSUPPORTED;
    if (a->B == 0 || a->L == 0 || a->H + a->H_kv == 0) return FF_OK;
    if (a->dtype == FF_F32) return ff::launch_apply_t<FF_F32>(a);
    if (a->dtype == FF_BF16) return ff::launch_apply_t<FF_BF16>(a);
    return ff::launch_apply_t<FF_F16>(a);
}
