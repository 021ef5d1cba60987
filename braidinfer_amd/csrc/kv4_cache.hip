// Rows into and out of the cache of 4-bit keys and values (layout and number format: kv4.h).
//
// Writing: x -> E = clamp(floor(log2 max|x|) - 2, -124, 125) of its 32 neighbours, the code nearest to x / 2^E (ties to the even
// code; the hardware's conversion).  The largest magnitude is taken of the floats' bits as integers: infinities and NaN come
// out above every number, and its exponent is their upper bits.
#include "kv4.h"

template <typename T> __device__ __forceinline__ void kv4_load16(const T* p, float* v);
template <> __device__ __forceinline__ void kv4_load16<float>(const float* p, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x4 q = *(const f32x4*)(p + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * i + e] = q[e];
    }
}
template <> __device__ __forceinline__ void kv4_load16<bf16>(const bf16* p, float* v) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bf16x8 q = *(const bf16x8*)(p + 8 * i);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * i + e] = (float)q[e];
    }
}
template <typename T> __device__ __forceinline__ void kv4_store16(T* p, unsigned w0, unsigned w1, float scale);
template <> __device__ __forceinline__ void kv4_store16<float>(float* p, unsigned w0, unsigned w1, float scale) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned w = i ? w1 : w0;
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
        const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
        *(f32x4*)(p + 8 * i) = f32x4{a[0], a[1], b[0], b[1]};
        *(f32x4*)(p + 8 * i + 4) = f32x4{c[0], c[1], d[0], d[1]};
    }
}
template <> __device__ __forceinline__ void kv4_store16<bf16>(bf16* p, unsigned w0, unsigned w1, float scale) {
    *(bf16x8*)p = kv4_to_bf16(w0, scale);
    *(bf16x8*)(p + 8) = kv4_to_bf16(w1, scale);
}

// Where token t of the step lives: the head-parts of its page from `page`, its place in it; false: nowhere (padding, or a
// page that is not there).
struct Kv4Place {
    const int* pos;
    const int* seq_of_token;
    const int* slots;
    const int* table;
    int n_seqs, n_slots, table_pages, n_pages;
    __device__ __forceinline__ bool find(int t, int& page, int& in_page) const {
        const int b = seq_of_token[t];
        if ((unsigned)b >= (unsigned)n_seqs) return false;
        const int slot = slots[b], p = pos[t];
        if ((unsigned)slot >= (unsigned)n_slots || p < 0 || p / KV4_PAGE >= table_pages) return false;
        page = table[(size_t)slot * table_pages + p / KV4_PAGE];
        in_page = p % KV4_PAGE;
        return (unsigned)page < (unsigned)n_pages;
    }
};

// A lane takes 16 elements (half a block) of a key or value row; neighbouring lanes its next 16, then the next token of a
// group of 8, then the next head: a wave's stores are runs of 8 tokens, which lie together in both orders of the page.
// What it moves is what bounds it; there is nothing to reuse.
// ROT: the keys are rotated first (pairs (p, p + rd / 2), or neighbours when `adjacent`), and further lanes rotate the
// queries in place, 8 pairs each.  The rotated keys are rounded to the rows' type before they are held, as the cache of
// that type holds them.
template <typename T, int M, bool ROT>
__global__ __launch_bounds__(256) void rope_kv4_write_kernel(T* __restrict__ qkv, const float* __restrict__ cs, const float* __restrict__ sn,
                                                             Kv4Place place, unsigned char* __restrict__ cache, int n_tokens, int nq,
                                                             int nkv, int rd, int adjacent, int write_cache, unsigned kv_blocks) {
    constexpr int HD = 32 * M, PIECES = 2 * M;
    typedef kv4_layout<M> L;
    const size_t width = (size_t)(nq + 2 * nkv) * HD;
    const int P = rd / 2;
    if (ROT && blockIdx.x >= kv_blocks) {
        const int units = (P + 7) / 8;
        const size_t u = (size_t)(blockIdx.x - kv_blocks) * 256 + threadIdx.x;
        const int w = (int)(u % units);
        const size_t th = u / units;
        const int t = (int)(th / nq), h = (int)(th % nq);
        if (t >= n_tokens) return;
        T* row = qkv + (size_t)t * width + (size_t)h * HD;
        const float* c = cs + (size_t)t * P;
        const float* s = sn + (size_t)t * P;
        if (8 * w + 8 <= P && (adjacent || P % 8 == 0)) {
            // 8 pairs whole: neighbours are 16 elements in a row, halves 8 and 8
            float a[8], b[8], co[8], si[8];
            T* lo = row + (adjacent ? 16 * w : 8 * w);
            T* hi = adjacent ? lo + 8 : lo + P;
            ew_load<T, 4>(lo, a); ew_load<T, 4>(lo + 4, a + 4); ew_load<T, 4>(hi, b); ew_load<T, 4>(hi + 4, b + 4);
            if (P % 4 == 0) {
                ew_load<float, 4>(c + 8 * w, co); ew_load<float, 4>(c + 8 * w + 4, co + 4);
                ew_load<float, 4>(s + 8 * w, si); ew_load<float, 4>(s + 8 * w + 4, si + 4);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) { co[e] = c[8 * w + e]; si[e] = s[8 * w + e]; }
            }
            float x[16];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = adjacent ? (e < 4 ? a[2 * (e & 3)] : b[2 * (e & 3)]) : a[e];
                const float g = adjacent ? (e < 4 ? a[2 * (e & 3) + 1] : b[2 * (e & 3) + 1]) : b[e];
                x[e] = f * co[e] - g * si[e];
                x[8 + e] = f * si[e] + g * co[e];
            }
            float y[16];
#pragma unroll
            for (int e = 0; e < 8; ++e) { y[2 * e] = x[e]; y[2 * e + 1] = x[8 + e]; }
#pragma unroll
            for (int i = 0; i < 4; ++i) ew_store<T, 4>((i < 2 ? lo : hi) + 4 * (i & 1), adjacent ? y + 4 * i : x + 4 * i);
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int p = 8 * w + e;
            if (p >= P) break;
            const int i0 = adjacent ? 2 * p : p, i1 = adjacent ? 2 * p + 1 : p + P;
            const float a = to_f32<T>(row[i0]), b = to_f32<T>(row[i1]);
            row[i0] = from_f32<T>(a * c[p] - b * s[p]);
            row[i1] = from_f32<T>(a * s[p] + b * c[p]);
        }
        return;
    }
    if (!write_cache) return;
    const size_t idx = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int piece = (int)(idx % PIECES);
    const size_t rest = idx / PIECES;
    const size_t gh = rest / 8;
    const int head = (int)(gh % (2 * nkv));
    const size_t t = gh / (2 * nkv) * 8 + rest % 8;
    int page = 0, in_page = 0;
    // lanes without a row stay for the exchange of the maxima: both halves of a block leave or store together
    const bool ok = t < (size_t)n_tokens && place.find((int)t, page, in_page);
    float x[16];
    if (ok) {
        const T* row = qkv + t * width + (size_t)(nq + head) * HD;
        const int d0 = piece * 16;
        kv4_load16<T>(row + d0, x);
        if (ROT && head < nkv && d0 < rd) {
            const float* c = cs + t * P;
            const float* s = sn + t * P;
            if (!adjacent && P % 16 == 0 && d0 + 16 <= rd) {
                const bool low = d0 < P;
                const int p0 = low ? d0 : d0 - P;
                float y[16], co[16], si[16];
                kv4_load16<T>(row + (low ? d0 + P : d0 - P), y);
                kv4_load16<float>(c + p0, co);
                kv4_load16<float>(s + p0, si);
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = to_f32<T>(from_f32<T>(low ? x[e] * co[e] - y[e] * si[e] : y[e] * si[e] + x[e] * co[e]));
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int d = d0 + e;
                    if (d >= rd) break;
                    const bool low = adjacent ? !(d & 1) : d < P;
                    const int p = adjacent ? d / 2 : (low ? d : d - P);
                    const int other = adjacent ? d ^ 1 : (low ? d + P : d - P);
                    const float y = to_f32<T>(row[other]);
                    x[e] = to_f32<T>(from_f32<T>(low ? x[e] * c[p] - y * s[p] : y * s[p] + x[e] * c[p]));
                }
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = 0.f;
    }
    unsigned big = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const unsigned b = __float_as_uint(x[e]) & 0x7fffffffu;
        big = b > big ? b : big;
    }
    const unsigned other = (unsigned)__shfl_xor((int)big, 1, WAVE);
    big = other > big ? other : big;
    if (!ok) return;
    const bool finite = big < 0x7f800000u;
    int s = (int)(big >> 23) - 2;                    // 127 + floor(log2(big)) - 2
    s = s < 3 ? 3 : s;
    const float scale = kv4_scale(s);
    unsigned w[2] = {0u, 0u};
    if (finite) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], x[8 * i], x[8 * i + 1], scale, 0);
            w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], x[8 * i + 2], x[8 * i + 3], scale, 1);
            w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], x[8 * i + 4], x[8 * i + 5], scale, 2);
            w[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[i], x[8 * i + 6], x[8 * i + 7], scale, 3);
        }
    }
    const unsigned char byte = (unsigned char)(finite ? s : 255);
    const bool is_k = head < nkv;
    unsigned char* part = cache + ((size_t)page * nkv + (is_k ? head : head - nkv)) * L::BYTES;
    if (is_k) {
        *(u32x2*)(part + L::KC + in_page * (16 * M) + piece * 8) = u32x2{w[0], w[1]};
        if (!(piece & 1)) part[L::KS + kv4_key_scale(in_page, piece >> 1, M)] = byte;
    } else {
        unsigned char* at = part + L::VC + ((in_page >> 3) * (4 * M) + 2 * piece) * 32 + (in_page & 7) * 4;
        *(unsigned*)at = w[0];
        *(unsigned*)(at + 32) = w[1];
        if (!(piece & 1)) part[L::VS + ((in_page >> 3) * M + (piece >> 1)) * 8 + (in_page & 7)] = byte;
    }
}

// Rows out of the pages, the same lanes the other way round.
template <typename T, int M>
__global__ __launch_bounds__(256) void kv4_read_kernel(T* __restrict__ k_out, T* __restrict__ v_out, Kv4Place place,
                                                       const unsigned char* __restrict__ cache, int n_tokens, int nkv) {
    constexpr int HD = 32 * M, PIECES = 2 * M;
    typedef kv4_layout<M> L;
    const size_t idx = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int piece = (int)(idx % PIECES);
    const size_t rest = idx / PIECES;
    const size_t gh = rest / 8;
    const int head = (int)(gh % (2 * nkv));
    const size_t t = gh / (2 * nkv) * 8 + rest % 8;
    int page, in_page;
    if (t >= (size_t)n_tokens || !place.find((int)t, page, in_page)) return;
    const bool is_k = head < nkv;
    const int kvh = is_k ? head : head - nkv;
    const unsigned char* part = cache + ((size_t)page * nkv + kvh) * L::BYTES;
    T* row = (is_k ? k_out : v_out) + (t * nkv + kvh) * HD + piece * 16;
    if (is_k) {
        const u32x2 w = *(const u32x2*)(part + L::KC + in_page * (16 * M) + piece * 8);
        kv4_store16<T>(row, w[0], w[1], kv4_scale(part[L::KS + kv4_key_scale(in_page, piece >> 1, M)]));
    } else {
        const unsigned char* at = part + L::VC + ((in_page >> 3) * (4 * M) + 2 * piece) * 32 + (in_page & 7) * 4;
        kv4_store16<T>(row, *(const unsigned*)at, *(const unsigned*)(at + 32),
                       kv4_scale(part[L::VS + ((in_page >> 3) * M + (piece >> 1)) * 8 + (in_page & 7)]));
    }
}

#define KV4_SIZES(F) F(1) F(2) F(3) F(4) F(5) F(6) F(7) F(8)

extern "C" int br_rope_kv4_write(void* qkv, int is_bf16, const float* cs, const float* sn, const int* pos, const int* seq_of_token,
                                 const int* slots, int n_seqs, const int* table, int n_slots, int table_pages, void* cache, int n_pages,
                                 int T, int nq, int nkv, int hd, int rd, int adjacent, int write_cache, hipStream_t s) {
    if (hd % 32 || hd < 32 || hd > 256 || rd < 0 || rd > hd || rd % 2 || nq < 0 || nkv < 1 || T < 0) return BR_BAD_ARG;
    const bool rot = cs && rd > 0;
    const unsigned long long kv = write_cache ? (unsigned long long)((T + 7) / 8) * 2 * nkv * 8 * (hd / 16) : 0;
    const unsigned long long q = rot ? (unsigned long long)T * nq * ((rd / 2 + 7) / 8) : 0;
    const unsigned long long kvb = (kv + 255) / 256, blocks = kvb + (q + 255) / 256;
    if (blocks == 0) return BR_OK;
    if (blocks > 0x7fffffffULL) return BR_TOO_LARGE;
    const Kv4Place place = {pos, seq_of_token, slots, table, n_seqs, n_slots, table_pages, n_pages};
#define GO(TT, M_, R) rope_kv4_write_kernel<TT, M_, R><<<(unsigned)blocks, 256, 0, s>>>((TT*)qkv, cs, sn, place, (unsigned char*)cache, T, nq, nkv, rd, adjacent, write_cache, (unsigned)kvb)
#define CASE(M_) case M_: if (is_bf16) { if (rot) GO(bf16, M_, true); else GO(bf16, M_, false); } else { if (rot) GO(float, M_, true); else GO(float, M_, false); } break;
    switch (hd / 32) { KV4_SIZES(CASE) }
#undef CASE
#undef GO
    return br_check_launch();
}

extern "C" int br_kv4_read(void* k_out, void* v_out, int is_bf16, const int* pos, const int* seq_of_token, const int* slots, int n_seqs,
                           const int* table, int n_slots, int table_pages, const void* cache, int n_pages, int T, int nkv, int hd, hipStream_t s) {
    if (hd % 32 || hd < 32 || hd > 256 || nkv < 1 || T < 0) return BR_BAD_ARG;
    const unsigned long long blocks = ((unsigned long long)((T + 7) / 8) * 2 * nkv * 8 * (hd / 16) + 255) / 256;
    if (blocks == 0) return BR_OK;
    if (blocks > 0x7fffffffULL) return BR_TOO_LARGE;
    const Kv4Place place = {pos, seq_of_token, slots, table, n_seqs, n_slots, table_pages, n_pages};
#define CASE(M_) case M_: if (is_bf16) kv4_read_kernel<bf16, M_><<<(unsigned)blocks, 256, 0, s>>>((bf16*)k_out, (bf16*)v_out, place, (const unsigned char*)cache, T, nkv); \
                          else kv4_read_kernel<float, M_><<<(unsigned)blocks, 256, 0, s>>>((float*)k_out, (float*)v_out, place, (const unsigned char*)cache, T, nkv); break;
    switch (hd / 32) { KV4_SIZES(CASE) }
#undef CASE
    return br_check_launch();
}
