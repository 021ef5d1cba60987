// Rows into and out of the cache of 4-bit keys and values (layout and number format: kv4.h).
//
// Writing: x -> E = clamp(floor(log2 max|x|) - 2, -124, 125) of its 32 neighbours, the code nearest to x / 2^E (ties to the even
// code; the hardware's conversion).  The largest magnitude is taken of the floats' bits as integers: infinities and NaN come
// out above every number, and its exponent is their upper bits.
#include "kv4.h"

// 8 elements of a row: one or two 16-byte loads or stores a lane, neighbouring lanes side by side
template <typename T> __device__ __forceinline__ void kv4_load8(const T* p, float* v) { ew_load<T, 4>(p, v); ew_load<T, 4>(p + 4, v + 4); }
template <> __device__ __forceinline__ void kv4_load8<bf16>(const bf16* p, float* v) {
    const bf16x8 q = *(const bf16x8*)p;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)q[e];
}
// (rows read back are stored around the caches: 32,768 tokens of 8 heads of 128 in 27.5 us, stored through them 47.7 us)
template <typename T> __device__ __forceinline__ void kv4_store8(T* p, unsigned w, float scale) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
    __builtin_nontemporal_store(f32x4{a[0], a[1], b[0], b[1]}, (f32x4*)p);
    __builtin_nontemporal_store(f32x4{c[0], c[1], d[0], d[1]}, (f32x4*)(p + 4));
}
template <> __device__ __forceinline__ void kv4_store8<bf16>(bf16* p, unsigned w, float scale) { __builtin_nontemporal_store(kv4_to_bf16(w, scale), (bf16x8*)p); }

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

// A lane takes elements of a key or value row 8 at a time (a quarter of a block), LANES neighbouring lanes a run of a token's row, and so
// on with the row's CHUNKS runs; 8 tokens lie in a wave, so that its stores fill the 32 bytes that 8 tokens of 8 value channels are.
template <int M> struct Kv4Rows {
    static constexpr int HD = 32 * M, LANES = M % 2 ? 4 : 8, CHUNKS = 4 * M / LANES, HEADS = 256 / (8 * LANES);
    int lane, head;
    long long token;
    __device__ __forceinline__ Kv4Rows() {
        const int u = threadIdx.x;
        lane = u % LANES;
        head = blockIdx.x * HEADS + u / (8 * LANES);
        token = ((long long)blockIdx.z * gridDim.y + blockIdx.y) * 8 + u / LANES % 8;
    }
    __device__ __forceinline__ int piece(int j) const { return lane + LANES * j; }
    static bool grid(dim3& g, long long tokens, int heads) {
        const long long n = (tokens + 7) / 8, y = n < 32768 ? n : 32768;
        g = dim3((unsigned)((heads + HEADS - 1) / HEADS), (unsigned)y, (unsigned)((n + y - 1) / (y ? y : 1)));
        return n <= 32768LL * 65535;
    }
};

// 8 pairs of one query head rotated in place: pairs 8 w .. of `row`.
template <typename T>
__device__ __forceinline__ void kv4_rotate_pairs(T* row, const float* c, const float* s, int w, int P, bool adjacent) {
    if (8 * w + 8 <= P && (adjacent || P % 8 == 0)) {
        // 8 pairs whole: neighbours are 16 elements in a row, halves 8 and 8
        float a[8], b[8], co[8], si[8];
        T* lo = row + (adjacent ? 16 * w : 8 * w);
        T* hi = adjacent ? lo + 8 : lo + P;
        kv4_load8<T>(lo, a);
        kv4_load8<T>(hi, b);
        if (P % 4 == 0) {
            kv4_load8<float>(c + 8 * w, co);
            kv4_load8<float>(s + 8 * w, si);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) { co[e] = c[8 * w + e]; si[e] = s[8 * w + e]; }
        }
        float x[16], y[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float f = adjacent ? (e < 4 ? a[2 * (e & 3)] : b[2 * (e & 3)]) : a[e];
            const float g = adjacent ? (e < 4 ? a[2 * (e & 3) + 1] : b[2 * (e & 3) + 1]) : b[e];
            x[e] = f * co[e] - g * si[e];
            x[8 + e] = f * si[e] + g * co[e];
        }
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
}

// ROT: the keys are rotated first (pairs (p, p + rd / 2), or neighbours when `adjacent`).  They are rounded to the rows' type before
// they are held, as the cache of that type holds them.  The first `kv_blocks` columns of the grid take keys and values; the others
// rotate the queries of the same 8 tokens where they stand.  A row and the look-up of its page are on their way together, and of 128
// and 256 channels a lane loads both halves of its pairs once: what is moved bounds the launch (16,384 rows of 32 + 2 x 8 heads of 128
// in 68 us, 5.3 TB/s of the bytes it has to move, the rate of a copy; the same rows again and again, partly from the caches, 58; 8 rows 3.2
// us, which is what a launch and two dependent loads take).
template <typename T, int M, bool ROT>
__global__ __launch_bounds__(256) void kv4_write_kernel(T* __restrict__ qkv, const float* __restrict__ cs, const float* __restrict__ sn,
                                                        Kv4Place place, unsigned char* __restrict__ cache, long long n_tokens, int nq,
                                                        int nkv, int rd, int adjacent, int kv_blocks) {
    typedef kv4_layout<M> L;
    typedef Kv4Rows<M> R;
    const size_t width = (size_t)(nq + 2 * nkv) * R::HD;
    const int P = rd / 2;
    if (ROT && (int)blockIdx.x >= kv_blocks) {
        const int units = (P + 7) / 8, u = ((int)blockIdx.x - kv_blocks) * 256 + threadIdx.x, th = u / units;
        const long long t = ((long long)blockIdx.z * gridDim.y + blockIdx.y) * 8 + th / nq;
        if (th < 8 * nq && t < n_tokens) kv4_rotate_pairs<T>(qkv + (size_t)t * width + (size_t)(th % nq) * R::HD, cs + t * P, sn + t * P, u % units, P, adjacent);
        return;
    }
    const R at;
    const int head = at.head;
    const bool is_k = head < nkv, row_there = at.token < n_tokens && head < 2 * nkv;
    const T* row = qkv + (size_t)at.token * width + (size_t)(nq + head) * R::HD;
    float x[R::CHUNKS][8];
#pragma unroll
    for (int j = 0; j < R::CHUNKS; ++j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[j][e] = 0.f;
        if (row_there) kv4_load8<T>(row + at.piece(j) * 8, x[j]);
    }
    int page = 0, p = 0;
    // lanes without a row stay for the exchange of the maxima: the lanes of a block store together or not at all
    const bool ok = row_there && place.find((int)at.token, page, p);
    unsigned char* part = cache + ((size_t)page * nkv + (is_k ? head : head - nkv)) * L::BYTES;
    // The usual rotation of 128 and 256 channels whole: a lane holds both halves of its pairs.
    const bool held = M % 4 == 0 && ROT && rd == R::HD && !adjacent, turn = ROT && ok && is_k;
    const float* c = cs + (size_t)at.token * P;
    const float* s = sn + (size_t)at.token * P;
    if constexpr (M % 4 == 0 && ROT) if (held && turn) {
#pragma unroll
        for (int j = 0; j < R::CHUNKS / 2; ++j) {
            float co[8], si[8];
            kv4_load8<float>(c + at.piece(j) * 8, co);
            kv4_load8<float>(s + at.piece(j) * 8, si);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float a = x[j][e], b = x[j + R::CHUNKS / 2][e];
                x[j][e] = to_f32<T>(from_f32<T>(a * co[e] - b * si[e]));
                x[j + R::CHUNKS / 2][e] = to_f32<T>(from_f32<T>(a * si[e] + b * co[e]));
            }
        }
    }
#pragma unroll
    for (int j = 0; j < R::CHUNKS; ++j) {
        float* v = x[j];
        const int piece = at.piece(j), d0 = piece * 8;
        if (turn && !held && d0 < rd) {
            if (adjacent) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    if (d0 + e >= rd) break;
                    const float a = v[e], b = v[e + 1], co = c[(d0 + e) / 2], si = s[(d0 + e) / 2];
                    v[e] = to_f32<T>(from_f32<T>(a * co - b * si));
                    v[e + 1] = to_f32<T>(from_f32<T>(a * si + b * co));
                }
            } else if (P % 8 == 0) {
                const bool low = d0 < P;
                const int p0 = low ? d0 : d0 - P;
                float y[8], co[8], si[8];
                kv4_load8<T>(row + (low ? d0 + P : d0 - P), y);
                kv4_load8<float>(c + p0, co);
                kv4_load8<float>(s + p0, si);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = to_f32<T>(from_f32<T>(low ? v[e] * co[e] - y[e] * si[e] : y[e] * si[e] + v[e] * co[e]));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = d0 + e;
                    if (d >= rd) break;
                    const bool low = d < P;
                    const int k = low ? d : d - P;
                    const float y = to_f32<T>(row[low ? d + P : d - P]);
                    v[e] = to_f32<T>(from_f32<T>(low ? v[e] * c[k] - y * s[k] : y * s[k] + v[e] * c[k]));
                }
            }
        }
        unsigned big = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned b = __float_as_uint(v[e]) & 0x7fffffffu;
            big = b > big ? b : big;
        }
        unsigned other = (unsigned)__shfl_xor((int)big, 1, WAVE);
        big = other > big ? other : big;
        other = (unsigned)__shfl_xor((int)big, 2, WAVE);
        big = other > big ? other : big;
        if (!ok) continue;
        const bool finite = big < 0x7f800000u;
        int byte = (int)(big >> 23) - 2;                 // 127 + floor(log2(big)) - 2
        byte = byte < 3 ? 3 : byte;
        const float scale = kv4_scale(byte);
        unsigned w = 0u;
        if (finite) {
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
        }
        *(unsigned*)(part + (is_k ? L::KC + p * (16 * M) + piece * 4 : L::VC + ((p >> 3) * (4 * M) + piece) * 32 + (p & 7) * 4)) = w;
        if (!(piece & 3)) part[is_k ? L::KS + kv4_key_scale(p, piece >> 2, M) : L::VS + ((p >> 3) * M + (piece >> 2)) * 8 + (p & 7)] = (unsigned char)(finite ? byte : 255);
    }
}

// Rows out of the pages, the same lanes the other way round.  What is moved bounds it: 32,768 tokens of 8 heads of 128 in 25.6 us, 6.6 TB/s;
// 777 tokens 3.3 us.
template <typename T, int M>
__global__ __launch_bounds__(256) void kv4_read_kernel(T* __restrict__ k_out, T* __restrict__ v_out, Kv4Place place,
                                                       const unsigned char* __restrict__ cache, long long n_tokens, int nkv) {
    typedef kv4_layout<M> L;
    typedef Kv4Rows<M> R;
    const R at;
    int page = 0, p = 0;
    if (at.token >= n_tokens || at.head >= 2 * nkv || !place.find((int)at.token, page, p)) return;
    const bool is_k = at.head < nkv;
    const int head = is_k ? at.head : at.head - nkv;
    const unsigned char* part = cache + ((size_t)page * nkv + head) * L::BYTES;
    T* row = (is_k ? k_out : v_out) + ((size_t)at.token * nkv + head) * R::HD;
    unsigned w[R::CHUNKS];
    unsigned char byte[R::CHUNKS];
#pragma unroll
    for (int j = 0; j < R::CHUNKS; ++j) {
        const int piece = at.piece(j);
        w[j] = *(const unsigned*)(part + (is_k ? L::KC + p * (16 * M) + piece * 4 : L::VC + ((p >> 3) * (4 * M) + piece) * 32 + (p & 7) * 4));
        byte[j] = part[is_k ? L::KS + kv4_key_scale(p, piece >> 2, M) : L::VS + ((p >> 3) * M + (piece >> 2)) * 8 + (p & 7)];
    }
#pragma unroll
    for (int j = 0; j < R::CHUNKS; ++j) kv4_store8<T>(row + at.piece(j) * 8, w[j], kv4_scale(byte[j]));
}

#define KV4_SIZES(F) F(1) F(2) F(3) F(4) F(5) F(6) F(7) F(8)

extern "C" int br_rope_kv4_write(void* qkv, int is_bf16, const float* cs, const float* sn, const int* pos, const int* seq_of_token,
                                 const int* slots, int n_seqs, const int* table, int n_slots, int table_pages, void* cache, int n_pages,
                                 int T, int nq, int nkv, int hd, int rd, int adjacent, int write_cache, hipStream_t s) {
    if (hd % 32 || hd < 32 || hd > 256 || rd < 0 || rd > hd || rd % 2 || nq < 0 || nkv < 1 || T < 0) return BR_BAD_ARG;
    const bool rot = cs && rd > 0;
    const long long turns = rot ? ((long long)8 * nq * ((rd / 2 + 7) / 8) + 255) / 256 : 0;
    if (turns > 0x3fffffff) return BR_TOO_LARGE;
    if (T == 0 || (!turns && !write_cache)) return BR_OK;
    const Kv4Place place = {pos, seq_of_token, slots, table, n_seqs, n_slots, table_pages, n_pages};
    dim3 grid;
#define GO(TT, M_, R) kv4_write_kernel<TT, M_, R><<<grid, 256, 0, s>>>((TT*)qkv, cs, sn, place, (unsigned char*)cache, T, nq, nkv, rd, adjacent, kv_blocks)
#define CASE(M_) case M_: { \
        if (!Kv4Rows<M_>::grid(grid, T, 2 * nkv)) return BR_TOO_LARGE; \
        const int kv_blocks = write_cache ? (int)grid.x : 0; \
        grid.x = (unsigned)(kv_blocks + turns); \
        if (is_bf16) { if (rot) GO(bf16, M_, true); else GO(bf16, M_, false); } else { if (rot) GO(float, M_, true); else GO(float, M_, false); } } break;
    switch (hd / 32) { KV4_SIZES(CASE) }
#undef CASE
#undef GO
    return br_check_launch();
}

extern "C" int br_kv4_read(void* k_out, void* v_out, int is_bf16, const int* pos, const int* seq_of_token, const int* slots, int n_seqs,
                           const int* table, int n_slots, int table_pages, const void* cache, int n_pages, int T, int nkv, int hd, hipStream_t s) {
    if (hd % 32 || hd < 32 || hd > 256 || nkv < 1 || T < 0) return BR_BAD_ARG;
    if (T == 0) return BR_OK;
    const Kv4Place place = {pos, seq_of_token, slots, table, n_seqs, n_slots, table_pages, n_pages};
    dim3 grid;
#define CASE(M_) case M_: if (!Kv4Rows<M_>::grid(grid, T, 2 * nkv)) return BR_TOO_LARGE; \
        if (is_bf16) kv4_read_kernel<bf16, M_><<<grid, 256, 0, s>>>((bf16*)k_out, (bf16*)v_out, place, (const unsigned char*)cache, T, nkv); \
        else kv4_read_kernel<float, M_><<<grid, 256, 0, s>>>((float*)k_out, (float*)v_out, place, (const unsigned char*)cache, T, nkv); break;
    switch (hd / 32) { KV4_SIZES(CASE) }
#undef CASE
    return br_check_launch();
}
