// Attention over the cache of 4-bit keys and values (layout and number format: kv4.h), on the gfx950 matrix cores.
//
// Per (query row, kv head) the online softmax m' = max(m, s), c = 2^(m - m'), l = l c + p, o = o c + p v with scores in base 2
// (scaled by scale * log2 e once), in float.  Codes become bfloat16 on their way into the matrix instructions: a code times its
// scale is exact there, so keys, values and queries enter exactly and only the probabilities are rounded (to bfloat16, half a
// step of 2^-8 each, which the sum over the keys averages).  The instructions that take 4-bit operands with their scales as they
// are would need the queries as two 8-bit parts, and add their products less exactly: up to 2e-5 of sum |q k| away for normal
// values, against 1e-7 this way.
//
// S^T = K Q^T leaves in a lane the scores of one query for 8 neighbouring tokens, which after exp and rounding are the B operand of
// O^T = V^T P^T as they stand: no exchange between the two products.
//
// What a page's unwritten tokens hold is left over from other sequences and may be NaN: their scores are replaced, not added to, and
// their values are zero before they are multiplied.  Pages that the table does not hold (numbers outside the cache) are left out.
#include "kv4.h"
#include "prefill_order.h"

#define LOG2E 1.4426950408889634f
__device__ __forceinline__ float kv4_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ bf16x8 kv4_zero8() {
    bf16x8 z;
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = (bf16)0.f;
    return z;
}

// What one query's row can see and where its sequence's pages are
struct Kv4Seqs {
    const int* slots;
    const int* ctx_lens;
    const int* table;
    int n_slots, table_pages, n_pages;
};

// ---------------------------------------------------------------------- decode ------
// One token per sequence.  grid = (runs, nkv * blocks of 16 heads, sequences), block = 256: the 4 waves take the pages of a
// run in turn, each with keys and values straight from memory into registers, the next page's in flight while one is
// multiplied, and are joined in LDS in wave order.  Nothing is shared between waves, so nothing passes through LDS before.
// MP: head size / 32 rounded up to a power of two, the lanes' share of a row (8 MP channels); blocks beyond M are zero.
template <int M>
struct Kv4Page {
    static constexpr int MP = M > 4 ? 8 : M == 3 ? 4 : M;
    static constexpr int KS = MP == 8 ? 2 : 1, VSETS = MP == 8 ? 2 : 1;
    unsigned k[4][MP];           // codes of the lane's token in each of the four 16-row tiles
    unsigned ks[KS];             // their scales, a byte a tile
    unsigned v[2][VSETS][8];     // codes of 8 tokens x 8 channels in each half of the page
    u32x2 vs[2][VSETS];          // the 8 tokens' scales

    __device__ __forceinline__ void load(const unsigned char* __restrict__ part, int c, int g) {
        typedef kv4_layout<M> L;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int t = 32 * (j >> 1) + 8 * (c >> 2) + 4 * (j & 1) + (c & 3);
            const unsigned char* row = part + L::KC + t * (16 * M) + g * (4 * MP);
            if constexpr (MP == 1) k[j][0] = *(const unsigned*)row;
            else if constexpr (MP == 2) { const u32x2 w = *(const u32x2*)row; k[j][0] = w[0]; k[j][1] = w[1]; }
            else {
#pragma unroll
                for (int i = 0; i < MP / 4; ++i) {
                    u32x4 w = {0u, 0u, 0u, 0u};
                    if (M == MP || (MP / 4) * g + i < M) w = *(const u32x4*)(row + 16 * i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) k[j][4 * i + e] = w[e];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const int blk = MP == 8 ? 2 * g + i : MP == 4 ? g : MP == 2 ? g >> 1 : 0;
            ks[i] = 0x7f7f7f7fu;
            if (M == MP || blk < M) ks[i] = *(const unsigned*)(part + L::KS + (c * M + blk) * 4);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < VSETS; ++s) {
                const int cg = MP == 8 ? 16 * s + c : MP == 4 ? c : MP == 2 ? c & 7 : c & 3, tg = 4 * h + g;
                u32x4 a = {0u, 0u, 0u, 0u}, b = a;
                vs[h][s] = u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
                if (M == MP || cg < 4 * M) {
                    const unsigned char* at = part + L::VC + (tg * (4 * M) + cg) * 32;
                    a = *(const u32x4*)at;
                    b = *(const u32x4*)(at + 16);
                    vs[h][s] = *(const u32x2*)(part + L::VS + (tg * M + (cg >> 2)) * 8);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) { v[h][s][e] = a[e]; v[h][s][4 + e] = b[e]; }
            }
    }
};

template <int M>
struct Kv4State {
    static constexpr int MP = Kv4Page<M>::MP;
    static constexpr int TILES = 2 * MP;        // 16-row tiles of O^T, a channel of the lane's row each
    bf16x8 q[MP];
    f32x4 o[TILES];
    float m, l;

    // tokens [lo, hi) of the page are seen; `edge`: not all 64
    __device__ __forceinline__ void page(const Kv4Page<M>& p, int lo, int hi, bool edge, float scale2, int c, int g) {
        f32x4 s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < MP; ++w)
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv4_to_bf16(p.k[j][w], kv4_scale((p.ks[MP == 8 ? w >> 2 : 0] >> (8 * j)) & 255u)), q[w],
                                                               s[j], 0, 0, 0);
        }
        // s[j][r]: token 32 (j / 2) + 8 g + 4 (j % 2) + r, head = this lane's column
        if (edge) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int t = 32 * (j >> 1) + 8 * g + 4 * (j & 1) + r;
                    s[j][r] = t >= lo && t < hi ? s[j][r] : -INFINITY;
                }
        }
        float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
        for (int j = 1; j < 4; ++j) mx = fmaxf(mx, fmaxf(fmaxf(s[j][0], s[j][1]), fmaxf(s[j][2], s[j][3])));
        mx = fmaxf(mx, __shfl_xor(mx, 16, WAVE));
        mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE)) * scale2;           // the scale is positive
        const float m_new = fmaxf(m, mx);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        if (__any(m_new > m)) {
            const float corr = kv4_exp2(m - m_use);
            l *= corr;
#pragma unroll
            for (int i = 0; i < TILES; ++i) o[i] *= corr;
        }
        m = m_new;
        float sum = 0.f;
        bf16x8 pr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = kv4_exp2(fmaf(s[2 * h + (e >> 2)][e & 3], scale2, -m_use));
                sum += x;
                pr[h][e] = (bf16)x;
            }
        l += sum;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int st = 0; st < Kv4Page<M>::VSETS; ++st) {
                unsigned v[8];
                float sc[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = p.v[h][st][e];
                    sc[e] = kv4_scale((p.vs[h][st][e >> 2] >> (8 * (e & 3))) & 255u);
                }
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int t = 32 * h + 8 * g + e;
                        const bool ok = t >= lo && t < hi;
                        v[e] = ok ? v[e] : 0u;
                        sc[e] = ok ? sc[e] : 1.f;
                    }
                }
                if constexpr (MP == 2) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] >>= 16 * (c >> 3);
                }
                if constexpr (MP == 1) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] >>= 8 * (c >> 2);
                }
                constexpr int PAIRS = MP >= 4 ? 4 : MP;
                u32x4 a[2 * PAIRS];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    unsigned x, y;
                    kv4_pair<0>(v[2 * e], sc[2 * e], v[2 * e + 1], sc[2 * e + 1], x, y);
                    a[0][e] = x; a[1][e] = y;
                    if constexpr (PAIRS >= 2) { kv4_pair<1>(v[2 * e], sc[2 * e], v[2 * e + 1], sc[2 * e + 1], x, y); a[2][e] = x; a[3][e] = y; }
                    if constexpr (PAIRS >= 4) {
                        kv4_pair<2>(v[2 * e], sc[2 * e], v[2 * e + 1], sc[2 * e + 1], x, y); a[4][e] = x; a[5][e] = y;
                        kv4_pair<3>(v[2 * e], sc[2 * e], v[2 * e + 1], sc[2 * e + 1], x, y); a[6][e] = x; a[7][e] = y;
                    }
                }
#pragma unroll
                for (int i = 0; i < 2 * PAIRS; ++i)
                    o[st * 8 + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[i]), pr[h], o[st * 8 + i], 0, 0, 0);
            }
    }
    // the channel of o[tile]'s row r (0..15)
    static __device__ __forceinline__ int channel(int tile, int r) {
        if constexpr (MP >= 4) return 8 * (r + 16 * (tile >> 3)) + (tile & 7);
        else if constexpr (MP == 2) return 8 * (r & 7) + 4 * (r >> 3) + tile;
        else return 8 * (r & 3) + 2 * (r >> 2) + tile;
    }
};

template <int M>
__global__ __launch_bounds__(256) void attn_decode_kv4_kernel(const bf16* __restrict__ q, size_t q_stride, bf16* __restrict__ out,
                                                              Kv4Seqs seqs, const unsigned char* __restrict__ cache, int nq, int nkv,
                                                              int window, float scale, int nsplit, float* __restrict__ part_o,
                                                              float* __restrict__ part_ml) {
    constexpr int HD = 32 * M, MP = Kv4Page<M>::MP, TILES = Kv4State<M>::TILES;
    typedef kv4_layout<M> L;
    extern __shared__ float lds[];
    const int G = nq / nkv, nhb = (G + 15) / 16;
    const int split = blockIdx.x, kvh = blockIdx.y / nhb, hb = blockIdx.y % nhb, b = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int nheads = (G - hb * 16 < 16) ? G - hb * 16 : 16;
    const int head0 = kvh * G + hb * 16;
    const int slot = seqs.slots[b];
    int ctx = (unsigned)slot < (unsigned)seqs.n_slots ? seqs.ctx_lens[b] : 0;
    if (ctx > seqs.table_pages * KV4_PAGE) ctx = seqs.table_pages * KV4_PAGE;
    const int lo = window > 0 && ctx - window > 0 ? ctx - window : 0;           // the query stands at ctx - 1
    const int pg_lo = lo / KV4_PAGE, npg = ctx > 0 ? (ctx - 1) / KV4_PAGE - pg_lo + 1 : 0;
    const int even = (npg + nsplit - 1) / nsplit, pps = even < 4 ? 4 : even;    // a page for every wave at least
    const int pg_begin = pg_lo + split * pps;
    const int pg_end = pg_begin + pps < pg_lo + npg ? pg_begin + pps : pg_lo + npg;
    if (nsplit > 1 && pg_begin >= pg_end) {             // nothing to add: the join uses no sums of such a run
        if ((int)threadIdx.x < nheads) {
            const size_t at = ((size_t)b * nq + head0 + threadIdx.x) * nsplit + split;
            part_ml[at * 2] = -INFINITY;
            part_ml[at * 2 + 1] = 0.f;
        }
        return;
    }
    Kv4State<M> st;
    const bool head_ok = c < nheads;
    const bf16* qrow = q + (size_t)b * q_stride + (size_t)(head0 + (head_ok ? c : 0)) * HD;
#pragma unroll
    for (int w = 0; w < MP; ++w) {
        const int d = g * (8 * MP) + 8 * w;
        st.q[w] = head_ok && d < HD ? *(const bf16x8*)(qrow + d) : kv4_zero8();
    }
#pragma unroll
    for (int i = 0; i < TILES; ++i) st.o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    st.m = -INFINITY;
    st.l = 0.f;
    const float scale2 = scale * LOG2E;
    const int* bt = seqs.table + (size_t)(slot < 0 ? 0 : slot) * seqs.table_pages;
    for (int pi = pg_begin + wave; pi < pg_end; pi += 4) {
        const int pg = bt[pi];
        if ((unsigned)pg >= (unsigned)seqs.n_pages) continue;
        Kv4Page<M> p;
        p.load(cache + ((size_t)pg * nkv + kvh) * L::BYTES, c, g);
        const int first = pi * KV4_PAGE, a = lo - first > 0 ? lo - first : 0, e = ctx - first < KV4_PAGE ? ctx - first : KV4_PAGE;
        st.page(p, a, e, a > 0 || e < KV4_PAGE, scale2, c, g);
    }
    st.l += __shfl_xor(st.l, 16, WAVE);
    st.l += __shfl_xor(st.l, 32, WAVE);
    // LDS: per wave [16 heads][HD] O, then [16] m, [16] l
    constexpr int WSTRIDE = 16 * HD + 32;
    float* my = lds + wave * WSTRIDE;
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = Kv4State<M>::channel(i, 4 * g + r);
            if (M == MP || d < HD) my[c * HD + d] = st.o[i][r];
        }
    if (g == 0) { my[16 * HD + c] = st.m; my[16 * HD + 16 + c] = st.l; }
    __syncthreads();
    for (int e = threadIdx.x; e < nheads * HD; e += 256) {
        const int h = e / HD, d = e % HD;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mx = fmaxf(mx, lds[w * WSTRIDE + 16 * HD + h]);
        const float use = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = kv4_exp2(lds[w * WSTRIDE + 16 * HD + h] - use);
            sum += lds[w * WSTRIDE + 16 * HD + 16 + h] * f;
            o += lds[w * WSTRIDE + h * HD + d] * f;
        }
        const int head = head0 + h;
        if (nsplit == 1) out[((size_t)b * nq + head) * HD + d] = (bf16)(sum == 0.f ? 0.f : o / sum);
        else {
            const size_t at = ((size_t)b * nq + head) * nsplit + split;
            part_o[at * HD + d] = o;
            if (d == 0) { part_ml[at * 2] = mx; part_ml[at * 2 + 1] = sum; }
        }
    }
}

// The runs of a row added in their order: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.  A wave a row (token, head).
// `last` (null: none): the number of tokens that sequences hold; rows behind them have no runs and stay as they are.
__global__ __launch_bounds__(256) void attn_kv4_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                                            bf16* __restrict__ out, size_t rows, int nq, int hd, int nsplit,
                                                            const int* __restrict__ last) {
    const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows || (last && row >= (size_t)(*last > 0 ? *last : 0) * nq)) return;
    // runs are at most 64, one a lane
    const float m = lane < nsplit ? part_ml[(row * nsplit + lane) * 2] : -INFINITY;
    const float l = lane < nsplit ? part_ml[(row * nsplit + lane) * 2 + 1] : 0.f;
    const float mx = wave_max(m);
    const float f = l == 0.f ? 0.f : kv4_exp2(m - (mx == -INFINITY ? 0.f : mx));
    const float sum = wave_sum(l * f);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int d = lane * 4; d < hd; d += 256) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < nsplit; ++i) {
            const float w = __shfl(f, i, WAVE);
            if (w == 0.f) continue;                           // a run without a token has written no sums
            o += w * *(const f32x4*)(part_o + (row * nsplit + i) * hd + d);
        }
        bf16x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (bf16)(o[e] * inv);
        *(bf16x4*)(out + row * hd + d) = r;
    }
}

// --------------------------------------------------------------------- prefill ------
// Several tokens per sequence.  A workgroup takes 32 NW rows of one kv head and sequence, row = token * G + head, 32 a wave, and
// walks the pages that they see.  A page's codes come to registers while the page before is multiplied, are turned into
// bfloat16 once for all waves and lie in LDS in the order of the matrix operands, 1 KB a wave-read, two pages deep; one barrier a page.
// Chunk [half][k-step][lane] of the keys: 8 channels of the key that row lane % 32 of a 32-key block stands for.  Chunk [32 channels]
// [16 tokens][lane] of the values: 8 tokens of a channel.  (A code and its scale become bfloat16 in half an instruction; read by
// every wave for itself they would cost NW times as many.)
//
// Values that are NaN (scale 255) would spoil rows that do not see them, since 0 * NaN is NaN: a page that holds any is said so, and
// is multiplied with zeros in their place, NaN going into the accumulators of the rows that see them only.
__device__ __forceinline__ int kv4_key_of_row(int c) { return 16 * (c >> 4) + 8 * ((c >> 2) & 1) + 4 * ((c >> 3) & 1) + (c & 3); }
__device__ __forceinline__ int kv4_row_of_key(int u) { return (u & 3) | (((u >> 2) & 1) << 3) | (((u >> 3) & 1) << 2) | (u & 16); }
// Place of a channel's row among a value chunk's 32: turned so that the 16 lanes that write different rows at a time reach different banks
__device__ __forceinline__ int kv4_value_row(int row, int i2) { return row ^ ((row >> 4) | ((i2 & 3) << 1)); }

template <int M, int NW>
__global__ __launch_bounds__(NW * 64) void attn_prefill_kv4_kernel(const bf16* __restrict__ q, size_t q_stride, bf16* __restrict__ out,
                                                                   const int* __restrict__ cu_seqlens, Kv4Seqs seqs,
                                                                   const unsigned char* __restrict__ cache, int nq, int nkv, int window,
                                                                   float scale, const PrefillOrder order, int n_tokens, int nsplit,
                                                                   float* __restrict__ part_o, float* __restrict__ part_ml) {
    constexpr int HD = 32 * M, NT = NW * 64, ROWS = 32 * NW;
    constexpr int KB = KV4_PAGE * HD * 2, STAGE = 2 * KB;                       // bytes of a page's keys; keys and values
    constexpr int UNITS = 64 * M, UPT = (UNITS + NT - 1) / NT;                  // 32-element units of each; per thread
    typedef kv4_layout<M> L;
    extern __shared__ __attribute__((aligned(1024))) unsigned char dsm[];
    int* nan_page = (int*)(dsm + 2 * STAGE);                                    // [2]: the page in a stage that holds NaN values, + 1
    int kvh, b, tile, split = 0;
    if (nsplit > 1) {                                                           // grid (tiles * runs, nkv, B)
        kvh = blockIdx.y;
        b = blockIdx.z;
        tile = blockIdx.x / nsplit;
        split = blockIdx.x % nsplit;
    } else order.place(kvh, b, tile);
    const int t0 = cu_seqlens[b], n_new = cu_seqlens[b + 1] - t0;
    const int G = nq / nkv;
    const long long rows_total = (long long)n_new * G;
    if (t0 < 0 || t0 + n_new > n_tokens || (long long)tile * ROWS >= rows_total) return;        // the whole workgroup leaves together
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row0 = tile * ROWS + wave * 32;
    const int c = lane & 31, g = lane >> 5;
    const int last = (int)rows_total - 1;
    const bool wave_ok = row0 <= last, row_ok = row0 + c <= last;
    const int rr = row_ok ? row0 + c : last;
    const int tok = rr / G, head = kvh * G + rr % G;
    const size_t orow = (size_t)(t0 + tok) * nq + head;
    const int slot = seqs.slots[b];
    const bool there = (unsigned)slot < (unsigned)seqs.n_slots;
    const int ctx = there ? seqs.ctx_lens[b] : 0, start = ctx - n_new;
    const int pq = start + tok;
    const int w_last = row0 + 31 < last ? row0 + 31 : last, g_last = tile * ROWS + ROWS - 1 < last ? tile * ROWS + ROWS - 1 : last;
    const int pq_min_w = start + (wave_ok ? row0 : last) / G, pq_max_w = start + w_last / G;
    const int pq_min_g = start + tile * ROWS / G, pq_max_g = start + g_last / G;
    int first_pg = window > 0 && pq_min_g - window + 1 > 0 ? (pq_min_g - window + 1) / KV4_PAGE : 0;
    int last_pg = pq_max_g < 0 ? -1 : pq_max_g / KV4_PAGE;
    if (last_pg >= seqs.table_pages) last_pg = seqs.table_pages - 1;
    if (!there) last_pg = -1;
    if (nsplit > 1) {
        const int n = last_pg - first_pg + 1, pps = n > 0 ? (n + nsplit - 1) / nsplit : 0;
        first_pg += split * pps;
        if (first_pg + pps - 1 < last_pg) last_pg = first_pg + pps - 1;
    }
    const int* bt = seqs.table + (size_t)(there ? slot : 0) * seqs.table_pages;

    bf16x8 qf[2 * M];
    const bf16* qrow = q + (size_t)(t0 + tok) * q_stride + (size_t)head * HD;
#pragma unroll
    for (int s = 0; s < 2 * M; ++s) qf[s] = *(const bf16x8*)(qrow + s * 16 + 8 * g);
    f32x16 o[M];
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float scale2 = scale * LOG2E;

    // A unit of the keys: a block of a token (token unit % 64, block unit / 64); of the values: 8 tokens of 4 channels, half a group of 8.
    // 16 neighbouring units of the values lie in 16 groups of channels, whose rows reach different banks.
    auto value_cg = [](int u) { return M % 4 == 0 ? (u & 15) + 16 * (u >> 8) : u % (4 * M); };
    auto value_half = [](int u) { return M % 4 == 0 ? (u >> 4) & 1 : u / (32 * M); };
    auto value_tg = [](int u) { return M % 4 == 0 ? (u >> 5) & 7 : u / (4 * M) & 7; };
    u32x4 kr[UPT], va[UPT], vb[UPT];
    u32x2 vsr[UPT];
    unsigned ksr[UPT];
    auto fetch = [&](const unsigned char* part) {
#pragma unroll
        for (int i = 0; i < UPT; ++i) {
            const int u = tid + i * NT;
            if (UNITS % NT == 0 || u < UNITS) {
                const int t = u & 63, blk = u >> 6;
                kr[i] = *(const u32x4*)(part + L::KC + t * (16 * M) + blk * 16);
                ksr[i] = part[L::KS + kv4_key_scale(t, blk, M)];
                const int cg = value_cg(u), tg = value_tg(u);
                const unsigned char* at = part + L::VC + (tg * (4 * M) + cg) * 32;
                va[i] = *(const u32x4*)at;
                vb[i] = *(const u32x4*)(at + 16);
                vsr[i] = *(const u32x2*)(part + L::VS + (tg * M + (cg >> 2)) * 8);
            }
        }
    };
    // `live`: tokens of the page that have been written
    auto put = [&](int buf, int live, int pi) {
        unsigned char* st = dsm + buf * STAGE;
#pragma unroll
        for (int i = 0; i < UPT; ++i) {
            const int u = tid + i * NT;
            if (UNITS % NT == 0 || u < UNITS) {
                const int t = u & 63, blk = u >> 6;
                const float ks = kv4_scale(ksr[i]);
                const int krow = kv4_row_of_key(t & 31);
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    *(bf16x8*)(st + (((t >> 5) * 2 * M + 2 * blk + (w >> 1)) * 64 + (w & 1) * 32 + krow) * 16) = kv4_to_bf16(kr[i][w], ks);
                const int cg = value_cg(u), tg = value_tg(u), half = value_half(u);
                unsigned v[8];
                float sc[8];
                bool nan = false;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const unsigned s8 = (vsr[i][e >> 2] >> (8 * (e & 3))) & 255u;
                    v[e] = (e < 4 ? va[i][e & 3] : vb[i][e & 3]) >> (16 * half);
                    sc[e] = kv4_scale(s8);
                    const bool ok = 8 * tg + e < live;
                    nan |= ok && s8 == 255u;
                    v[e] = ok ? v[e] : 0u;
                    sc[e] = ok ? sc[e] : 1.f;
                }
                if (nan) nan_page[buf] = pi + 1;
                u32x4 a[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    unsigned x, y;
                    kv4_pair<0>(v[2 * e], sc[2 * e], v[2 * e + 1], sc[2 * e + 1], x, y);
                    a[0][e] = x; a[1][e] = y;
                    kv4_pair<1>(v[2 * e], sc[2 * e], v[2 * e + 1], sc[2 * e + 1], x, y);
                    a[2][e] = x; a[3][e] = y;
                }
                const int i2 = cg >> 2;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = (cg & 3) * 8 + half * 4 + e;
                    *(u32x4*)(st + KB + ((i2 * 4 + (tg >> 1)) * 64 + (tg & 1) * 32 + kv4_value_row(row, i2)) * 16) = a[e];
                }
            }
        }
    };
    // the next page from pi on that is there, or last_pg + 1
    auto next_page = [&](int pi) {
        while (pi <= last_pg && (unsigned)bt[pi] >= (unsigned)seqs.n_pages) ++pi;
        return pi;
    };

    if (tid < 2) nan_page[tid] = 0;
    int pi = next_page(first_pg);
    __syncthreads();
    if (pi <= last_pg) {
        fetch(cache + ((size_t)bt[pi] * nkv + kvh) * L::BYTES);
        put(0, ctx - pi * KV4_PAGE, pi);
    }
    __syncthreads();
    for (int buf = 0; pi <= last_pg; buf ^= 1) {
        const int pn = next_page(pi + 1);
        if (pn <= last_pg) fetch(cache + ((size_t)bt[pn] * nkv + kvh) * L::BYTES);
        const unsigned char* st = dsm + buf * STAGE;
        const bool has_nan = nan_page[buf] == pi + 1;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int kb = pi * KV4_PAGE + 32 * half;
            // blocks that no row of this wave sees are skipped
            if (!wave_ok || kb > pq_max_w || (window > 0 && kb + 31 <= pq_min_w - window)) continue;
            f32x16 s;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
            for (int k = 0; k < 2 * M; ++k)
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(st + ((half * 2 * M + k) * 64 + lane) * 16), qf[k], s, 0, 0, 0);
            // s[r]: key kb + 16 (r / 8) + 8 g + r % 8, row = this lane's column
            const bool whole = row0 + 31 <= last && kb + 31 <= pq_min_w && (window <= 0 || kb > pq_max_w - window);
            if (!whole) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = kb + 16 * (r >> 3) + 8 * g + (r & 7);
                    const bool ok = row_ok && key <= pq && (window <= 0 || key > pq - window);
                    s[r] = ok ? s[r] : -INFINITY;
                }
            }
            float mx = fmaxf(fmaxf(s[0], s[1]), s[2]);
#pragma unroll
            for (int r = 3; r < 15; r += 2) mx = fmaxf(fmaxf(mx, s[r]), s[r + 1]);
            mx = fmaxf(mx, s[15]);
            mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE)) * scale2;               // the scale is positive
            const float m_new = fmaxf(m, mx);
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            if (__any(m_new > m)) {
                const float corr = kv4_exp2(m - m_use);
                l *= corr;
#pragma unroll
                for (int i = 0; i < M; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[i][r] *= corr;
            }
            m = m_new;
            float sum0 = 0.f, sum1 = 0.f;
            bf16x8 p[2];
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = kv4_exp2(fmaf(s[r], scale2, -m_use)), y = kv4_exp2(fmaf(s[r + 1], scale2, -m_use));
                sum0 += x;
                sum1 += y;
                p[r >> 3][r & 7] = (bf16)x;
                p[r >> 3][(r & 7) + 1] = (bf16)y;
            }
            l += sum0 + sum1;
#pragma unroll
            for (int i = 0; i < M; ++i)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    bf16x8 v = *(const bf16x8*)(st + KB + ((i * 4 + 2 * half + x) * 64 + 32 * g + kv4_value_row(c, i)) * 16);
                    if (has_nan) {
                        unsigned gone = 0;                              // tokens 16 x + 8 g + e of the half whose block i is NaN
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const bool n = (float)v[e] != (float)v[e];
                            const unsigned long long who = __ballot(n);
                            if ((unsigned)who) gone |= 1u << e;
                            if (who >> 32) gone |= 1u << (8 + e);
                            if (n) v[e] = (bf16)0.f;
                        }
                        bool seen = false;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int key = kb + 16 * x + e;
                            seen |= (gone >> e & 1) && row_ok && key <= pq && (window <= 0 || key > pq - window);
                        }
                        if (seen) {
#pragma unroll
                            for (int r = 0; r < 16; ++r) o[i][r] = NAN;
                        }
                    }
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, p[x], o[i], 0, 0, 0);
                }
        }
        if (pn <= last_pg) put(buf ^ 1, ctx - pn * KV4_PAGE, pn);
        __syncthreads();
        pi = pn;
    }
    l += __shfl_xor(l, 32, WAVE);
    if (!row_ok) return;
    const float inv = nsplit > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
    const size_t at = nsplit > 1 ? orow * nsplit + split : orow;
    if (nsplit > 1 && g == 0) { part_ml[at * 2] = m; part_ml[at * 2 + 1] = l; }
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = i * 32 + 8 * r4 + 4 * g;
            if (nsplit > 1) *(f32x4*)(part_o + at * HD + d) = f32x4{o[i][4 * r4], o[i][4 * r4 + 1], o[i][4 * r4 + 2], o[i][4 * r4 + 3]};
            else {
                bf16x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (bf16)(o[i][4 * r4 + e] * inv);
                *(bf16x4*)(out + at * HD + d) = x;
            }
        }
}

#define KV4_SIZES(F) F(1) F(2) F(3) F(4) F(5) F(6) F(7) F(8)

static int kv4_join(const float* part_o, const float* part_ml, void* out, long long tokens, int nq, int hd, int nsplit, const int* last,
                    hipStream_t s) {
    const size_t rows = (size_t)tokens * nq;
    attn_kv4_join_kernel<<<(unsigned)((rows + 3) / 4), 256, 0, s>>>(part_o, part_ml, (bf16*)out, rows, nq, hd, nsplit, last);
    return br_check_launch();
}

extern "C" int br_attn_decode_kv4(const void* q, size_t q_stride, void* out, const int* slots, const int* ctx_lens, const int* table,
                                  int n_slots, int table_pages, const void* cache, int n_pages, int B, int nq, int nkv, int hd, int window,
                                  float scale, int nsplit, float* part_o, float* part_ml, hipStream_t s) {
    if (hd % 32 || hd < 32 || hd > 256 || nkv < 1 || nq < nkv || nq % nkv || B < 0 || B > 65535 || nsplit < 1 || nsplit > 64 ||
        table_pages > 0x7fffffff / KV4_PAGE || (nsplit > 1 && (!part_o || !part_ml))) return BR_BAD_ARG;
    const int nhb = (nq / nkv + 15) / 16;
    if ((long long)nkv * nhb > 65535) return BR_BAD_ARG;
    if (B == 0) return BR_OK;
    const dim3 grid(nsplit, nkv * nhb, B);
    const size_t lds = 4 * (16 * (size_t)hd + 32) * sizeof(float);
    const Kv4Seqs seqs = {slots, ctx_lens, table, n_slots, table_pages, n_pages};
#define CASE(M_) case M_: \
        if (lds > 65536 && hipFuncSetAttribute((const void*)attn_decode_kv4_kernel<M_>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) return BR_LAUNCH_FAILED; \
        attn_decode_kv4_kernel<M_><<<grid, 256, lds, s>>>((const bf16*)q, q_stride, (bf16*)out, seqs, (const unsigned char*)cache, nq, nkv, window, scale, nsplit, part_o, part_ml); break;
    switch (hd / 32) { KV4_SIZES(CASE) }
#undef CASE
    const int rc = br_check_launch();
    return rc != BR_OK || nsplit == 1 ? rc : kv4_join(part_o, part_ml, out, B, nq, hd, nsplit, nullptr, s);
}

extern "C" int br_attn_prefill_kv4(const void* q, size_t q_stride, void* out, const int* cu_seqlens, const int* slots, const int* ctx_lens,
                                   const int* table, int n_slots, int table_pages, const void* cache, int n_pages, int B, int max_new,
                                   int n_tokens, int nq, int nkv, int hd, int window, float scale, int nsplit, float* part_o, float* part_ml,
                                   hipStream_t s) {
    constexpr int NW = 8;
    if (hd % 32 || hd < 32 || hd > 256 || nkv < 1 || nkv > 65535 || nq < nkv || nq % nkv || B < 0 || B > 65535 || max_new < 0 || nsplit < 1 ||
        nsplit > 64 || table_pages > 0x7fffffff / KV4_PAGE || (long long)n_tokens * nq > 0x7fffffffLL || n_tokens < max_new || (nsplit > 1 && (!part_o || !part_ml))) return BR_BAD_ARG;
    const long long rows = (long long)max_new * (nq / nkv);
    if (rows > 0x7fffffffLL - 32 * NW) return BR_BAD_ARG;
    if (B == 0 || max_new == 0) return BR_OK;
    PrefillOrder order = {};
    dim3 grid;
    // the order counts in tiles of 128 rows: half as many rows in tiles of twice as many
    if (!prefill_order(order, grid, (rows + 1) / 2, nkv, B, br_device_cus(), hd <= 128 ? 2 : 1)) return BR_BAD_ARG;
    if (nsplit > 1) {
        const long long x = (rows + 32 * NW - 1) / (32 * NW) * nsplit;
        if (x > 0x7fffffffLL) return BR_BAD_ARG;
        grid = dim3((unsigned)x, nkv, B);
    }
    const size_t lds = 2 * (size_t)2 * KV4_PAGE * hd * 2 + 16;
    const Kv4Seqs seqs = {slots, ctx_lens, table, n_slots, table_pages, n_pages};
#define CASE(M_) case M_: \
        if (hipFuncSetAttribute((const void*)attn_prefill_kv4_kernel<M_, NW>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) return BR_LAUNCH_FAILED; \
        attn_prefill_kv4_kernel<M_, NW><<<grid, NW * 64, lds, s>>>((const bf16*)q, q_stride, (bf16*)out, cu_seqlens, seqs, (const unsigned char*)cache, nq, nkv, window, scale, order, n_tokens, nsplit, part_o, part_ml); break;
    switch (hd / 32) { KV4_SIZES(CASE) }
#undef CASE
    const int rc = br_check_launch();
    return rc != BR_OK || nsplit == 1 ? rc : kv4_join(part_o, part_ml, out, n_tokens, nq, hd, nsplit, cu_seqlens + B, s);
}
