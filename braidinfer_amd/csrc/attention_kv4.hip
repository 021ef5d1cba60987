// Attention over the cache of 4-bit keys and values (layout and number format: kv4.h), on the gfx950 matrix cores.
//
// Per (query row, kv head) the online softmax c = 2^(m - m'), l = l c + p, o = o c + p v, p = 2^(s - m') with scores in base 2
// (scaled by scale * log2 e once) and m' no less than any of them, in float.  Codes become bfloat16 on their way into the matrix instructions: a code times its
// scale is exact there, so keys, values and queries enter exactly and only the probabilities are rounded (to bfloat16, half a
// step of 2^-8 each, which the sum over the keys averages; their sum l is taken of the rounded ones).  The instructions that take 4-bit operands with their scales as they
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
#define KV4_ABOVE 8.f
__device__ __forceinline__ float kv4_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ bf16x8 kv4_zero8() {
    bf16x8 z;
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = (bf16)0.f;
    return z;
}

// sum + p[0] + p[1] in float.  The weights' sum is taken of the weights as they are rounded for the product with the values: what rounding
// does to a weight that outweighs the others then goes out again in the division.
__device__ __forceinline__ float kv4_add_pair(bf16x2 p, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(p, bf16x2{(bf16)1.f, (bf16)1.f}, sum, false);
}

// A word that all lanes ask for, through the scalar cache: such a load neither waits for the vector loads in flight nor holds them up.
// (Nothing that a kernel here reads this way is written while it runs.)
__device__ __forceinline__ int kv4_uniform(const int* p) { return *(const __attribute__((address_space(4))) int*)p; }

// A barrier that orders what lies in LDS and no more: loads from memory stay in flight over it (__syncthreads waits for them).
__device__ __forceinline__ void kv4_lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// What one query's row can see and where its sequence's pages are
struct Kv4Seqs {
    const int* slots;
    const int* ctx_lens;
    const int* table;
    int n_slots, table_pages, n_pages;
};

// ---------------------------------------------------------------------- decode ------
// One token per sequence.  All pages that a step's tokens see, sequence by sequence for one kv head (and block of GB query heads), then for the
// next, are one list, of which every workgroup takes as many places in a row: with runs by the longest sequence, or as many for each, those of a
// batch of unequal lengths differ several times in length, and a workgroup's start (its lengths, table, first page: one wait for the
// memory each) is paid again for every run.  The lists' lengths are on the device only, so each workgroup adds them up for itself.
// A sequence and group take KV4_SWITCH places more than their pages, in front of them: what it costs to begin with another one
// (queries, maxima, joining the waves), in pages.
#define KV4_SWITCH 4
struct Kv4Runs {
    int B, window, groups, wgs, nsplit;          // groups: kv heads x blocks of query heads; nsplit: pieces that a sequence may come in
    float per_wg, per_piece;                     // a little more than groups / wgs and 1 / (nsplit - 1)

    // sequence b's context, the first token that it sees, and the pages between
    __device__ __forceinline__ int pages(const Kv4Seqs& s, int slot, int length, int& ctx, int& lo) const {
        ctx = length;
        if ((unsigned)slot >= (unsigned)s.n_slots || ctx < 0) ctx = 0;
        if (ctx > s.table_pages * KV4_PAGE) ctx = s.table_pages * KV4_PAGE;
        lo = window > 0 && ctx - window > 0 ? ctx - window : 0;                // the query stands at ctx - 1
        return ctx > 0 ? (ctx - 1) / KV4_PAGE - lo / KV4_PAGE + 1 : 0;
    }
    // inclusive sums and maxima over the lanes
    static __device__ __forceinline__ int scan(int x) {
        x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);       // from the lane 1, 2, 4, 8 below in a row of 16
        x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
        x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
        x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
        x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);      // a row's last lane to the next row, rows 1 and 3
        x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);      // lane 31 to rows 2 and 3
        return x;
    }
    static __device__ __forceinline__ int most(int x) {                      // of numbers that are not negative; in lane 63
        auto up = [](int a, int b) { return a > b ? a : b; };
        x = up(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true));
        x = up(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true));
        x = up(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true));
        x = up(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true));
        x = up(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
        return up(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
    }
};

// The list, as a wave sees it: lane i holds sequence base + i.
struct Kv4List {
    int slot, length;               // of the lane's sequence
    int n, upto, base;              // its places in a group's part of the list, and of all up to it
    int total, p;                   // places of a group's part; places that a workgroup takes

    static __device__ __forceinline__ int places(const Kv4Runs& r, const Kv4Seqs& s, int slot, int length) {
        int ctx, lo;
        const int n = r.pages(s, slot, length, ctx, lo);
        return n ? n + KV4_SWITCH : 0;
    }
    __device__ __forceinline__ void at(const Kv4Runs& r, const Kv4Seqs& s, int from, int sum, int lane) {
        base = from;
        slot = from + lane < r.B ? s.slots[from + lane] : -1;
        length = from + lane < r.B ? s.ctx_lens[from + lane] : 0;
        n = places(r, s, slot, length);
        upto = sum + Kv4Runs::scan(n);
    }
    __device__ __forceinline__ int end() const { return __builtin_amdgcn_readlane(upto, 63); }
    __device__ __forceinline__ void start(const Kv4Runs& r, const Kv4Seqs& s, int lane) {
        at(r, s, 0, 0, lane);
        int longest = n, sum = n;
        total = end();
        if (r.B > WAVE) {
            for (int b = WAVE + lane; b < r.B; b += WAVE) {
                const int x = places(r, s, s.slots[b], s.ctx_lens[b]);
                longest = longest > x ? longest : x;
                sum += x;
            }
            total = __builtin_amdgcn_readlane(Kv4Runs::scan(sum), 63);
        }
        longest = __builtin_amdgcn_readlane(Kv4Runs::most(longest), 63);
        // an even share, a page for each wave at least, and no sequence in more than nsplit pieces (it may begin and end inside a
        // workgroup's places); the factors are rounded up, so a product that is cut off is the share or more once 1 is added
        p = 4 + KV4_SWITCH;
        const int even = (int)((float)total * r.per_wg) + 1, least = (int)((float)longest * r.per_piece) + 1;
        p = p > even ? p : even;
        p = p > least ? p : least;
    }
    // the sequence that holds place y of a group's part, its places and the place where they begin; y does not fall but to 0
    __device__ __forceinline__ int find(const Kv4Runs& r, const Kv4Seqs& s, int y, int& own, int& first, int& its_slot, int& its_length, int lane) {
        if (y < __builtin_amdgcn_readlane(upto, 0) - __builtin_amdgcn_readlane(n, 0)) at(r, s, 0, 0, lane);
        while (y >= end()) at(r, s, base + WAVE, end(), lane);
        const int i = __builtin_ctzll(__ballot(upto > y));
        own = __builtin_amdgcn_readlane(n, i);
        first = __builtin_amdgcn_readlane(upto, i) - own;
        its_slot = __builtin_amdgcn_readlane(slot, i);
        its_length = __builtin_amdgcn_readlane(length, i);
        return base + i;
    }
};

// Place C behind lane offset `off` of a part: a uniform base, 32 bits of offset a lane and what an instruction holds of the rest.
template <int C> __device__ __forceinline__ const unsigned char* kv4_at(const unsigned char* part, unsigned off) {
    if constexpr (C < 4064) return part + off + C;
    else return part + (off + (unsigned)C);
}
// Where a lane's share of a page begins: row c, quarter g (see kv4.h)
template <int M>
struct Kv4Lane {
    int c, g;
    unsigned k, ks, v, vs;
    __device__ __forceinline__ Kv4Lane(int lane) : c(lane & 15), g(lane >> 4) {
        typedef kv4_layout<M> L;
        constexpr int MP = M > 4 ? 8 : M == 3 ? 4 : M;
        const int blk = MP == 8 ? 2 * g : MP == 4 ? g : MP == 2 ? g >> 1 : 0, cg = MP >= 4 ? c : MP == 2 ? c & 7 : c & 3;
        k = (8 * (c >> 2) + (c & 3)) * (16 * M) + g * (4 * MP) + L::KC;
        ks = (c * M + blk) * 4 + L::KS;
        v = (g * (4 * M) + cg) * 32 + L::VC;
        vs = (g * M + (cg >> 2)) * 8 + L::VS;
        asm volatile("" : "+v"(k), "+v"(ks), "+v"(v), "+v"(vs));           // kept, not worked out again for every load
    }
};

// MP: head size / 32 rounded up to a power of two, the lanes' share of a row (8 MP channels); blocks beyond M are zero.
template <int M>
struct Kv4Keys {
    static constexpr int MP = M > 4 ? 8 : M == 3 ? 4 : M, KS = MP == 8 ? 2 : 1;
    unsigned k[4][MP];           // codes of the lane's token in each of the page's four 16-row tiles
    unsigned ks[KS];             // their scales, a byte a tile

    __device__ __forceinline__ void load(const unsigned char* __restrict__ part, const Kv4Lane<M>& lane) {
        typedef kv4_layout<M> L;
        load<0>(part, lane);
        load<1>(part, lane);
        load<2>(part, lane);
        load<3>(part, lane);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            ks[i] = 0x7f7f7f7fu;
            if (M == MP || KS * lane.g + i < M) ks[i] = __builtin_nontemporal_load((const unsigned*)(part + lane.ks + 4 * i));
        }
    }
    template <int J> __device__ __forceinline__ void load(const unsigned char* __restrict__ part, const Kv4Lane<M>& lane) {
        const unsigned char* row = kv4_at<(32 * (J >> 1) + 4 * (J & 1)) * (16 * M)>(part, lane.k);
        if constexpr (MP == 1) k[J][0] = __builtin_nontemporal_load((const unsigned*)row);
        else if constexpr (MP == 2) { const u32x2 w = __builtin_nontemporal_load((const u32x2*)row); k[J][0] = w[0]; k[J][1] = w[1]; }
        else {
#pragma unroll
            for (int i = 0; i < MP / 4; ++i) {
                u32x4 w = {0u, 0u, 0u, 0u};
                if (M == MP || (MP / 4) * lane.g + i < M) w = __builtin_nontemporal_load((const u32x4*)(row + 16 * i));
#pragma unroll
                for (int e = 0; e < 4; ++e) k[J][4 * i + e] = w[e];
            }
        }
    }
};
template <int M>
struct Kv4Values {
    static constexpr int MP = Kv4Keys<M>::MP, SETS = MP == 8 ? 2 : 1;
    unsigned v[SETS][8];         // codes of 8 tokens x 8 channels of half a page
    u32x2 vs[SETS];              // the 8 tokens' scales

    template <int H> __device__ __forceinline__ void load(const unsigned char* __restrict__ part, const Kv4Lane<M>& lane) {
        set<H, 0>(part, lane);
        if constexpr (SETS == 2) set<H, 1>(part, lane);
    }
    template <int H, int S> __device__ __forceinline__ void set(const unsigned char* __restrict__ part, const Kv4Lane<M>& lane) {
        u32x4 a = {0u, 0u, 0u, 0u}, b = a;
        vs[S] = u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
        if (M == MP || 16 * S + lane.c < 4 * M) {
            const unsigned char* at = kv4_at<H * (512 * M) + S * 512>(part, lane.v);
            a = __builtin_nontemporal_load((const u32x4*)at);
            b = __builtin_nontemporal_load((const u32x4*)(at + 16));
            vs[S] = __builtin_nontemporal_load((const u32x2*)(kv4_at<H * (32 * M) + S * 32>(part, lane.vs)));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[S][e] = a[e]; v[S][4 + e] = b[e]; }
    }
};

// GB heads are the columns of the products.  With 4 or 8 of them the 16 columns hold them NK = 4 or 2 times over, and a lane works on
// the scores of its copy's own tiles only, 16 / GB of the page's tokens each.  Two of the copies then split the values' channels: a
// converted byte of codes is two channels of one token, and as two neighbouring k-slots of A it meets (p, 0) in the even copy's
// columns, which gives the one channel, and (0, p) in the odd one's, which gives the other.  So nothing is moved from pairs of channels to
// pairs of tokens, there are half as many accumulators, and a quarter (half) of the exponentials of a product whose
// columns are copies or empty: 270 vector instructions a page and wave for 4 heads of 128 instead of 420.
template <int M, int GB>
struct Kv4State {
    static constexpr int MP = Kv4Keys<M>::MP, NK = 16 / GB, OWN = 4 / NK;
    static constexpr bool SPLIT = GB < 16;
    static constexpr int TILES = SPLIT ? MP : 2 * MP;
    bf16x8 q[MP];
    f32x4 o[TILES];
    float m, l;
    bf16x8 pr[2];                  // weights of a page: GB 16, by halves
    unsigned pw[OWN][2];           // GB 4, 8: of the lane's own tiles, two tokens a word

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < TILES; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        m = -INFINITY;
        l = 0.f;
    }
    // the largest of (or the sum over) the lanes of a head
    static __device__ __forceinline__ float largest(float x) {
        if constexpr (GB == 4) x = fmaxf(x, __shfl_xor(x, 4, WAVE));
        if constexpr (GB <= 8) x = fmaxf(x, __shfl_xor(x, 8, WAVE));
        x = fmaxf(x, __shfl_xor(x, 16, WAVE));
        return fmaxf(x, __shfl_xor(x, 32, WAVE));
    }
    static __device__ __forceinline__ float sum(float x) {
        if constexpr (GB == 4) x += __shfl_xor(x, 4, WAVE);
        if constexpr (GB <= 8) x += __shfl_xor(x, 8, WAVE);
        x += __shfl_xor(x, 16, WAVE);
        return x + __shfl_xor(x, 32, WAVE);
    }
    // s[j][r]: token 32 (j / 2) + 8 g + 4 (j % 2) + r, head = this lane's column
    __device__ __forceinline__ void scores(const Kv4Keys<M>& p, f32x4* s) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < MP; ++w)
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv4_to_bf16(p.k[j][w], kv4_scale_of(p.ks[MP == 8 ? w >> 2 : 0], j)), q[w],
                                                               s[j], 0, 0, 0);
        }
    }
    // tokens [lo, hi) of the page are seen; `edge`: not all 64
    __device__ __forceinline__ void weights(const f32x4* s, int lo, int hi, bool edge, float scale2, int c, int g) {
        const int k = c / GB;
        f32x4 t[OWN];
#pragma unroll
        for (int i = 0; i < OWN; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (GB == 4) t[i][r] = k < 2 ? (k == 0 ? s[0][r] : s[1][r]) : (k == 2 ? s[2][r] : s[3][r]);
                else if constexpr (GB == 8) t[i][r] = k == 0 ? s[2 * i][r] : s[2 * i + 1][r];
                else t[i][r] = s[i][r];
            }
        if (edge) {
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                const int j = GB == 4 ? k : GB == 8 ? 2 * i + k : i, first = 32 * (j >> 1) + 8 * g + 4 * (j & 1);
                const int a = lo - first, e = hi - first;
#pragma unroll
                for (int r = 0; r < 4; ++r) t[i][r] = r >= a && r < e ? t[i][r] : -INFINITY;
            }
        }
        float mx = fmaxf(fmaxf(t[0][0], t[0][1]), fmaxf(t[0][2], t[0][3]));
#pragma unroll
        for (int i = 1; i < OWN; ++i) mx = fmaxf(mx, fmaxf(fmaxf(t[i][0], t[i][1]), fmaxf(t[i][2], t[i][3])));
        mx *= scale2;                                                // the scale is positive
        // What is subtracted need not be the largest score: it is KV4_ABOVE powers of two beyond the largest one of the time it was chosen, and the
        // lanes' maxima are brought together, and the sums rescaled, only when a score is beyond it.  Weights of 2^-KV4_ABOVE lose
        // nothing in float or bfloat16, and none is above 1: sums of weights and values stay within what the values themselves reach.
        if (__any(mx > m)) {
            const float m_new = fmaxf(m, largest(mx) + KV4_ABOVE);
            const float corr = m_new == -INFINITY ? 1.f : kv4_exp2(m - m_new);
            m = m_new;
            l *= corr;
#pragma unroll
            for (int i = 0; i < TILES; ++i) o[i] *= corr;
        }
        const float m_use = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            float x[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[r] = kv4_exp2(fmaf(t[i][r], scale2, -m_use));
            }
            const bf16x2 a = {(bf16)x[0], (bf16)x[1]}, b = {(bf16)x[2], (bf16)x[3]};
            l = kv4_add_pair(b, kv4_add_pair(a, l));
            if constexpr (SPLIT) {
                pw[i][0] = __builtin_bit_cast(unsigned, a);
                pw[i][1] = __builtin_bit_cast(unsigned, b);
            } else {
                bf16x8& p = pr[i >> 1];
                p[4 * (i & 1)] = a[0]; p[4 * (i & 1) + 1] = a[1]; p[4 * (i & 1) + 2] = b[0]; p[4 * (i & 1) + 3] = b[1];
            }
        }
    }
    // SPLIT: B of tile J, (p, 0) in the first copy's columns and (0, p) in the second's; sel: `perm`'s selectors that say so
    template <int J>
    __device__ __forceinline__ bf16x8 operand(unsigned sel0, unsigned sel1) const {
        u32x4 b;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            unsigned u = pw[GB == 8 ? J >> 1 : 0][x], v = u;
            // from the copy that worked on tile J: lanes of a row of 16 take the value 4, 8 or 12 lanes on (0x100 +) or back (0x110 +)
            if constexpr (GB == 8) {
                if constexpr (J & 1) v = __builtin_amdgcn_update_dpp(u, u, 0x108, 0xf, 0x3, false);
                else v = __builtin_amdgcn_update_dpp(u, u, 0x118, 0xf, 0xc, false);
            } else {
                if constexpr (J == 0) v = __builtin_amdgcn_update_dpp(u, u, 0x114, 0xf, 0x2, false);
                else if constexpr (J == 1) v = __builtin_amdgcn_update_dpp(u, u, 0x104, 0xf, 0x1, false);
                else if constexpr (J == 2) v = __builtin_amdgcn_update_dpp(__builtin_amdgcn_update_dpp(u, u, 0x108, 0xf, 0x1, false), u, 0x104, 0xf, 0x2, false);
                else v = __builtin_amdgcn_update_dpp(__builtin_amdgcn_update_dpp(u, u, 0x10c, 0xf, 0x1, false), u, 0x108, 0xf, 0x2, false);
            }
            b[2 * x] = __builtin_amdgcn_perm(0u, v, sel0);
            b[2 * x + 1] = __builtin_amdgcn_perm(0u, v, sel1);
        }
        return __builtin_bit_cast(bf16x8, b);
    }
    // two channels of the lane's row, byte B of its tokens' words
    template <int B>
    __device__ __forceinline__ void bytes(const unsigned* v, const float* sc, int st, int h, const bf16x8& b0, const bf16x8& b1) {
        if constexpr (SPLIT) {
            u32x4 a0, a1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                a0[e] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[e], sc[e], B));
                a1[e] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v[4 + e], sc[4 + e], B));
            }
            f32x4& x = o[st * 4 + B];
            x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a0), b0, x, 0, 0, 0);
            x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a1), b1, x, 0, 0, 0);
        } else {
            u32x4 a, b;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                unsigned x, y;
                kv4_pair<B>(v[2 * e], sc[2 * e], v[2 * e + 1], sc[2 * e + 1], x, y);
                a[e] = x;
                b[e] = y;
            }
            f32x4 &x = o[st * 8 + 2 * B], &y = o[st * 8 + 2 * B + 1];
            x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), pr[h], x, 0, 0, 0);
            y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), pr[h], y, 0, 0, 0);
        }
    }
    // half H of the page's values
    template <int H>
    __device__ __forceinline__ void add(const Kv4Values<M>& p, int lo, int hi, bool edge, unsigned sel0, unsigned sel1, int c, int g) {
        bf16x8 b0, b1;
        if constexpr (SPLIT) {
            b0 = operand<2 * H>(sel0, sel1);
            b1 = operand<2 * H + 1>(sel0, sel1);
        }
#pragma unroll
        for (int st = 0; st < Kv4Values<M>::SETS; ++st) {
            unsigned v[8];
            float sc[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = p.v[st][e];
                sc[e] = kv4_scale_of(p.vs[st][e >> 2], e & 3);
            }
            if (edge) {
                const int a = lo - 32 * H - 8 * g, b = hi - 32 * H - 8 * g;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool ok = e >= a && e < b;
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
            bytes<0>(v, sc, st, H, b0, b1);
            if constexpr (MP >= 2) bytes<1>(v, sc, st, H, b0, b1);
            if constexpr (MP >= 4) {
                bytes<2>(v, sc, st, H, b0, b1);
                bytes<3>(v, sc, st, H, b0, b1);
            }
        }
    }
    // Row r (0..15) of the accumulators of one set is PER neighbouring channels from `channel` on: number e of them in tile set PER + e, or, SPLIT,
    // in tile (set PER + e) / 2 of copy e % 2.
    static constexpr int PER = MP >= 4 ? 8 : MP == 2 ? 4 : 2, SETS = 2 * MP / PER;
    static __device__ __forceinline__ int channel(int set, int r) {
        if constexpr (MP >= 4) return 8 * (r + 16 * set);
        else if constexpr (MP == 2) return 8 * (r & 7) + 4 * (r >> 3);
        else return 8 * (r & 3) + 2 * (r >> 2);
    }
};

// How many workgroups a compute unit holds: what their registers allow.  With two of 16 heads beyond 128 28 to 37 spill: 64 sequences of 128 to 8,192
// tokens through 8 kv heads of 256 183 us, so 140; 32 of 2,000 of 160 38.7 and 31.7.  A step's shares are as many as are resident: 3 a unit where 1 is
// 159, where 2 are (32 heads of 256 over 8, 11 sequences to 6,799; 128 of 128, 16 of 8,000) 37 us against 29 and 44 against 35.
constexpr int kv4_decode_resident(int hd, int gb) { return hd <= 128 ? (gb < 16 ? 3 : 2) : gb < 16 ? 2 : 1; }

// block = 256: the 4 waves take the pages of a stretch in turn, each with keys and values straight from memory into registers, and are
// joined in LDS in wave order where the stretch ends; nothing else is shared between them.  A wave's next page, of this stretch or
// the next, is asked for piece by piece, each as soon as the registers that held the present page's are free.
// `runs.nsplit` 1: a workgroup for every sequence and group, grid = (groups, B); else grid = `runs.wgs`.
// Bytes bound it where there are many: 16 sequences of 32,768 (8 kv heads of 128) in 93 us, 6.1 TB/s, 64 of 128 to 8,192 in 52 us, 5.6 TB/s; the
// waits for lengths, table and first page (together 5 us) where there are few: one of 1,088 in 9 us.
template <int M, int GB>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kv4_decode_resident(32 * M, GB), kv4_decode_resident(32 * M, GB)))) void attn_decode_kv4_kernel(
    const bf16* __restrict__ q, size_t q_stride, bf16* __restrict__ out, Kv4Seqs seqs, Kv4Runs runs, const unsigned char* __restrict__ cache,
    int nq, int nkv, float scale, float* __restrict__ part_o, float* __restrict__ part_ml) {
    typedef Kv4State<M, GB> State;
    typedef kv4_layout<M> L;
    constexpr int HD = 32 * M, MP = State::MP, PER = State::PER;
    constexpr int OS = State::TILES * 256, WSTRIDE = OS + 2 * GB;
    extern __shared__ float lds[];                      // per wave its accumulators register by register, [TILES][4][64 lanes], then [GB] m, [GB] l
    const int G = nq / nkv, nhb = (G + GB - 1) / GB;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Kv4Lane<M> at(lane);
    const int c = at.c, g = at.g;
    const bool pieces = runs.nsplit > 1;
    Kv4List list;
    int x = 0, end = 0;                                 // this workgroup's places of the list
    if (pieces) {
        list.start(runs, seqs, lane);
        const int all = list.total * runs.groups;       // below 2^30; shares that begin behind it may begin behind 2^31 as well
        const long long from = (long long)blockIdx.x * list.p;
        x = from < all ? (int)from : all;
        end = all - x > list.p ? x + list.p : all;
        // sequences of no tokens are in nobody's part
        for (int from = blockIdx.x * WAVE; from < runs.B; from += gridDim.x * WAVE) {
            Kv4List some = list;
            if (from > 0) some.at(runs, seqs, from, 0, lane);
            for (unsigned long long none = __ballot(some.n == 0 && from + lane < runs.B); none; none &= none - 1) {
                const size_t row = (size_t)(from + __builtin_ctzll(none)) * nq * HD;
                for (int i = threadIdx.x; i < nq * HD; i += 256) out[row + i] = (bf16)0.f;
            }
        }
        if (x >= end) return;
    }
    // a stretch of pages of one sequence and group (none if the places end before its first page)
    struct Stretch { int b, group, ctx, lo, first, n, places; bool whole; size_t piece; const int* bt; };
    auto stretch = [&](int place) {
        Stretch r;
        int slot, length;
        if (pieces) {
            int begin, own;
            r.group = place / list.total;
            r.b = list.find(runs, seqs, place - r.group * list.total, own, begin, slot, length, lane);
            begin += r.group * list.total;
            const int from = place - begin, upto = own < end - begin ? own : end - begin;        // of its own places
            r.places = upto - from;
            r.first = from > KV4_SWITCH ? from - KV4_SWITCH : 0;
            r.n = upto - KV4_SWITCH - r.first > 0 ? upto - KV4_SWITCH - r.first : 0;
            r.whole = r.n == own - KV4_SWITCH;
            // the first piece is the workgroup's that has its first page
            r.piece = from <= KV4_SWITCH ? 0 : blockIdx.x - (begin + KV4_SWITCH) / list.p;
            runs.pages(seqs, slot, length, r.ctx, r.lo);
        } else {
            r.b = blockIdx.y;
            r.group = blockIdx.x;
            r.first = 0;
            slot = kv4_uniform(seqs.slots + r.b);
            length = kv4_uniform(seqs.ctx_lens + r.b);
            r.n = r.places = runs.pages(seqs, slot, length, r.ctx, r.lo);
            r.whole = true;
            r.piece = 0;
        }
        r.first += r.lo / KV4_PAGE;
        r.bt = seqs.table + (size_t)(r.n ? slot : 0) * seqs.table_pages;
        return r;
    };
    Stretch now = stretch(x);
    // the page that this wave has asked for: number `i` of stretch `ahead`, whose places begin at `xa`; none if part is null
    Stretch ahead = now;
    int xa = x, ia = wave;
    const unsigned char* part = nullptr;
    auto seek = [&]() {
        for (;;) {
            if (ia < ahead.n) {
                const int pg = __builtin_amdgcn_readfirstlane(kv4_uniform(ahead.bt + ahead.first + ia));
                if ((unsigned)pg < (unsigned)seqs.n_pages) {
                    part = cache + ((size_t)pg * nkv + __builtin_amdgcn_readfirstlane(ahead.group / nhb)) * L::BYTES;
                    return;
                }
                ia += 4;
            } else {
                xa += ahead.places;
                if (!pieces || xa >= end) { part = nullptr; return; }
                ahead = stretch(xa);
                ia = wave;
            }
        }
    };
    State st;
    int nheads, head0;
    auto queries = [&]() {
        const int hb = now.group % nhb;
        head0 = now.group / nhb * G + hb * GB;
        nheads = G - hb * GB < GB ? G - hb * GB : GB;
        const bool ok = c % GB < nheads;
        const bf16* row = q + (size_t)now.b * q_stride + (size_t)(head0 + (ok ? c % GB : 0)) * HD;
#pragma unroll
        for (int w = 0; w < MP; ++w) {
            const int d = g * (8 * MP) + 8 * w;
            st.q[w] = ok && d < HD ? *(const bf16x8*)(row + d) : kv4_zero8();
        }
    };
    queries();                                          // before the pages: a wait for them is then none for the pages
    Kv4Keys<M> keys;
    Kv4Values<M> v0, v1;
    seek();
    if (part) {
        keys.load(part, at);
        v0.template load<0>(part, at);
        v1.template load<1>(part, at);
    }
    const float scale2 = scale * LOG2E;
    const unsigned odd = c / GB & 1, sel0 = odd ? 0x01000c0cu : 0x0c0c0100u, sel1 = odd ? 0x03020c0cu : 0x0c0c0302u;
    for (;;) {
        if (pieces && now.n == 0) return;               // the places end here
        st.clear();
        while (part && xa == x) {                       // the page that is there is of this stretch
            const int tok = (now.first + ia) * KV4_PAGE, a = now.lo - tok > 0 ? now.lo - tok : 0, e = now.ctx - tok < KV4_PAGE ? now.ctx - tok : KV4_PAGE;
            const bool edge = a > 0 || e < KV4_PAGE;
            f32x4 s[4];
            st.scores(keys, s);
            ia += 4;
            seek();
            if (part) keys.load(part, at);
            st.weights(s, a, e, edge, scale2, c, g);
            st.template add<0>(v0, a, e, edge, sel0, sel1, c, g);
            if (part) v0.template load<0>(part, at);
            st.template add<1>(v1, a, e, edge, sel0, sel1, c, g);
            if (part) v1.template load<1>(part, at);
        }
        st.l = State::sum(st.l);
        // Register by register no two lanes meet in a bank, neither here nor where they are read (16 heads of 256, head by head and channel by
        // channel: all 64 lanes in one, 7 us a stretch).
        float* my = lds + wave * WSTRIDE;
        const int copy = c / GB;
#pragma unroll
        for (int i = 0; i < State::TILES; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) my[(4 * i + r) * 64 + lane] = st.o[i][r];
        if (g == 0 && copy == 0) { my[OS + c] = st.m; my[OS + GB + c] = st.l; }
        __syncthreads();
        for (int u = threadIdx.x; u < GB * 16 * State::SETS; u += 256) {
            const int h = u % GB, ug = u / GB & 3, ur = u / (4 * GB) & 3, set = u / (16 * GB), d = State::channel(set, 4 * ug + ur);
            if (h >= nheads || (M != MP && d >= HD)) continue;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4; ++w) mx = fmaxf(mx, lds[w * WSTRIDE + OS + h]);
            const float use = mx == -INFINITY ? 0.f : mx;
            float sum = 0.f, v[PER];
#pragma unroll
            for (int e = 0; e < PER; ++e) v[e] = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = kv4_exp2(lds[w * WSTRIDE + OS + h] - use);
                sum += lds[w * WSTRIDE + OS + GB + h] * f;
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const int tile = State::SPLIT ? (set * PER + e) / 2 : set * PER + e;
                    v[e] += lds[w * WSTRIDE + (4 * tile + ur) * 64 + 16 * ug + (State::SPLIT ? (e & 1) * GB : 0) + h] * f;
                }
            }
            const size_t row = (size_t)now.b * nq + head0 + h;
            typedef float vf __attribute__((ext_vector_type(PER)));
            typedef bf16 vb __attribute__((ext_vector_type(PER)));
            if (now.whole) {
                vb y;
#pragma unroll
                for (int e = 0; e < PER; ++e) y[e] = (bf16)(sum == 0.f ? 0.f : v[e] / sum);
                *(vb*)(out + row * HD + d) = y;
            } else {
                const size_t i_ = row * runs.nsplit + now.piece;
                vf y;
#pragma unroll
                for (int e = 0; e < PER; ++e) y[e] = v[e];
                *(vf*)(part_o + i_ * HD + d) = y;
                if (d == 0) { part_ml[i_ * 2] = mx; part_ml[i_ * 2 + 1] = sum; }
            }
        }
        x += now.places;
        if (!pieces || x >= end) return;
        now = stretch(x);
        queries();
        __syncthreads();
    }
}

// The runs of a row added in their order: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.  A wave a row (token, head).
// `cu` (null: none): the step's B + 1 offsets; rows in front of the first sequence and behind the last have no runs and stay as they are.
// RUNS: rows of single tokens, in as many pieces each as the list's places say; those of one are there already.
template <bool RUNS>
__global__ __launch_bounds__(256) void attn_kv4_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                                            bf16* __restrict__ out, size_t rows, int nq, int hd, int nsplit,
                                                            const int* __restrict__ cu, int B, Kv4Seqs seqs, Kv4Runs runs, int G, int gb) {
    const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows) return;
    if (cu) {
        const long long first = (long long)cu[0] * nq, end = (long long)cu[B] * nq;
        if ((long long)row < first || (long long)row >= end) return;
    }
    // runs are at most 64, one a lane; 16 lanes take 64 channels, so that a run's row is hd / 64 groups of them and the others take
    // further runs at the same time.  Everything is asked for before it is known how many runs there are: of the others nothing is used.
    const float m_ = lane < nsplit ? part_ml[(row * nsplit + lane) * 2] : -INFINITY;
    const float l_ = lane < nsplit ? part_ml[(row * nsplit + lane) * 2 + 1] : 0.f;
    const int per = (hd + 63) / 64, sub = (lane >> 4) / per, many = 4 / per, d = ((lane >> 4) % per) * 64 + (lane & 15) * 4;
    auto fetch = [&](int i) { return i < nsplit && sub < many && d < hd ? *(const f32x4*)(part_o + (row * nsplit + i) * hd + d) : f32x4{0.f, 0.f, 0.f, 0.f}; };
    f32x4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = fetch(j * many + sub);
    int n_runs = nsplit;
    if (RUNS) {
        const int b = __builtin_amdgcn_readfirstlane((int)(row / nq)), head = __builtin_amdgcn_readfirstlane((int)(row % nq));
        Kv4List list;
        list.start(runs, seqs, lane);
        while (b >= list.base + WAVE) list.at(runs, seqs, list.base + WAVE, list.end(), lane);
        const int own = __builtin_amdgcn_readlane(list.n, b - list.base);
        const int group = head / G * ((G + gb - 1) / gb) + head % G / gb;
        const int first = __builtin_amdgcn_readlane(list.upto, b - list.base) - own + group * list.total;
        n_runs = own ? (first + own - 1) / list.p - (first + KV4_SWITCH) / list.p + 1 : 1;
        if (n_runs == 1) return;
    }
    const float m = lane < n_runs ? m_ : -INFINITY, l = lane < n_runs ? l_ : 0.f;
    const float mx = wave_max(m);
    const float f = l == 0.f ? 0.f : kv4_exp2(m - (mx == -INFINITY ? 0.f : mx));
    const float sum = wave_sum(l * f);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < n_runs; i0 += 4 * many) {
        if (i0 > 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = fetch(i0 + j * many + sub);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + j * many + sub;
            const float w = __shfl(f, i < n_runs ? i : 0, WAVE);
            if (i < n_runs) o += w * x[j];         // of a weight of 0 as well: its sums are NaN where a value that the row sees is
        }
    }
    if (sub >= many) o = f32x4{0.f, 0.f, 0.f, 0.f};
    if (per <= 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], 32, WAVE);
    }
    if (per == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], 16, WAVE);
    }
    if (sub == 0 && d < hd) {
        bf16x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (bf16)(o[e] * inv);
        *(bf16x4*)(out + row * hd + d) = r;
    }
}

// --------------------------------------------------------------------- prefill ------
// Several tokens per sequence.  A workgroup takes `tile_rows` <= 32 NW / KH rows of one kv head and sequence, row = token * G + head, 32 a wave, and
// walks the pages that they see.  A page's codes come to registers while the page before is multiplied, are turned into
// bfloat16 once for all waves and lie in LDS in the order of the matrix operands, 1 KB a wave-read, two pages deep; one barrier a page.
// Two waves a SIMD overlap each other's products and softmax: 8,192 tokens of 32 heads of 128 over 8 in 550 us, 1.0 PFLOP/s (a wave's own 32 x 32
// scores take 0.93 us alone and 0.5 of the SIMD's time beside another; whole pages at a time, for more to overlap within a wave, 580 us).
// KH 2: a row has two waves, one for each half of every page, joined at the end: half as many rows, and a page in 1.7 us instead of 2.5.
// Chunk [half][k-step][lane] of the keys: 8 channels of the key that row lane % 32 of a 32-key block stands for.  Chunk [32 channels]
// [16 tokens][lane] of the values: 8 tokens of a channel.  (A code and its scale become bfloat16 in half an instruction; read by
// every wave for itself they would cost NW times as many.)
//
// Values that are NaN (scale 255) would spoil rows that do not see them, since 0 * NaN is NaN: they go into LDS as zeros, and which tokens'
// they were beside them, and NaN goes into the accumulators of the rows that see them only.
__device__ __forceinline__ int kv4_key_of_row(int c) { return 16 * (c >> 4) + 8 * ((c >> 2) & 1) + 4 * ((c >> 3) & 1) + (c & 3); }
__device__ __forceinline__ int kv4_row_of_key(int u) { return (u & 3) | (((u >> 2) & 1) << 3) | (((u >> 3) & 1) << 2) | (u & 16); }
// Place of a channel's row among a value chunk's 32: turned so that the 16 lanes that write different rows at a time reach different banks
__device__ __forceinline__ int kv4_value_row(int row, int i2) { return row ^ ((row >> 4) | ((i2 & 3) << 1)); }

template <int M, int NW, int KH>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(NW == 4 ? 1 : M <= 2 ? 4 : 2, M <= 2 ? 4 : 2))) void attn_prefill_kv4_kernel(const bf16* __restrict__ q, size_t q_stride, bf16* __restrict__ out,
                                                                   const int* __restrict__ cu_seqlens, Kv4Seqs seqs,
                                                                   const unsigned char* __restrict__ cache, int nq, int nkv, int window,
                                                                   float scale, const PrefillOrder order, int n_tokens, int tile_rows, int nsplit,
                                                                   float* __restrict__ part_o, float* __restrict__ part_ml) {
    constexpr int HD = 32 * M, NT = NW * 64, RW = NW / KH;
    constexpr int KB = KV4_PAGE * HD * 2, STAGE = 2 * KB;                       // bytes of a page's keys; keys and values
    constexpr int UNITS = 64 * M, UPT = (UNITS + NT - 1) / NT;                    // units of 32 elements of the keys, as many of the values; of each a thread
    typedef kv4_layout<M> L;
    extern __shared__ __attribute__((aligned(1024))) unsigned char dsm[];
    int* nan_page = (int*)(dsm + 2 * STAGE);                                    // [2]: the page in a stage that holds NaN values, + 1
    unsigned char* nan_tokens = dsm + 2 * STAGE + 16;                           // [2][M blocks][8 bytes]: which tokens' values those are
    int kvh, b, tile, split = 0;
    if (nsplit > 1) {                                                           // grid (tiles * runs, nkv, B)
        kvh = blockIdx.y;
        b = blockIdx.z;
        tile = blockIdx.x / nsplit;
        split = blockIdx.x % nsplit;
    } else order.place(kvh, b, tile);
    // asked for together, not one behind the other (67 tokens 9.2 us, 9.4)
    const int t0 = kv4_uniform(cu_seqlens + b), t1 = kv4_uniform(cu_seqlens + b + 1), slot = kv4_uniform(seqs.slots + b), length = kv4_uniform(seqs.ctx_lens + b);
    const int n_new = t1 - t0;
    const int G = nq / nkv;
    const long long rows_total = (long long)n_new * G;
    if (t0 < 0 || t0 + n_new > n_tokens || (long long)tile * tile_rows >= rows_total) return;        // the whole workgroup leaves together
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = KH == 1 ? wave : wave % RW, kh = KH == 1 ? 0 : wave / RW;   // the wave's 32 rows and, of KH 2, its half of every page
    const int row0 = tile * tile_rows + rw * 32;
    const int c = lane & 31, g = lane >> 5;
    const int last = (int)(rows_total < (long long)(tile + 1) * tile_rows ? rows_total : (long long)(tile + 1) * tile_rows) - 1;       // of the tile's
    const bool wave_ok = row0 <= last, row_ok = row0 + c <= last;
    const int rr = row_ok ? row0 + c : last;                                     // lanes behind the last row work on it too and store nothing
    const int tok = rr / G, head = kvh * G + rr % G;
    const size_t orow = (size_t)(t0 + tok) * nq + head;
    const bool there = (unsigned)slot < (unsigned)seqs.n_slots;
    const int ctx = there ? length : 0, start = ctx - n_new;
    const int pq = start + tok;
    const int w_last = row0 + 31 < last ? row0 + 31 : last, g_last = last;
    const int pq_min_w = start + (wave_ok ? row0 : last) / G, pq_max_w = start + w_last / G;
    const int pq_min_g = start + tile * tile_rows / G, pq_max_g = start + g_last / G;
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
    // 16 neighbouring units of the values lie in 16 groups of channels, whose rows reach different banks.  For heads of 128 and 8 waves
    // the first four convert and the others, on the same SIMDs, are at their products meanwhile: units spread over all waves are
    // slower (8,192 tokens: 647 us against 615; all of them behind the products 715).
    auto value_cg = [](int u) { return M % 4 == 0 ? (u & 15) + 16 * (u >> 8) : u % (4 * M); };
    auto value_half = [](int u) { return M % 4 == 0 ? (u >> 4) & 1 : u / (32 * M); };
    auto value_tg = [](int u) { return M % 4 == 0 ? (u >> 5) & 7 : u / (4 * M) & 7; };
    // Waves without rows, the last ones, convert where a tile has such; the first ones in full tiles (8,192 tokens: 547 us against 585 by the last).
    const int with_rows = tile_rows / 32;
    const int turn = KH == 1 ? (with_rows < NW ? NW - 1 - wave : wave) : rw >= with_rows ? (rw - with_rows) * 2 + kh : 2 * (RW - with_rows) + kh * with_rows + rw;
    const int unit0 = turn * 64 + lane;
    u32x4 kr[UPT], va[UPT], vb[UPT];
    u32x2 vsr[UPT];
    unsigned ksr[UPT];
    auto fetch = [&](const unsigned char* part) {
#pragma unroll
        for (int i = 0; i < UPT; ++i) {
            const int u = unit0 + i * NT;
            if (UNITS % NT == 0 || u < UNITS) {
                const int t = u & 63, blk = u >> 6, cg = value_cg(u), tg = value_tg(u);
                kr[i] = *(const u32x4*)(part + L::KC + t * (16 * M) + blk * 16);
                ksr[i] = part[L::KS + kv4_key_scale(t, blk, M)];
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
            const int u = unit0 + i * NT;
            if (UNITS % NT == 0 || u < UNITS) {
                const int t = u & 63, blk = u >> 6, krow = kv4_row_of_key(t & 31);
                const float ks = kv4_scale(ksr[i]);
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    *(bf16x8*)(st + (((t >> 5) * 2 * M + 2 * blk + (w >> 1)) * 64 + (w & 1) * 32 + krow) * 16) = kv4_to_bf16(kr[i][w], ks);
                const int cg = value_cg(u), tg = value_tg(u), half = value_half(u);
                unsigned v[8];
                float sc[8];
                u32x2 vs = vsr[i];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = (e < 4 ? va[i][e & 3] : vb[i][e & 3]) >> (16 * half);
                if (live < KV4_PAGE) {                                  // what is not written yet: zeros with a scale of 1
                    const int n = live - 8 * tg;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e >= n) {
                            v[e] = 0u;
                            vs[e >> 2] = (vs[e >> 2] & ~(255u << (8 * (e & 3)))) | (127u << (8 * (e & 3)));
                        }
                }
                // a byte of 255 in either word: all of its lower bits carry into the one above, which is set as well
                unsigned bad = 0;
                if (((((vs[0] & 0x7f7f7f7fu) + 0x01010101u) & vs[0]) | (((vs[1] & 0x7f7f7f7fu) + 0x01010101u) & vs[1])) & 0x80808080u) {
                    nan_page[buf] = pi + 1;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if ((vs[e >> 2] >> (8 * (e & 3)) & 255u) == 255u) {
                            bad |= 1u << e;
                            v[e] = 0u;
                            vs[e >> 2] ^= 128u << (8 * (e & 3));        // 127: 1
                        }
                }
                nan_tokens[(buf * M + (cg >> 2)) * 8 + tg] = (unsigned char)bad;     // the same from all units of the block
#pragma unroll
                for (int e = 0; e < 8; ++e) sc[e] = kv4_scale_of(vs[e >> 2], e & 3);
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
    // The numbers of 64 pages lie in the lanes, so that no turn waits for the table.  `next_page`: the next page from pi on that is there
    // (its number in `number`), or last_pg + 1.
    int held = first_pg, numbers = held + lane <= last_pg ? bt[held + lane] : 0, number = 0;
    auto next_page = [&](int pi) {
        for (; pi <= last_pg; ++pi) {
            if (pi >= held + 64) {
                held = pi;
                numbers = held + lane <= last_pg ? bt[held + lane] : 0;
            }
            number = __builtin_amdgcn_readlane(numbers, pi - held);
            if ((unsigned)number < (unsigned)seqs.n_pages) break;
        }
        return pi;
    };
    auto part_of = [&]() { return cache + ((size_t)number * nkv + kvh) * L::BYTES; };

    if (tid < 2) nan_page[tid] = 0;
    int pi = next_page(first_pg);
    if (pi <= last_pg) fetch(part_of());
    kv4_lds_barrier();
    if (pi <= last_pg) put(0, ctx - pi * KV4_PAGE, pi);
    int pn = next_page(pi + 1);
    if (pn <= last_pg) fetch(part_of());
    kv4_lds_barrier();
    for (int buf = 0; pi <= last_pg; buf ^= 1) {
        const int pm = next_page(pn + 1);
        auto bring = [&]() {
            if (pn <= last_pg) put(buf ^ 1, ctx - pn * KV4_PAGE, pn);
            if (pm <= last_pg) fetch(part_of());
        };
        const unsigned char* st = dsm + buf * STAGE;
        if (__builtin_amdgcn_readfirstlane(nan_page[buf]) == pi + 1) {
            // tokens [a, e) of the page are seen by this lane's row
            const int kb = pi * KV4_PAGE, a = window > 0 && pq - window + 1 - kb > 0 ? pq - window + 1 - kb : 0, e = pq + 1 - kb < KV4_PAGE ? pq + 1 - kb : KV4_PAGE;
            const unsigned long long seen = row_ok && a < e ? (~0ULL >> (64 - (e - a))) << a : 0;
#pragma unroll
            for (int i = 0; i < M; ++i)
                if (seen & ((const unsigned long long*)nan_tokens)[buf * M + i]) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[i][r] = NAN;
                }
        }
        auto block = [&](int half) {
            const int kb = pi * KV4_PAGE + 32 * half;
            const unsigned char* ks = st + (half * 2 * M * 64 + lane) * 16;
            f32x16 s;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
            for (int k = 0; k < 2 * M; ++k) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(ks + k * 1024), qf[k], s, 0, 0, 0);
            // s[r]: key kb + 16 (r / 8) + 8 g + r % 8, row = this lane's column
            const bool whole = kb + 31 <= pq_min_w && (window <= 0 || kb > pq_max_w - window);
            if (!whole) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = kb + 16 * (r >> 3) + 8 * g + (r & 7);
                    const bool ok = key <= pq && (window <= 0 || key > pq - window);
                    s[r] = ok ? s[r] : -INFINITY;
                }
            }
            float mx = fmaxf(fmaxf(s[0], s[1]), s[2]);
#pragma unroll
            for (int r = 3; r < 15; r += 2) mx = fmaxf(fmaxf(mx, s[r]), s[r + 1]);
            mx = fmaxf(mx, s[15]) * scale2;                                  // the scale is positive
            if (__any(mx > m)) {                                             // see Kv4State::weights
                const float m_new = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32, WAVE)) + KV4_ABOVE);
                const float corr = m_new == -INFINITY ? 1.f : kv4_exp2(m - m_new);
                m = m_new;
                l *= corr;
#pragma unroll
                for (int i = 0; i < M; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[i][r] *= corr;
            }
            const float m_use = m == -INFINITY ? 0.f : m;
            float sum0 = 0.f, sum1 = 0.f;
            bf16x8 p[2];
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = kv4_exp2(fmaf(s[r], scale2, -m_use)), y = kv4_exp2(fmaf(s[r + 1], scale2, -m_use));
                const bf16x2 w = {(bf16)x, (bf16)y};
                if (r & 2) sum1 = kv4_add_pair(w, sum1);
                else sum0 = kv4_add_pair(w, sum0);
                p[r >> 3][r & 7] = w[0];
                p[r >> 3][(r & 7) + 1] = w[1];
            }
            l += sum0 + sum1;
            const unsigned char* vs = st + KB + half * 2048;
#pragma unroll
            for (int i = 0; i < M; ++i)
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(vs + (4 * i + x) * 1024 + (32 * g + kv4_value_row(c, i)) * 16), p[x], o[i],
                                                                   0, 0, 0);
        };
        // halves that no row of this wave sees are left out
        const int kb = pi * KV4_PAGE;
        const bool s0 = wave_ok && kb <= pq_max_w && (window <= 0 || kb + 31 > pq_min_w - window);
        const bool s1 = wave_ok && kb + 32 <= pq_max_w && (window <= 0 || kb + 63 > pq_min_w - window);
        if constexpr (KH == 1) {
            if (s0) block(0);
            if (s1) block(1);
        } else if (kh ? s1 : s0) block(kh);
        bring();
        kv4_lds_barrier();
        pi = pn;
        pn = pm;
    }
    l += __shfl_xor(l, 32, WAVE);
    if constexpr (KH == 2) {
        // the second half's sums go to the wave of the same rows through LDS, where no page is needed any more
        f32x4* const theirs = (f32x4*)dsm + (size_t)rw * (4 * M * 64) + lane;
        float* const ml = (float*)(dsm + (size_t)RW * M * 4096) + rw * 128 + lane;
        if (kh) {
#pragma unroll
            for (int i = 0; i < M; ++i)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) theirs[(4 * i + r4) * 64] = f32x4{o[i][4 * r4], o[i][4 * r4 + 1], o[i][4 * r4 + 2], o[i][4 * r4 + 3]};
            ml[0] = m;
            ml[64] = l;
        }
        __syncthreads();
        if (kh) return;
        const float m1 = ml[0], l1 = ml[64], both = fmaxf(m, m1), use = both == -INFINITY ? 0.f : both, f0 = kv4_exp2(m - use), f1 = kv4_exp2(m1 - use);
        m = both;
        l = l * f0 + l1 * f1;
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const f32x4 x = theirs[(4 * i + r4) * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][4 * r4 + e] = o[i][4 * r4 + e] * f0 + x[e] * f1;
            }
    }
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

// LDS beyond 64 KB is asked for once for every kernel and device (`told`, a bit a device: a kernel always asks for the same).
static bool kv4_allow(const void* kernel, size_t lds, unsigned long long& told) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0) return false;
    if (dev < 64 && (__atomic_load_n(&told, __ATOMIC_RELAXED) >> dev & 1)) return true;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) return false;
    if (dev < 64) __atomic_fetch_or(&told, 1ULL << dev, __ATOMIC_RELAXED);
    return true;
}

#define KV4_SIZES(F) F(1) F(2) F(3) F(4) F(5) F(6) F(7) F(8)

template <bool RUNS>
static int kv4_join(const float* part_o, const float* part_ml, void* out, long long tokens, int nq, int hd, int nsplit, const int* cu, int B,
                    const Kv4Seqs& seqs, const Kv4Runs& runs, int G, int gb, hipStream_t s) {
    const size_t rows = (size_t)tokens * nq;
    attn_kv4_join_kernel<RUNS><<<(unsigned)((rows + 3) / 4), 256, 0, s>>>(part_o, part_ml, (bf16*)out, rows, nq, hd, nsplit, cu, B, seqs, runs, G, gb);
    return br_check_launch();
}

extern "C" int br_attn_decode_kv4(const void* q, size_t q_stride, void* out, const int* slots, const int* ctx_lens, const int* table,
                                  int n_slots, int table_pages, const void* cache, int n_pages, int B, int nq, int nkv, int hd, int window,
                                  float scale, int nsplit, float* part_o, float* part_ml, hipStream_t s) {
    if (hd % 32 || hd < 32 || hd > 256 || nkv < 1 || nq < nkv || nq % nkv || B < 0 || B > 65535 || nsplit < 1 || nsplit > 64 ||
        table_pages > 0x7fffffff / KV4_PAGE || (nsplit > 1 && (!part_o || !part_ml))) return BR_BAD_ARG;
    // heads that share a kv head go as columns of one product: 4, 8 or 16 at a time
    const int G = nq / nkv, gb = G <= 4 ? 4 : G <= 8 ? 8 : 16, groups = nkv * ((G + gb - 1) / gb);
    if ((long long)B * nq > 0x7fffffffLL) return BR_BAD_ARG;
    const int cus = br_device_cus(), all = (cus > 0 ? cus : 256) * kv4_decode_resident(hd, gb);
    const long long seen = window > 0 && (window + 2LL * KV4_PAGE - 2) / KV4_PAGE < table_pages ? (window + 2LL * KV4_PAGE - 2) / KV4_PAGE : table_pages;
    const long long pages = B * seen * groups, places = pages + (long long)B * groups * KV4_SWITCH;        // of the list at most
    if (places > 0x3fffffffLL) return BR_TOO_LARGE;
    if (B == 0) return BR_OK;
    const int wgs = (int)((pages + 3) / 4 < all ? (pages + 3) / 4 > 0 ? (pages + 3) / 4 : 1 : all);
    const Kv4Runs runs = {B, window, groups, wgs, nsplit, (float)(1.00001 * groups / wgs), (float)(1.00001 / (nsplit > 1 ? nsplit - 1 : 1))};
    const dim3 grid = nsplit > 1 ? dim3(wgs) : dim3(groups, B);
    const int mp = hd > 128 ? 8 : hd == 96 ? 4 : hd / 32;                   // Kv4Keys::MP
    const size_t lds = 4 * ((size_t)(gb < 16 ? mp : 2 * mp) * 256 + 2 * gb) * sizeof(float);
    const Kv4Seqs seqs = {slots, ctx_lens, table, n_slots, table_pages, n_pages};
#define GO(M_, GB_) { \
        static unsigned long long told; \
        if (lds > 65536 && !kv4_allow((const void*)attn_decode_kv4_kernel<M_, GB_>, lds, told)) return BR_LAUNCH_FAILED; \
        attn_decode_kv4_kernel<M_, GB_><<<grid, 256, lds, s>>>((const bf16*)q, q_stride, (bf16*)out, seqs, runs, (const unsigned char*)cache, nq, nkv, scale, part_o, part_ml); }
#define CASE(M_) case M_: if (gb == 4) GO(M_, 4) else if (gb == 8) GO(M_, 8) else GO(M_, 16) break;
    switch (hd / 32) { KV4_SIZES(CASE) }
#undef CASE
#undef GO
    const int rc = br_check_launch();
    return rc != BR_OK || nsplit == 1 ? rc : kv4_join<true>(part_o, part_ml, out, B, nq, hd, nsplit, nullptr, B, seqs, runs, G, gb, s);
}

extern "C" int br_attn_prefill_kv4(const void* q, size_t q_stride, void* out, const int* cu_seqlens, const int* slots, const int* ctx_lens,
                                   const int* table, int n_slots, int table_pages, const void* cache, int n_pages, int B, int max_new,
                                   int n_tokens, int nq, int nkv, int hd, int window, float scale, int nsplit, float* part_o, float* part_ml,
                                   hipStream_t s) {
    if (hd % 32 || hd < 32 || hd > 256 || nkv < 1 || nkv > 65535 || nq < nkv || nq % nkv || B < 0 || B > 65535 || max_new < 0 || nsplit < 1 ||
        nsplit > 64 || table_pages > 0x7fffffff / KV4_PAGE || (long long)n_tokens * nq > 0x7fffffffLL || n_tokens < max_new || (nsplit > 1 && (!part_o || !part_ml))) return BR_BAD_ARG;
    const long long rows = (long long)max_new * (nq / nkv);
    if (rows > 0x7fffffffLL - 256) return BR_BAD_ARG;
    if (B == 0 || max_new == 0) return BR_OK;
    // 8 waves convert a page once for 256 rows.  Tiles of 128 rows, two waves to 32 of them and each with a half of every page, where 256 would
    // leave units without a tile or a few long ones last: 128 tokens of 32 heads of 128 over 8 in 10.7 us, not 13.1, 512 18.5 / 24.1, 2,048
    // 62 / 72, but 3,000 122 / 99; for several sequences, whose tiles differ less, earlier: twice 1,500 75 / 54, 8 times 250 24.9 / 20.3.  Of heads
    // of up to 64 two workgroups share a unit (32 over 4 heads of 64: 2,000 tokens 43.7 / 54.0, 16 times 500 51 / 38, 8,192 365 / 321; five of
    // 1,357 to 93 have 128 rows by this rule, 45 / 41.5).
    // In runs: 5 tokens behind 3,800 of 8 users 26.3 / 29.6, 16 behind 16,000 22.7 / 24.0, 32 behind 16,352 28.8 / 27.4.
    const int cus = br_device_cus() > 0 ? br_device_cus() : 256, each = hd <= 64 ? 2 : 1;
    const long long filled = ((long long)n_tokens * (nq / nkv) + 255) / 256 * nkv;
    // Heads beyond 128 have no registers for 256 rows, and from 8 waves of 256 channels 34 spill: two prompts of 158 and 109 tokens of 12 heads
    // over 4 and 24 over 8 take 4 waves of 32 rows, each alone on its SIMD, 18.6 and 19.0 us, 8 waves 19.6 and 20.2; 1,646 tokens 65 / 59, 8,192 960 / 758 (of
    // heads of 160 740 / 469).  Of heads of 64, four waves a SIMD with 128 registers each, 2 spill.
    const bool half = hd < 256 || nsplit > 1 || max_new > 256;
    const bool wide = hd <= 128 && (nsplit > 1 ? rows > 64 : filled > (each == 2 || B == 1 ? each * cus : cus / 2));
    const int most = wide ? 256 : 128;
    const long long tiles = (rows + most - 1) / most;
    PrefillOrder order = {};
    dim3 grid;
    int tile_rows = most;
    if (nsplit > 1) {
        // tiles of about equal height: 67 tokens of 4 heads are 160 and 108 rows, not 256 and 12
        tile_rows = (int)(((rows + tiles - 1) / tiles + 31) / 32 * 32);
        if (tiles * nsplit > 0x7fffffffLL) return BR_BAD_ARG;
        grid = dim3((unsigned)(tiles * nsplit), nkv, B);
    } else if (!prefill_order(order, grid, wide ? (rows + 1) / 2 : rows, nkv, B, cus, each)) return BR_BAD_ARG;   // it counts in tiles of 128
    const size_t lds = 2 * (size_t)2 * KV4_PAGE * hd * 2 + (!wide && half ? 4 * 128 * sizeof(float) : 16 + 2 * (hd / 32) * 8);
    const Kv4Seqs seqs = {slots, ctx_lens, table, n_slots, table_pages, n_pages};
#define GO(M_, NW_, KH_) { \
        static unsigned long long told; \
        if (lds > 65536 && !kv4_allow((const void*)attn_prefill_kv4_kernel<M_, NW_, KH_>, lds, told)) return BR_LAUNCH_FAILED; \
        attn_prefill_kv4_kernel<M_, NW_, KH_><<<grid, NW_ * 64, lds, s>>>((const bf16*)q, q_stride, (bf16*)out, cu_seqlens, seqs, (const unsigned char*)cache, nq, nkv, window, scale, order, n_tokens, tile_rows, nsplit, part_o, part_ml); }
#define BOTH(M_) case M_: if (wide) GO(M_, 8, 1) else GO(M_, 8, 2) break;
#define HALF(M_) case M_: GO(M_, 8, 2) break;
    switch (hd / 32) {
        BOTH(1) BOTH(2) BOTH(3) BOTH(4) HALF(5) HALF(6) HALF(7)
        case 8: if (half) GO(8, 8, 2) else GO(8, 4, 1) break;
    }
#undef HALF
#undef BOTH
#undef GO
    const int rc = br_check_launch();
    return rc != BR_OK || nsplit == 1 ? rc : kv4_join<false>(part_o, part_ml, out, n_tokens, nq, hd, nsplit, cu_seqlens, B, seqs, Kv4Runs{}, 1, 1, s);
}
