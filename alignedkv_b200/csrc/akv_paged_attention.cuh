// Attention of the newest tokens of each sequence over its pages.
//   attend_kernel   query rows of a (sequence, KV head) against its tokens; one pass with a running maximum and sum
//   join_kernel     joins the partial results of units that several CTAs share
//
//   s_rj = scale q_r . k_j, o_r = sum_j exp(s_rj - m_r) v_j / l_r, l_r = sum_j exp(s_rj - m_r), over the tokens j that row r sees.
//
// Every byte of the tokens is read once: bound by HBM in 16 and 8 bits (8 x 32 x 4096 tokens of 128 channels, e4m3: 48.5 us, 5.6 TB/s; up to 8192 of
// 64 x 8 heads: 95.5 us, 5.8 TB/s), in 4 by the instructions that unpack the codes and by their chains (8 heads x 131072 tokens: 43.9 us, 3.5 TB/s, 62% of the issue
// slots, no pipe full), and with many rows by the chain of products and softmax in few warps (20 rows, 32 x 8 heads x up to 4096: 59.8 us).
// Work: a unit is the query rows of one (sequence, KV head), up to 32, its tokens in chunks of 64.  The chunks of all units in a row are dealt in
// equal contiguous runs to the CTAs, then to a CTA's warps: lengths are only known on the device, and every SM gets the same whatever they
// are.  Each CTA adds up the lengths itself.  A warp needs no other one: it fills a ring in shared memory by asynchronous copies and drains it, codes go
// from there into registers as operand fragments.  (Loads straight into registers: 75 us where the ring took 63.  A ring for the whole CTA would
// need a barrier a step.)  Where a run begins or ends inside a unit it leaves a record, and the CTA joins those of its warps; what is left
// between CTAs is join_kernel's.  With few units and short tables a cluster has a unit to itself and joins its records in shared memory.
//
// Operands: tokens are the rows of the products' first operand, query rows the columns of the second - 8 of them, which one KV head's query heads
// fill, where the other way round 16 would be half empty.  Which channel is which k, and which token which row, is free as long as both
// operands agree, and chosen so that a lane's loads are 16 bytes and need the fewest permutations.
#pragma once
#include "akv_paged_attention.h"

namespace akv {
namespace {

constexpr float LN2 = 0.6931471805599453f;
// Probabilities (times 2^exponent of their token's values) enter their product as fp16, since both operands have one type and the codes are exact there;
// relative to the largest and times 2^15 they keep all 11 bits down to 2^-29 of it.  What the rounding takes is rounded to fp16 as well and multiplied too:
// 22 bits of a probability, 2^-39 of the largest at the least.  Against 64 bits outputs are then off by their own rounding alone (2.06 to 2.11e-4 in the 2-norm, to
// the digit what sums in 32 bits give; without the second part up to 3% more, 9 to 19% of the outputs a step away, where now 0.4 to 0.8% are, and an average of
// equal values was not that value).  It costs 0 to 2% up to 4 rows (`TWICE`) and 2 to 16% with more
// (32 x 8 heads x up to 4096 tokens: 12 rows fp16 56.9 -> 57.5 us, e4m3 38.5 -> 41.5, e2m1 39.8 -> 43.7; 20 rows 66.7 -> 69.6, 54.6 -> 59.6, 54.7 -> 59.8; 32 rows
// 83.7 -> 89.6, 74.6 -> 86.7, 73.3 -> 79.9).
constexpr float LIFT = 32768.f;


template <int F, int D, int NT>
struct Shape {
    static constexpr int ROW = row_bytes<F>(D);
    static constexpr int KW = ROW / 8;                        // words of 16 tokens of K (or of V) in a lane
    // (four for narrow rows: what a step costs beside its products is that of 32 tokens; 64 sequences of up to 8192 tokens, 8 heads, e4m3: 61.9 -> 56.2 us)
    static constexpr int U = ROW == 256 ? 1 : ROW < 128 && D == 64 && NT <= 2 ? 4 : 2;     // 16-token tiles of a step
    static constexpr int TOKENS = 16 * U, TEAM_TOKENS = TOKENS > 32 ? TOKENS : 32;         // tokens of a cluster's chunk
    static constexpr int KS = D / 16;                         // products over the channels; tiles of 16 channels of the output
    static constexpr int SCALES = F == AKV_PAGE_E2M1 ? D : 0; // bytes of a tile's scales (of K or of V)
    static constexpr int MORE = F == AKV_PAGE_FP16 ? 0 : 2 * SCALES + 32;                  // ... of its scales and exponents
    // A step in shared memory: a tile's codes of K and of V, the next tile's, then scales of K, of V, exponents of K, of V by tile.
    static constexpr int STEP = (U * (32 * ROW + MORE) + 127) / 128 * 128;
    static constexpr bool MANY = warps_of(F, D, NT) == 16;
    static constexpr int STEPS = ROW >= 128 || MANY ? 2 : F == AKV_PAGE_E2M1 && D == 128 ? 3 : D == 64 && NT == 3 ? (F == AKV_PAGE_E4M3 ? 3 : 4)
                                 : F == AKV_PAGE_E4M3 ? (U == 4 ? 2 : 4) : (U == 4 ? 3 : 6);
    // Up to 16 rows: operands of the queries stay in registers.  More: in shared memory.
    // (20 rows of 4 bits, 32 x 8 heads x up to 4096 tokens, 56 us then: ten warps spill, 69; steps of 16 tokens 63; units of 16 rows 67, of 8 64.)
    static constexpr bool FEW = NT <= 2;
    static constexpr int WARPS = warps_of(F, D, NT);
    static constexpr int RECORD = 8 * NT * (D + 4);           // floats: rows of D sums, then the maximum and the sum
    static constexpr int TABLE = F == AKV_PAGE_FP16 ? 0 : TOKENS * 16;       // of a step's tokens: factor, exponent, weight
    static constexpr int RING = STEPS * STEP, QUERIES = FEW ? 0 : KS * 4 * 32 * 8, OWN = RING + QUERIES + TABLE, SMEM = WARPS * OWN;
    static_assert(OWN >= RECORD * 4, "a run's last record lies where its ring was");
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// 16 bytes global -> shared past L1; with `there` false zeros, and nothing is read.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ int lds8_signed(uint32_t a) {
    int v;
    asm volatile("ld.shared.s8 %0, [%1];\n" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t halves_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// ---------------------------------------------------------------- which chunks are whose
// cum[b]: chunks of one unit of the sequences before b; a sequence without tokens has one, so that its rows are written.
template <int TOKENS>
__device__ __forceinline__ int chunks_of(int n) { return max(1, (n + TOKENS - 1) / TOKENS); }

template <int THREADS>
__device__ __forceinline__ void add_lengths(const AttendArgs& a, int* cum, int* sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += THREADS) {
        const int b = b0 + tid;
        int x = b < a.B ? chunks_of<CHUNK>(length_of(a.pool, b)) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w == warp) x += total;
            total += sums[w];
        }
        if (b < a.B) cum[b + 1] = before + x;
        before += total;
        __syncthreads();
    }
    if (tid == 0) cum[0] = 0;
    __syncthreads();
}
// First to the CTAs, each within one of the others, then to a CTA's warps: an SM's warps share what it gets of the bandwidth (dealt to all warps in a row, the
// first fifth of the CTAs had a tenth more: 8 x 32 heads x 4096 tokens 48.8 us, now 48.3; 64 x 8 heads x up to 8192 96.7, now 95.2).
struct Deal {
    int each, more, ctas, warps;        // chunks of a CTA: `each`, one more for the first `more`
    __device__ __forceinline__ Deal(int total, int of_ctas, int of_warps) : ctas(of_ctas), warps(of_warps) {
        each = (unsigned)total / (unsigned)ctas;
        more = total - each * ctas;
    }
    // First chunk of a CTA; of the next one: its end.
    __device__ __forceinline__ int start(int cta) const { return cta * each + min(cta, more); }
    // ... of the run of its warp w.
    __device__ __forceinline__ int start(int cta, int w) const {
        const int n = each + (cta < more), part = (unsigned)n / (unsigned)warps;
        return start(cta) + w * part + min(w, n - part * warps);
    }
    // CTA that has chunk i.
    __device__ __forceinline__ int cta_with(int i) const {
        const int bound = more * (each + 1);
        return i < bound ? i / (each + 1) : more + (i - bound) / each;
    }
    // Runs that have a chunk, and CTA and warp of the i-th.
    __device__ __forceinline__ int runs() const { return more * min(warps, each + 1) + (ctas - more) * min(warps, each); }
    __device__ __forceinline__ int2 run(int i) const {
        const int big = min(warps, each + 1), bound = more * big;
        if (i < bound) return make_int2(i / big, i % big);
        const int small = min(warps, each);
        return make_int2(more + (i - bound) / small, (i - bound) % small);
    }
};
// A run's part of one unit.
struct Part {
    int b, unit, h, group, first, last, chunks;   // sequence; unit of all; KV head, group of its rows; chunks of the unit: [first, last) of `chunks`
    // u: of the sequence's units
    __device__ __forceinline__ void place(int u, int groups) {
        h = groups == 1 ? u : (unsigned)u / (unsigned)groups;
        group = u - h * groups;
    }
    // The part that begins with chunk `at`, of a run that ends with `end`; b: where to begin looking.
    __device__ __forceinline__ void find(const int* cum, int units, int groups, int b0, int at, int end) {
        b = b0;
        while (at >= cum[b + 1] * units) ++b;
        chunks = cum[b + 1] - cum[b];
        const int rest = at - cum[b] * units, u = (unsigned)rest / (unsigned)chunks;
        unit = b * units + u;
        place(u, groups);
        first = rest - u * chunks;
        last = min(chunks, first + end - at);
    }
    __device__ __forceinline__ bool whole() const { return first == 0 && last == chunks; }
};
__device__ __forceinline__ int sequence_with(const int* cum, int B, int units, int at) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cum[mid] * units <= at) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ int2* borders(const AttendArgs& a) { return reinterpret_cast<int2*>(a.part + (2ll + MOST_WARPS) * a.ctas * a.record); }

// Rows of q, out and lse [B,T,H*G] that a unit's rows stand for.
struct Rows {
    int first, base;                    // first row of the unit among the KV head's T * G; row of the tensors for query 0, head 0 of the KV head
    __device__ __forceinline__ Rows(const AttendArgs& a, int b, int h, int group) : first(group * a.rows), base(b * a.T * a.pool.H * a.G + h * a.G) {}
    // The tensors' row of row r and its query; -1 behind the last.  (Fewer than 64 rows: the quotient by G is that of a multiplication.)
    __device__ __forceinline__ int row(const AttendArgs& a, int r, int* query) const {
        const int R = first + r, t = (R * a.over_g) >> 16;
        *query = t;
        return r >= a.rows || t >= a.T ? -1 : base + t * (a.pool.H * a.G) + R - t * a.G;
    }
};
__device__ __forceinline__ Rows rows_of(const AttendArgs& a, int unit) {
    const unsigned bh = (unsigned)unit / (unsigned)a.groups, b = bh / (unsigned)a.pool.H;
    return Rows(a, b, bh - b * a.pool.H, unit - bh * a.groups);
}

// ---------------------------------------------------------------- a warp's ring
// Where 16-byte piece c of row r of a tile lies, so that the 8 lanes of a 16-byte load's (16 of an 8-byte load's) phase read different banks: lane
// (g, t) = (lane / 4, lane % 4) reads pieces by t of K's rows g, and pieces by g of V's rows 2t, 2t + 1.
template <int ROW>
__device__ __forceinline__ int piece(int r, int c) {
    if constexpr (ROW >= 128) return r * ROW + ((c ^ (r & 7)) << 4);
    const int line = r * ROW >> 7, slot = ((r * ROW & 127) >> 4) + c;
    return line * 128 + ((slot ^ (2 * (line & (ROW == 64 ? 3 : 1)))) << 4);
}

// Steps of a run, copied to shared memory STEPS - 1 ahead by the warp's own asynchronous copies.  ONE: a step's tokens are in one page.
template <int F, int D, int NT, bool ONE, bool TEAM>
struct Ring {
    using S = Shape<F, D, NT>;
    static constexpr int U = S::U, ROW = S::ROW, PAGES = ONE ? 1 : U, TOKENS_OF = TEAM ? S::TEAM_TOKENS : CHUNK;    // (of a chunk)
    const AttendArgs& a;
    const int* cum;
    uint32_t base, mine;                 // of the ring; where this lane's first piece of codes goes within a tile
    const uint8_t* more;                 // this lane's piece of scales or exponents: its tensor, bytes of a token there
    int per_token, lane, put, get;
    Part part;                           // what is copied next
    int units, end, at, n, token, stop, page[PAGES];
    int cached;                          // this lane's entry of the table, of the 32 from cached_from on
    unsigned cached_from;
    uint32_t gone;                       // PAGES bits a step, the oldest in the lowest: the page is not there

    // (begins with a part whose first chunk is `from`, and ends in front of chunk `last`)
    __device__ __forceinline__ Ring(const AttendArgs& args, const int* lengths, uint32_t to, int of_lane, int run_units, const Part& begin, int from, int last)
        : a(args), cum(lengths), base(to), lane(of_lane), put(0), get(0), part(begin), units(run_units), end(last), at(from), gone(0) {
        const int bytes = lane * 16;
        mine = piece<ROW>(bytes / ROW, bytes % ROW / 16);
        more = nullptr;
        per_token = 0;
        if constexpr (F != AKV_PAGE_FP16) {
            constexpr int N = S::SCALES / 16;                 // pieces of a tile's scales
            if (lane < 2 * N) {
                more = (lane < N ? a.pool.ks : a.pool.vs) + lane % (N ? N : 1) * 16;
                per_token = D / 16;
            } else if (lane < 2 * N + 2) {
                more = reinterpret_cast<const uint8_t*>(lane == 2 * N ? a.pool.ke : a.pool.ve);
                per_token = 1;
            }
        }
        enter();
        look();
#pragma unroll 1
        for (int i = 0; i < S::STEPS - 1; ++i) fill();
    }
    __device__ __forceinline__ void enter() {
        n = length_of(a.pool, part.b);
        token = part.first * TOKENS_OF;
        stop = min(n, part.last * TOKENS_OF);
        cached_from = 1u << 31;              // (far from any page: the first look reads)
    }
    // Pages of the step at `token`; -1 where there is none or nothing of the sequence in it.  The table is read 32 entries at a time, one per lane.
    __device__ __forceinline__ void look() {
#pragma unroll
        for (int u = 0; u < PAGES; ++u) {
            const int at_page = (token + 16 * u) >> a.pool.shift;
            if (at_page - cached_from >= 32u) {
                cached_from = at_page;
                cached = -1;
                if (at_page + lane <= (n - 1) >> a.pool.shift) cached = __ldg(a.pool.table + (unsigned)part.b * (unsigned)a.pool.width + at_page + lane);
            }
            const int x = __shfl_sync(0xFFFFFFFFu, cached, at_page - cached_from);
            page[u] = token + 16 * u < n ? x : -1;
        }
    }
    // The next step, if there is one; always a group, so that the groups count the steps.
    __device__ __forceinline__ void fill() {
        if (at < end) {
            const uint32_t to = base + put * S::STEP;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int x = page[ONE ? 0 : u], from = ONE ? token : token + 16 * u;
                const bool there = (unsigned)x < (unsigned)a.pool.n_pages;
                const unsigned row = (((unsigned)(there ? x : 0) * (unsigned)a.pool.H + part.h) << a.pool.shift) + (from & ((1 << a.pool.shift) - 1)) + (ONE ? 16 * u : 0);
                const unsigned long long byte = (unsigned long long)row * ROW + lane * 16;
                const uint8_t *k = a.pool.kc + byte, *v = a.pool.vc + byte;
                const uint32_t tile = to + u * 32 * ROW;
#pragma unroll
                for (int j = 0; j < ROW / 32; ++j) {
                    // (512 bytes further: 2, 4, 8 or 16 rows)
                    const uint32_t dst = tile + (ROW >= 128 ? (mine ^ ((j * (512 / ROW) & 7) << 4)) : mine) + j * 512;
                    copy16(dst, k + j * 512, there);
                    copy16(dst + 16 * ROW, v + j * 512, there);
                }
                if constexpr (F != AKV_PAGE_FP16)
                    if (per_token) copy16(to + U * 32 * ROW + u * S::MORE + lane * 16, more + (unsigned long long)row * per_token, there);
            }
            uint32_t bits = 0;
#pragma unroll
            for (int u = 0; u < PAGES; ++u) bits |= (unsigned)((unsigned)page[u] >= (unsigned)a.pool.n_pages) << u;
            gone |= bits << ((put >= get ? put - get : put - get + S::STEPS) * PAGES);
            token += S::TOKENS;
            if (token >= stop) {
                at += part.last - part.first;
                if (at < end) {
                    part.find(cum, units, a.groups, part.b, at, end);
                    enter();
                }
            }
            if (at < end) look();
        }
        cp_async_commit();
        put = put + 1 == S::STEPS ? 0 : put + 1;
    }
    // Waits for the step that is read next, requests the one whose place the last read has left; pages that are not there.
    __device__ __forceinline__ uint32_t take(uint32_t& without) {
        cp_async_wait<S::STEPS - 2>();
        __syncwarp();
        fill();
        const uint32_t from = base + get * S::STEP;
        without = gone & ((1u << PAGES) - 1);
        gone >>= PAGES;
        get = get + 1 == S::STEPS ? 0 : get + 1;
        return from;
    }
};

// ---------------------------------------------------------------- a warp's unit
// TWICE: 4 rows or fewer.  Their tile has them twice, in its columns 0 to 3 and 4 to 7: the scores are the same, and the values' product takes the rounded
// probabilities in the first and what rounding took in the others, so that it needs no second one (8 heads x 131072 tokens, e2m1: 43.9 us, with a second
// product 46.3).
template <int F, int D, int NT, bool ONE, bool TWICE>
struct Unit {
    static_assert(!TWICE || NT == 1, "one tile");
    using S = Shape<F, D, NT>;
    static constexpr int U = S::U, KW = S::KW, KS = S::KS, ROW = S::ROW;
    const AttendArgs& a;
    int g, t;
    uint32_t at_k, at_v;                 // of this lane's first piece within a tile
    uint32_t queries, table;             // shared memory
    uint32_t q[S::FEW ? KS : 1][NT][2];
    float acc[KS][NT][4], m[NT][2], l[NT][2];

    __device__ __forceinline__ Unit(const AttendArgs& args, int lane, uint32_t own)
        : a(args), g(lane >> 2), t(lane & 3), queries(own + S::RING), table(own + S::RING + S::QUERIES) {
        at_k = ROW >= 128 ? piece<ROW>(g, 2 * t) : ROW == 64 ? piece<ROW>(g, t) : piece<ROW>(g, t >> 1) + (t & 1) * 8;
        at_v = 16 * ROW + (ROW >= 128 ? piece<ROW>(2 * t, g) : ROW == 64 ? piece<ROW>(2 * t, g >> 1) + (g & 1) * 8 : piece<ROW>(2 * t, g >> 2) + (g & 3) * 4);
    }

    // Channels of the first operand's k = 2t, 2t + 1, 2t + 8, 2t + 9 in product s: this one and the next three.
    __device__ __forceinline__ int k_channel(int s) const {
        if constexpr (ROW == 256) return (s >> 2) * 64 + t * 16 + (s & 3) * 4;
        return t * (D / 4) + s * 4;
    }
    // Channel of row g of output tile i; that of row g + 8 is the next.
    __device__ __forceinline__ int v_channel(int i) const {
        if constexpr (ROW == 256) return (i >> 2) * 64 + g * 8 + (i & 3) * 2;
        return g * (D / 8) + 2 * i;
    }

    // (operands of two groups of 8 rows side by side)
    __device__ __forceinline__ uint32_t query_place(int s, int nt) const { return queries + (((s * 2 + (nt >> 1)) * 32 + 4 * g + t) * 2 + (nt & 1)) * 8; }
    __device__ __forceinline__ void multiply_keys(float (&s)[NT][4], int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
        if constexpr (S::FEW) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma(s[nt], a0, a1, a2, a3, q[i][nt][0], q[i][nt][1]);
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; nt += 2) {
                const uint4 w = lds128(query_place(i, nt));
                mma(s[nt], a0, a1, a2, a3, w.x, w.y);
                if (nt + 1 < NT) mma(s[nt + 1], a0, a1, a2, a3, w.z, w.w);
            }
        }
    }

    // Row of the unit that column c of tile nt has.
    __device__ __forceinline__ int row_at(int nt, int c) const { return 8 * nt + (TWICE ? c & 3 : c); }

    __device__ __forceinline__ void begin(const Rows& rows) {
        if constexpr (!S::FEW) __syncwarp();     // (the last unit's have been read)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            int query;
            const long long row = rows.row(a, row_at(nt, g), &query);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                uint2 w = make_uint2(0, 0);
                if (row >= 0) w = *reinterpret_cast<const uint2*>(a.q + row * D + k_channel(s));
                if constexpr (S::FEW) {
                    q[s][nt][0] = w.x;
                    q[s][nt][1] = w.y;
                } else {
                    asm volatile("st.shared.v2.u32 [%0], {%1,%2};\n" ::"r"(query_place(s, nt)), "r"(w.x), "r"(w.y) : "memory");
                }
            }
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < KS; ++i) acc[i][nt][0] = acc[i][nt][1] = acc[i][nt][2] = acc[i][nt][3] = 0.f;
        }
        if constexpr (!S::FEW) __syncwarp();
    }

    // What a step's exponents are needed as, a token per lane: its scores' factor, the exponent of its values, its values' weight.  (An exponent of
    // -128 comes out as a factor of -infinity: times the row's zeros NaN, as it should; the maximum takes -40, below what there is.)
    __device__ __forceinline__ void unfold(uint32_t step) {
        if constexpr (F != AKV_PAGE_FP16) {
#pragma unroll
            for (int i = 4 * g + t; i < S::TOKENS; i += 32) {
                const uint32_t from = step + U * 32 * ROW + (i >> 4) * S::MORE + 2 * S::SCALES + (i & 15);
                const int k = lds8_signed(from), v = lds8_signed(from + 16);
                const float weight = v == EXP_NAN ? NAN : __int_as_float((v + 127 + 15) << 23);
                asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%3};\n" ::"r"(table + i * 16), "f"(a.scale2 * __int_as_float((k + 127) << 23)),
                             "f"((float)max(v, -40)), "f"(weight) : "memory");
            }
            __syncwarp();
        }
    }

    // Scores of a step's tokens, s[u][nt]: rows g (first two) and g + 8 by query rows 2t, 2t + 1.
    __device__ __forceinline__ void scores(float (&s)[U][NT][4], uint32_t step) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t from = step + u * 32 * ROW + at_k;
            constexpr int H = KW / 2;
            uint32_t k[2][H];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if constexpr (ROW == 32) {
                    const uint2 w = lds64(from + half * 8 * ROW);
                    k[half][0] = w.x;
                    k[half][1] = w.y;
                } else {
#pragma unroll
                    for (int c = 0; c < H / 4; ++c) {
                        const uint4 w = lds128((from ^ ((c & 1) << 4)) + half * 8 * ROW + (c >> 1) * 128);
#pragma unroll
                        for (int i = 0; i < 4; ++i) k[half][4 * c + i] = u4w(w, i);
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[u][nt][0] = s[u][nt][1] = s[u][nt][2] = s[u][nt][3] = 0.f;
            if constexpr (F == AKV_PAGE_FP16) {
#pragma unroll
                for (int i = 0; i < KS; ++i) multiply_keys(s[u], i, k[0][2 * i], k[1][2 * i], k[0][2 * i + 1], k[1][2 * i + 1]);
            } else if constexpr (F == AKV_PAGE_E4M3) {
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t x[2], y[2];
                    e4m3_word(x, k[0][i]);
                    e4m3_word(y, k[1][i]);
                    multiply_keys(s[u], i, x[0], y[0], x[1], y[1]);
                }
            } else {
                const uint32_t scales = step + U * 32 * ROW + u * S::MORE + g * (D / 16) + t * (D / 64);
                const uint32_t s0 = e4m3_halves(D == 128 ? lds16(scales) : lds8(scales));
                const uint32_t s1 = e4m3_halves(D == 128 ? lds16(scales + D / 2) : lds8(scales + D / 2));
#pragma unroll
                for (int w = 0; w < H; ++w) {
                    // (8 channels of a word: two products; 16 have a scale)
                    const uint32_t f0 = __byte_perm(s0, s0, D == 128 && w >= 2 ? 0x3232 : 0x1010), f1 = __byte_perm(s1, s1, D == 128 && w >= 2 ? 0x3232 : 0x1010);
                    uint32_t x[4], y[4];
                    e2m1_word(x, k[0][w]);
                    e2m1_word(y, k[1][w]);
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        multiply_keys(s[u], 2 * w + i, hmul2_bits(x[2 * i], f0), hmul2_bits(y[2 * i], f1), hmul2_bits(x[2 * i + 1], f0),
                                      hmul2_bits(y[2 * i + 1], f1));
                }
            }
        }
    }

    // Scores to weights of the values, in place, and the running maximum and sum with them.  seen(nt, c): tokens below it are seen by the row;
    // without: bits of the pages that are not there.  ALL: every row sees the whole step.
    template <bool ALL>
    __device__ __forceinline__ void soften(float (&s)[U][NT][4], uint32_t without, int at, const int (&seen)[NT][2]) {
        float top[NT][2], f[U][2], unit[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float e = 0.f;
                f[u][half] = a.scale2;
                unit[u][half] = LIFT;
                if constexpr (F != AKV_PAGE_FP16) {
                    const uint4 w = lds128(table + (16 * u + 8 * half + g) * 16);
                    f[u][half] = __uint_as_float(w.x);
                    e = __uint_as_float(w.y);
                    unit[u][half] = __uint_as_float(w.z);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float& x = s[u][nt][2 * half + c];
                        if (!ALL) {
                            x *= f[u][half];
                            if (missing(without, u) || at + 16 * u + g + 8 * half >= seen[nt][c]) x = -INFINITY;
                        }
                        const float y = ALL ? fmaf(x, f[u][half], e) : x + e;
                        top[nt][c] = u == 0 && half == 0 ? y : fmaxf(top[nt][c], y);
                    }
            }
        bool higher = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) top[nt][c] = fmaxf(top[nt][c], __shfl_xor_sync(0xFFFFFFFFu, top[nt][c], o));
                higher |= top[nt][c] > m[nt][c];
            }
        if (__any_sync(0xFFFFFFFFu, higher)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float g2[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float y = fmaxf(top[nt][c], m[nt][c]);
                    g2[c] = y == m[nt][c] ? 1.f : ex2(m[nt][c] - y);
                    m[nt][c] = y;
                    l[nt][c] *= g2[c];
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    acc[i][nt][0] *= g2[0];
                    acc[i][nt][1] *= g2[1];
                    acc[i][nt][2] *= g2[0];
                    acc[i][nt][3] *= g2[1];
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float base = m[nt][c] == -INFINITY ? 0.f : m[nt][c];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float& x = s[u][nt][2 * half + c];
                        const bool gone = !ALL && (missing(without, u) || at + 16 * u + g + 8 * half >= seen[nt][c]);
                        const float p = ex2(ALL ? fmaf(x, f[u][half], -base) : x - base);
                        l[nt][c] += p;                              // (of what is not seen: 0)
                        x = gone ? 0.f : p * unit[u][half];
                    }
            }
    }

    static __device__ __forceinline__ bool missing(uint32_t without, int u) { return (without >> (ONE ? 0 : u)) & 1; }

    // A tile's values: tokens 2t, 2t + 1, 2t + 8, 2t + 9; zeros for those that lie behind the sequence (limit: tokens of the tile that do not),
    // whatever is there.
    __device__ __forceinline__ void load_v(uint32_t (&v)[KW], uint32_t (&scale)[2], uint32_t step, int u, int limit) {
        constexpr int W = KW / 4;
        const uint32_t from = step + u * 32 * ROW + at_v;
        uint32_t bytes[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x = (ROW >= 128 ? (from ^ ((i & 1) << 4)) + (i & 1) * ROW : from ^ ((i & 1) * ROW)) + (i >> 1) * 8 * ROW;
            if constexpr (ROW >= 128) {
#pragma unroll
                for (int c = 0; c < W / 4; ++c) {
                    const uint4 w = lds128(x + c * 128);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i * W + 4 * c + j] = u4w(w, j);
                }
            } else if constexpr (ROW == 64) {
                const uint2 w = lds64(x);
                v[i * W] = w.x;
                v[i * W + 1] = w.y;
            } else {
                v[i] = lds32(x);
            }
            bytes[i] = 0;
            if constexpr (F == AKV_PAGE_E2M1)
                bytes[i] = lds8(step + U * 32 * ROW + u * S::MORE + S::SCALES + (2 * t + (i & 1) + (i >> 1) * 8) * (D / 16) + (D == 128 ? g : g >> 1));
        }
        if (limit < 16) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (2 * t + (i & 1) + (i >> 1) * 8 >= limit) {
                    bytes[i] = 0;
#pragma unroll
                    for (int j = 0; j < W; ++j) v[i * W + j] = 0;
                }
        }
        if constexpr (F == AKV_PAGE_E2M1) {
            scale[0] = e4m3_halves(__byte_perm(bytes[0], bytes[1], 0x0040));
            scale[1] = e4m3_halves(__byte_perm(bytes[2], bytes[3], 0x0040));
        }
    }
    // fn(i, a0, a1, a2, a3): the first operand of output tile i.
    template <class Fn>
    __device__ __forceinline__ void tiles(const uint32_t (&v)[KW], const uint32_t (&scale)[2], Fn fn) {
        constexpr int W = KW / 4;              // words of a token
        if constexpr (F == AKV_PAGE_FP16) {
#pragma unroll
            for (int i = 0; i < KS; ++i)
                fn(i, __byte_perm(v[i], v[W + i], 0x5410), __byte_perm(v[i], v[W + i], 0x7632),
                   __byte_perm(v[2 * W + i], v[3 * W + i], 0x5410), __byte_perm(v[2 * W + i], v[3 * W + i], 0x7632));
        } else if constexpr (F == AKV_PAGE_E4M3) {
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint32_t x = __byte_perm(v[i >> 1], v[W + (i >> 1)], i & 1 ? 0x7362 : 0x5140);
                const uint32_t y = __byte_perm(v[2 * W + (i >> 1)], v[3 * W + (i >> 1)], i & 1 ? 0x7362 : 0x5140);
                uint32_t p[2], r[2];
                e4m3_word(p, x);
                e4m3_word(r, y);
                fn(i, p[0], p[1], r[0], r[1]);
            }
        } else {
#pragma unroll
            for (int w = 0; w < W; ++w) {
                constexpr uint32_t LOW = 0x0F0F0F0Fu;
                // two tokens' nibbles of one channel in a byte: even channels, odd ones
                const uint32_t e0 = (v[w] & LOW) | ((v[W + w] << 4) & ~LOW), o0 = ((v[w] >> 4) & LOW) | (v[W + w] & ~LOW);
                const uint32_t e1 = (v[2 * W + w] & LOW) | ((v[3 * W + w] << 4) & ~LOW), o1 = ((v[2 * W + w] >> 4) & LOW) | (v[3 * W + w] & ~LOW);
                uint32_t x0[4], y0[4], x1[4], y1[4];
                e2m1_word(x0, e0);
                e2m1_word(y0, o0);
                e2m1_word(x1, e1);
                e2m1_word(y1, o1);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    fn(4 * w + i, hmul2_bits(x0[i], scale[0]), hmul2_bits(y0[i], scale[0]), hmul2_bits(x1[i], scale[1]), hmul2_bits(y1[i], scale[1]));
            }
        }
    }
    // limit: tokens of the step that are the sequence's.  (rest: what rounding took from the probabilities)
    __device__ __forceinline__ void add_values(const float (&s)[U][NT][4], uint32_t step, int at, int limit, const int (&seen)[NT][2]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint32_t v[KW], scale[2], w[NT][2], rest[NT][2];
            load_v(v, scale, step, u, limit - 16 * u);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float x = s[u][nt][2 * i], y = s[u][nt][2 * i + 1];
                    const uint32_t near = halves_bits(x, y);
                    const float2 f = halves_floats(near);
                    rest[nt][i] = halves_bits(x - f.x, y - f.y);
                    w[nt][i] = transposed(TWICE && t >= 2 ? rest[nt][i] : near);
                    if (!TWICE) rest[nt][i] = transposed(rest[nt][i]);
                }
            if (F == AKV_PAGE_FP16 && __any_sync(0xFFFFFFFFu, odd(v))) {
                add_odd_values(v, w, rest, at + 16 * u, at + limit, seen);
                continue;
            }
            tiles(v, scale, [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma(acc[i][nt], a0, a1, a2, a3, w[nt][0], w[nt][1]);
                if (TWICE) return;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma(acc[i][nt], a0, a1, a2, a3, rest[nt][0], rest[nt][1]);
            });
        }
    }
    // The same where some values are not finite (fp16 pages alone: elsewhere codes are).  0 * inf would be NaN: every query's product is formed by
    // itself, without the newest tokens that it does not see, and comes out as if those were not there.  What rounding took from a probability has any
    // sign, and multiplies the finite values alone.
    __device__ __forceinline__ void add_odd_values(const uint32_t (&v)[KW], const uint32_t (&w)[NT][2], const uint32_t (&rest)[NT][2], int at, int n,
                                                   const int (&seen)[NT][2]) {
        const uint32_t none[2] = {0, 0};
#pragma unroll 1
        for (int limit = n - a.T + 1; limit <= n; ++limit) {
            bool there[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) there[i] = at + 2 * t + (i & 1) + (i >> 1) * 8 < limit;
            const uint32_t m01 = (there[0] ? 0xFFFFu : 0u) | (there[1] ? 0xFFFF0000u : 0u), m23 = (there[2] ? 0xFFFFu : 0u) | (there[3] ? 0xFFFF0000u : 0u);
            tiles(v, none, [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                a0 &= m01, a1 &= m01, a2 &= m23, a3 &= m23;
                const uint32_t f0 = finite(a0), f1 = finite(a1), f2 = finite(a2), f3 = finite(a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float c[4] = {acc[i][nt][0], acc[i][nt][1], acc[i][nt][2], acc[i][nt][3]};
                    float y[4] = {c[0], c[1], c[2], c[3]};
                    mma(c, a0, a1, a2, a3, w[nt][0], w[nt][1]);
                    mma(TWICE ? y : c, f0, f1, f2, f3, TWICE ? w[nt][0] : rest[nt][0], TWICE ? w[nt][1] : rest[nt][1]);
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        if (TWICE && t >= 2) c[x] = y[x];
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        if (seen[nt][x & 1] == limit) acc[i][nt][x] = c[x];
                }
            });
        }
    }
    static __device__ __forceinline__ uint32_t finite(uint32_t w) {
        if ((w & 0x7C00u) == 0x7C00u) w &= 0xFFFF0000u;
        return (w & 0x7C000000u) == 0x7C000000u ? w & 0xFFFFu : w;
    }
    static __device__ __forceinline__ bool odd(const uint32_t (&v)[KW]) {
        uint32_t x[2] = {0, 0};                  // (0 as long as all are finite, then NaN)
#pragma unroll
        for (int i = 0; i < KW; ++i) x[i & 1] = hfma2_bits(v[i], 0, x[i & 1]);
        return finite(x[0]) != x[0] || finite(x[1]) != x[1];
    }

    // The unit's result: sums over the lanes, then to rows.
    __device__ __forceinline__ void close() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[nt][c] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][c], o);
        if (TWICE) {                             // (columns 4 to 7 to 0 to 3)
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[i][0][x] += __shfl_xor_sync(0xFFFFFFFFu, acc[i][0][x], 2);
        }
    }
    __device__ __forceinline__ void write(const Rows& rows) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                int query;
                const long long row = rows.row(a, 8 * nt + 2 * t + c, &query);
                if (row < 0) continue;
                const float inv = l[nt][c] == 0.f ? 0.f : 1.f / (l[nt][c] * LIFT);
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const __half2 h = __floats2half2_rn(acc[i][nt][c] * inv, acc[i][nt][2 + c] * inv);
                    *reinterpret_cast<__half2*>(a.out + row * D + v_channel(i)) = h;
                }
                if (a.lse && g == 0) a.lse[row] = l[nt][c] == 0.f ? -INFINITY : (m[nt][c] + log2f(l[nt][c])) * LN2;
            }
    }
    // Record: rows of D + 4 floats, output sums, then maximum and sum.
    __device__ __forceinline__ void record(float* to) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (8 * nt + 2 * t + c >= a.rows) continue;
                float* row = to + (8 * nt + 2 * t + c) * (D + 4);
#pragma unroll
                for (int i = 0; i < KS; ++i)
                    *reinterpret_cast<float2*>(row + v_channel(i)) = make_float2(acc[i][nt][c], acc[i][nt][2 + c]);
                if (g == 0) *reinterpret_cast<float2*>(row + D) = make_float2(m[nt][c], l[nt][c]);
            }
    }
};

// A row's result to out and lse: sums x of 4 channels from `channel` on, over (maximum, sum).
template <int D>
__device__ __forceinline__ void write_row(const AttendArgs& a, int unit, int r, int channel, float4 x, float top, float sum) {
    int query;
    const long long row = rows_of(a, unit).row(a, r, &query);
    if (row < 0) return;
    const float inv = sum == 0.f ? 0.f : 1.f / (sum * LIFT);
    const __half2 lo = __floats2half2_rn(x.x * inv, x.y * inv), hi = __floats2half2_rn(x.z * inv, x.w * inv);
    *reinterpret_cast<uint2*>(a.out + row * D + channel) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    if (a.lse && channel == 0) a.lse[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * LN2;
}
// Joins a row of `count` records by 8 lanes (sub: which of them); fn(i) = the row in the i-th.  (A warp has four rows at a time: what it waits for are a
// few loads, one after the other.)
template <int D, class Fn>
__device__ __forceinline__ void join_few(const AttendArgs& a, int unit, int r, int count, int sub, Fn fn, float* record) {
    constexpr int N = D / 32;
    float top = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int i = 0; i < count; ++i) top = fmaxf(top, fn(i)[D]);
    const float base = top == -INFINITY ? 0.f : top;
    float4 o[N];
#pragma unroll
    for (int c = 0; c < N; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int i = 0; i < count; ++i) {
        const float* x = fn(i);
        const float2 ml = *reinterpret_cast<const float2*>(x + D);
        const float f = ex2(ml.x - base);
        sum = fmaf(f, ml.y, sum);
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const float4 y = *reinterpret_cast<const float4*>(x + 32 * c + 4 * sub);
            o[c] = make_float4(fmaf(f, y.x, o[c].x), fmaf(f, y.y, o[c].y), fmaf(f, y.z, o[c].z), fmaf(f, y.w, o[c].w));
        }
    }
#pragma unroll
    for (int c = 0; c < N; ++c) {
        if (record) *reinterpret_cast<float4*>(record + 32 * c + 4 * sub) = o[c];
        else write_row<D>(a, unit, r, 32 * c + 4 * sub, o[c], top, sum);
    }
    if (record && sub == 0) *reinterpret_cast<float2*>(record + D) = make_float2(top, sum);
}

// The same, two records at a time and their maxima with their sums: where a CTA has many rows to join its warps wait for these loads again and again (20
// rows, 32 x 8 heads x up to 4096 tokens, 4 bits: 56.1 -> 54.7 us; one query row a head 31.6 -> 32.1).
template <int D, class Fn>
__device__ __forceinline__ void join_pairs(const AttendArgs& a, int unit, int r, int count, int sub, Fn fn, float* record) {
    constexpr int N = D / 32;
    float top = -INFINITY, sum = 0.f;
    float4 o[N];
#pragma unroll
    for (int c = 0; c < N; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int i = 0; i < count; i += 2) {
        const bool two = i + 1 < count;
        const float *x = fn(i), *z = two ? fn(i + 1) : x;
        const float2 ml = *reinterpret_cast<const float2*>(x + D);
        float2 nl = *reinterpret_cast<const float2*>(z + D);
        float4 y[N], w[N];
#pragma unroll
        for (int c = 0; c < N; ++c) {
            y[c] = *reinterpret_cast<const float4*>(x + 32 * c + 4 * sub);
            w[c] = *reinterpret_cast<const float4*>(z + 32 * c + 4 * sub);
        }
        if (!two) {
            nl = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int c = 0; c < N; ++c) w[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const float m = fmaxf(top, fmaxf(ml.x, nl.x)), base = m == -INFINITY ? 0.f : m;
        const float was = ex2(top - base), f = ex2(ml.x - base), g = ex2(nl.x - base);
        sum = fmaf(g, nl.y, fmaf(f, ml.y, was * sum));
        top = m;
#pragma unroll
        for (int c = 0; c < N; ++c)
            o[c] = make_float4(fmaf(g, w[c].x, fmaf(f, y[c].x, was * o[c].x)), fmaf(g, w[c].y, fmaf(f, y[c].y, was * o[c].y)),
                               fmaf(g, w[c].z, fmaf(f, y[c].z, was * o[c].z)), fmaf(g, w[c].w, fmaf(f, y[c].w, was * o[c].w)));
    }
#pragma unroll
    for (int c = 0; c < N; ++c) {
        if (record) *reinterpret_cast<float4*>(record + 32 * c + 4 * sub) = o[c];
        else write_row<D>(a, unit, r, 32 * c + 4 * sub, o[c], top, sum);
    }
    if (record && sub == 0) *reinterpret_cast<float2*>(record + D) = make_float2(top, sum);
}

// Joins the records first .. last - 1 of a row by a warp, 4 channels a lane (of 128; of 64 half of the lanes have none); row(i): the i-th.
template <int D, class Fn>
__device__ __forceinline__ void join_row(int first, int last, int lane, Fn row, float4& o, float& top, float& sum) {
    const int channel = 4 * lane;
    top = -INFINITY;
    sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = first; i0 < last; i0 += 32) {
        float2 ml = make_float2(-INFINITY, 0.f);
        if (i0 + lane < last) ml = *reinterpret_cast<const float2*>(row(i0 + lane) + D);
        float m = ml.x;
#pragma unroll
        for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, x));
        m = fmaxf(m, top);
        const float base = m == -INFINITY ? 0.f : m, was = ex2(top - base), f = ex2(ml.x - base);
        o = make_float4(o.x * was, o.y * was, o.z * was, o.w * was);
        sum *= was;
        top = m;
        const int here = min(32, last - i0);
#pragma unroll 8
        for (int i = 0; i < here; ++i) {
            const float g = __shfl_sync(0xFFFFFFFFu, f, i);
            sum = fmaf(g, __shfl_sync(0xFFFFFFFFu, ml.y, i), sum);
            if (channel < D) {
                const float4 y = *reinterpret_cast<const float4*>(row(i0 + i) + channel);
                o = make_float4(fmaf(g, y.x, o.x), fmaf(g, y.y, o.y), fmaf(g, y.z, o.z), fmaf(g, y.w, o.w));
            }
        }
    }
}
// Row r of `count` records by `shares` warps, of which this is number `share`, through parts [shares][D + 4] in shared memory.  Every warp of the
// block calls it (it synchronises), those without a row with count 0.
template <int D, class Fn>
__device__ __forceinline__ void join_many(const AttendArgs& a, int unit, int r, int count, int share, int shares, int lane, float (*parts)[D + 4], Fn row) {
    const int each = (count + shares - 1) / shares, first = share * each;
    float4 o;
    float top, sum;
    join_row<D>(first, min(count, first + each), lane, row, o, top, sum);
    if (shares == 1) {
        if (count > 0 && 4 * lane < D) write_row<D>(a, unit, r, 4 * lane, o, top, sum);
        return;
    }
    if (count > 0) {
        if (4 * lane < D) *reinterpret_cast<float4*>(parts[share] + 4 * lane) = o;
        if (lane == 0) *reinterpret_cast<float2*>(parts[share] + D) = make_float2(top, sum);
    }
    __syncthreads();
    if (count > 0 && share == 0 && lane < 8) join_few<D>(a, unit, r, min(shares, (count + each - 1) / each), lane, [&](int i) { return parts[i]; }, nullptr);
    __syncthreads();
}

// TEAM: a cluster of CTAs has one unit, and its records are joined there.
template <int F, int D, int NT, bool ONE, bool TEAM, bool TWICE>
__global__ void __launch_bounds__(32 * Shape<F, D, NT>::WARPS, 1) attend_kernel(AttendArgs a) {
    using S = Shape<F, D, NT>;
    constexpr int WARPS = S::WARPS;
    extern __shared__ __align__(128) uint8_t rings[];
    int* cum = reinterpret_cast<int*>(rings + S::SMEM);
    __shared__ int sums[WARPS], s_unit[2 * WARPS], s_tasks;     // (s_unit: units of the records of each run's first part and of its last, or -1)
    __shared__ int4 s_task[2 * WARPS];                         // unit, its first of s_slots, how many, where they go
    __shared__ int s_slots[2 * WARPS];
    __shared__ int2 s_border;
    __shared__ __align__(16) float s_parts[TEAM ? WARPS : 1][D + 4];
    pdl_turn();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int units = a.pool.H * a.groups;
    // what is dealt: the chunks of all units to all warps, or the chunks of the cluster's unit to its warps
    Part part;
    int total, ctas = gridDim.x, cta = blockIdx.x;
    if constexpr (TEAM) {
        ctas = a.team;
        part.unit = blockIdx.x / ctas;
        cta = blockIdx.x - part.unit * ctas;
        part.b = part.unit / units;
        part.place(part.unit - part.b * units, a.groups);
        total = part.chunks = chunks_of<S::TEAM_TOKENS>(length_of(a.pool, part.b));
    } else {
        add_lengths<32 * WARPS>(a, cum, sums);
        total = cum[a.B] * units;
    }
    const Deal deal(total, ctas, WARPS);
    int at = deal.start(cta, warp), end = deal.start(cta, warp + 1);
    if (!TEAM && lane < 2) s_unit[2 * warp + lane] = -1;
    __syncwarp();
    // Records: of a part that ends its run in the run's ring, which nobody needs any more; of one in front of others in global memory.
    float* last_record = reinterpret_cast<float*>(rings + warp * S::OWN);
    float* first_record = a.part + (2ll * gridDim.x + blockIdx.x * WARPS + warp) * S::RECORD;
    if (at < end) {
        if constexpr (TEAM) {
            part.first = at;
            part.last = end;
        } else {
            part.find(cum, units, a.groups, sequence_with(cum, a.B, units, at), at, end);
        }
        Ring<F, D, NT, ONE, TEAM> ring(a, cum, smem_u32(last_record), lane, units, part, at, end);
        Unit<F, D, NT, ONE, TWICE> unit(a, lane, smem_u32(last_record));
        for (;;) {
            constexpr int TOKENS_OF = TEAM ? S::TEAM_TOKENS : CHUNK;
            const Rows rows(a, part.b, part.h, part.group);
            const int n = length_of(a.pool, part.b), stop = min(n, part.last * TOKENS_OF);
            int seen[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    int query;
                    seen[nt][c] = rows.row(a, unit.row_at(nt, 2 * unit.t + c), &query) < 0 ? 0 : n - a.T + 1 + query;
                }
            unit.begin(rows);
            int token = part.first * TOKENS_OF;
#pragma unroll 1
            do {
                uint32_t without;
                const uint32_t step = ring.take(without);
                float s[S::U][NT][4];
                unit.unfold(step);
                unit.scores(s, step);
                if (token + S::TOKENS <= n - a.T + 1 && without == 0) unit.template soften<true>(s, without, token, seen);
                else unit.template soften<false>(s, without, token, seen);
                unit.add_values(s, step, token, n - token, seen);
                token += S::TOKENS;
            } while (token < stop);
            unit.close();
            at += part.last - part.first;
            if (part.whole()) {
                unit.write(rows);
            } else {
                const bool over = TEAM || at >= end;
                if (over) {
                    cp_async_wait<0>();
                    __syncwarp();
                }
                unit.record(over ? last_record : first_record);
                if (!TEAM && lane == 0) s_unit[2 * warp + over] = part.unit;
            }
            if (TEAM || at >= end) break;
            part.find(cum, units, a.groups, part.b, at, end);
        }
    }
    if constexpr (TEAM) {
        if (total == 1) return;                                // (written; the same in the whole cluster)
        cluster_sync();
        // Runs that got something, in order; the cluster's CTAs take the rows in turn, a warp or more of them a row.
        const int count = deal.runs(), rows = (a.rows - cta + ctas - 1) / ctas;
        const int shares = count <= 8 ? 1 : max(1, WARPS / max(1, rows)), at_once = WARPS / shares, mine = warp / shares;
        for (int x0 = 0; x0 < rows; x0 += at_once) {
            const int x = x0 + mine, r = cta + x * ctas;
            join_many<D>(a, part.unit, r, mine < at_once && x < rows ? count : 0, warp % shares, shares, lane, s_parts + mine * shares, [&](int i) -> const float* {
                const int2 run = deal.run(i);
                unsigned long long there;
                asm("mapa.u64 %0, %1, %2;\n" : "=l"(there) : "l"(rings + run.y * S::OWN), "r"(run.x));
                return reinterpret_cast<const float*>(there) + r * (D + 4);
            });
        }
        cluster_sync();                                        // (nobody leaves while its records are read)
        return;
    }
    __syncthreads();
    // A unit whose records all are in this CTA is written, of another one record is left: the CTA's first where it began in front of it, else its
    // second, and for the kernel that joins those the unit and the last CTA that has a part of it.
    if (warp == 0) {
        const int unit = lane < 2 * WARPS ? s_unit[lane] : -1;
        const unsigned same = __match_any_sync(0xFFFFFFFFu, unit);
        const bool leads = unit >= 0 && (same & ((1u << lane) - 1)) == 0;
        const unsigned leaders = __ballot_sync(0xFFFFFFFFu, leads), below = (1u << lane) - 1;
        const int place = __popc(__ballot_sync(0xFFFFFFFFu, unit >= 0) & below);       // records in front of this one
        if (unit >= 0) s_slots[place] = lane;
        if (lane == 0) {
            s_tasks = __popc(leaders);
            s_border = make_int2(-1, 0);
        }
        __syncwarp();
        if (leads) {
            const int b = unit / units, chunks = cum[b + 1] - cum[b], from = cum[b] * units + (unit - b * units) * chunks;
            const bool before = from < deal.start(blockIdx.x), after = from + chunks > deal.start(blockIdx.x + 1);
            if (!before && after) s_border = make_int2(unit, deal.cta_with(from + chunks - 1));
            s_task[__popc(leaders & below)] = make_int4(unit, place, __popc(same), before ? 0 : after ? 1 : -1);
        }
        __syncwarp();
        if (lane == 0) borders(a)[blockIdx.x] = s_border;
    }
    __syncthreads();
    // A row by a warp where there are few (8 x 32 heads x 4096 tokens: 51.6 us, four rows at a time 55.3), else four (32 sequences of 5 tokens and 4
    // heads a row: 66 us, one 81).
    const int rows = s_tasks * a.rows;
    const bool few = rows <= 2 * WARPS;
    for (int x = few ? warp : warp * 4 + (lane >> 3); x < rows; x += few ? WARPS : 4 * WARPS) {
        const int i = x / a.rows, r = x - i * a.rows;
        const int4 task = s_task[i];
        float* record = task.w < 0 ? nullptr : a.part + ((long long)(2 * blockIdx.x + task.w) * 8 * NT + r) * (D + 4);
        auto row = [&](int k) {
            const int slot = s_slots[task.y + k], w = slot >> 1;
            return (slot & 1 ? reinterpret_cast<const float*>(rings + w * S::OWN) : a.part + (2ll * gridDim.x + blockIdx.x * WARPS + w) * S::RECORD) + r * (D + 4);
        };
        if (few) {
            float4 o;
            float top, sum;
            join_row<D>(0, task.z, lane, row, o, top, sum);
            if (4 * lane < D) {
                if (record) *reinterpret_cast<float4*>(record + 4 * lane) = o;
                else write_row<D>(a, task.x, r, 4 * lane, o, top, sum);
            }
            if (record && lane == 0) *reinterpret_cast<float2*>(record + D) = make_float2(top, sum);
        } else {
            if constexpr (NT == 1) join_few<D>(a, task.x, r, task.z, lane & 7, row, record);
            else join_pairs<D>(a, task.x, r, task.z, lane & 7, row, record);
        }
    }
}

// One CTA per CTA of attend_kernel: where a unit begins there and ends in another one, its records are joined: a row by a warp, by all that
// there are for it where the records are many (their parts are joined in shared memory).  Bound by latency: the first two records, if there are any, lie
// where they always do and are loaded before it is known whether there are.
constexpr int JOINERS = 16;
template <int D, int NT>
__global__ void __launch_bounds__(32 * JOINERS) join_kernel(AttendArgs a) {
    __shared__ __align__(16) float parts[JOINERS][D + 4];
    pdl_turn();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, from = blockIdx.x;
    auto record = [&](int r, int i) { return a.part + ((long long)(2 * (from + i) + (i == 0)) * 8 * NT + r) * (D + 4); };
    float4 y[2];
    float2 ml[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool there = warp < a.rows && from + 1 < a.ctas;
        y[i] = there && 4 * lane < D ? *reinterpret_cast<const float4*>(record(warp, i) + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
        ml[i] = there ? *reinterpret_cast<const float2*>(record(warp, i) + D) : make_float2(0.f, 0.f);
    }
    const int2 border = borders(a)[from];
    if (border.x < 0) return;
    const int count = border.y - from + 1;
    if (count <= 8) {
        for (int r = warp; r < a.rows; r += JOINERS) {
            float4 o;
            float top, sum;
            if (r == warp) {
                join_row<D>(2, count, lane, [&](int i) { return record(r, i); }, o, top, sum);
                const float m = fmaxf(top, fmaxf(ml[0].x, ml[1].x)), base = m == -INFINITY ? 0.f : m;
                const float f = ex2(top - base), f0 = ex2(ml[0].x - base), f1 = ex2(ml[1].x - base);
                o = make_float4(fmaf(f0, y[0].x, fmaf(f1, y[1].x, f * o.x)), fmaf(f0, y[0].y, fmaf(f1, y[1].y, f * o.y)),
                                fmaf(f0, y[0].z, fmaf(f1, y[1].z, f * o.z)), fmaf(f0, y[0].w, fmaf(f1, y[1].w, f * o.w)));
                sum = fmaf(f0, ml[0].y, fmaf(f1, ml[1].y, f * sum));
                top = m;
            } else {
                join_row<D>(0, count, lane, [&](int i) { return record(r, i); }, o, top, sum);
            }
            if (4 * lane < D) write_row<D>(a, border.x, r, 4 * lane, o, top, sum);
        }
        return;
    }
    const int shares = max(1, JOINERS / a.rows), at_once = JOINERS / shares, mine = warp / shares;      // (warps of a row, rows at a time)
    for (int r0 = 0; r0 < a.rows; r0 += at_once) {
        const int r = r0 + mine;
        join_many<D>(a, border.x, r, mine < at_once && r < a.rows ? count : 0, warp % shares, shares, lane, parts + mine * shares,
                     [&](int i) { return record(r, i); });
    }
}

template <int F, int D, int NT, bool ONE, bool TEAM, bool TWICE>
int launch(const AttendArgs& a, const Plan& p, bool joined, cudaStream_t st) {
    using S = Shape<F, D, NT>;
    static_assert(S::WARPS <= MOST_WARPS, "workspace");
    const int smem = S::SMEM + (a.B + 1) * 4;
    static thread_local int set_for = -1;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && set_for != dev) {
        // (the most it is ever launched with)
        e = cudaFuncSetAttribute(attend_kernel<F, D, NT, ONE, TEAM, TWICE>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM + 4097 * 4);
        if (e == cudaSuccess) set_for = dev;
    }
    if (e != cudaSuccess) return cuda_status(e, "paged_attention");
    if constexpr (TEAM) {
        launch_cluster(attend_kernel<F, D, NT, ONE, TEAM, TWICE>, a.team, dim3((unsigned)(a.B * a.pool.H * a.groups * a.team)), dim3(32 * S::WARPS), S::SMEM, st, a);
        return cuda_status(cudaGetLastError(), "paged_attention launch");
    }
    launch_chained(attend_kernel<F, D, NT, ONE, TEAM, TWICE>, dim3(p.ctas), dim3(32 * S::WARPS), smem, st, a);
    const int rc = cuda_status(cudaGetLastError(), "paged_attention launch");
    if (rc != AKV_OK || !joined || p.ctas == 1) return rc;
    launch_chained(join_kernel<D, NT>, dim3(p.ctas), dim3(32 * JOINERS), 0, st, a);
    return cuda_status(cudaGetLastError(), "paged_attention join launch");
}
template <int F, int D, int NT, bool ONE, bool TEAM>
int launch_twice(const AttendArgs& a, const Plan& p, bool joined, cudaStream_t st) {
    if constexpr (NT == 1)
        if (a.rows <= 4) return launch<F, D, NT, ONE, TEAM, true>(a, p, joined, st);
    return launch<F, D, NT, ONE, TEAM, false>(a, p, joined, st);
}
template <int F, int D, int NT>
int launch_pages(const AttendArgs& a, const Plan& p, bool joined, cudaStream_t st) {
    if constexpr (Shape<F, D, NT>::U > 1)
        if (Shape<F, D, NT>::TOKENS > 1 << a.pool.shift)
            return a.team ? launch_twice<F, D, NT, false, true>(a, p, joined, st) : launch_twice<F, D, NT, false, false>(a, p, joined, st);
    return a.team ? launch_twice<F, D, NT, true, true>(a, p, joined, st) : launch_twice<F, D, NT, true, false>(a, p, joined, st);
}
template <int F, int D>
int launch_rows(const AttendArgs& a, const Plan& p, bool joined, cudaStream_t st) {
    if (p.nt == 1) return launch_pages<F, D, 1>(a, p, joined, st);
    if (p.nt == 2) return launch_pages<F, D, 2>(a, p, joined, st);
    if (p.nt == 3) return launch_pages<F, D, 3>(a, p, joined, st);
    return launch_pages<F, D, 4>(a, p, joined, st);
}

}  // namespace
}  // namespace akv
