// Attention of the newest tokens of each sequence over its pages.
//   attend_kernel   query rows of a (sequence, KV head) against its tokens; one pass with a running maximum and sum
//   join_kernel     joins the partial results of units that several CTAs share
//
//   s_rj = scale q_r . k_j, o_r = sum_j exp(s_rj - m_r) v_j / l_r, l_r = sum_j exp(s_rj - m_r), over the tokens j that row r sees.
//
// Every byte of the tokens is read once: bound by HBM, and for the 4-bit format almost as much by the instructions that unpack it.
// Work: a unit is up to 16 query rows of one (sequence, KV head), its tokens in chunks of 64.  The chunks of all units in a row are dealt to
// the warps in equal contiguous runs: lengths are only known on the device, and every SM gets the same whatever they are.  Each CTA
// adds up the lengths itself.  A warp needs no other one: codes come straight into registers as operand fragments (no shared memory is
// on their way), the next step's while this one's are multiplied.  Where a run begins or ends inside a unit it leaves a record, and
// the CTA joins those of its warps; what is left between CTAs is join_kernel's.
//
// Operands: tokens are the rows of the products' first operand, query rows the columns of the second - 8 of them, which one KV head's query heads
// fill, where the other way round 16 would be half empty.  Which channel is which k, and which token which row, is free as long as both
// operands agree, and chosen so that a lane's loads are 16 bytes and need the fewest permutations.
#include "akv_paged.cuh"

namespace akv {
namespace {

constexpr int CHUNK = 64;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// Probabilities enter their product as two halves (what the first leaves out is the second), times 2^15: 22 bits of each, as long as it is above
// 2^-28 of the largest, of which the 11 bits of one half would show beside the output's own rounding.
constexpr float LIFT = 32768.f;

struct AttendArgs {
    Pool pool;
    const __half* q;
    __half* out;
    float *lse, *part;
    int B, T, G, groups, rows;      // units per (sequence, KV head), query rows of a unit
    float scale2;                   // scale * log2(e)
};

template <int F, int D, int NT>
struct Shape {
    static constexpr int ROW = row_bytes<F>(D);
    static constexpr int KW = ROW / 8;                        // words of 16 tokens of K (or of V) in a lane
    static constexpr int U = KW >= 32 ? 1 : KW >= 8 ? 2 : 4;  // 16-token tiles of a step
    static constexpr int TOKENS = 16 * U;
    static constexpr int KS = D / 16;                         // products over the channels; tiles of 16 channels of the output
    static constexpr int WARPS = NT == 1 ? 12 : 8;
    static constexpr int RECORD = 8 * NT * (D + 4);           // floats: rows of D sums, then the maximum and the sum
    static constexpr int SMEM = WARPS * 2 * RECORD * 4;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// Streamed once: past L1.
__device__ __forceinline__ uint4 stream16(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 stream8(const uint8_t* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t stream4(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];\n" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load4(const void* p) {
    uint32_t v;
    asm volatile("ld.global.nc.u32 %0, [%1];\n" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load2(const void* p) {
    uint16_t v;
    asm volatile("ld.global.nc.u16 %0, [%1];\n" : "=h"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load1(const void* p) {
    uint32_t v;
    asm volatile("ld.global.nc.u8 %0, [%1];\n" : "=r"(v) : "l"(p));
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
__device__ __forceinline__ int exponent_byte(uint32_t word, int i) { return (int)(int8_t)((word >> (8 * i)) & 0xFFu); }

// ---------------------------------------------------------------- which chunks are whose
// cum[b]: chunks of one unit of the sequences before b; a sequence without tokens has one, so that its rows are written.
__device__ __forceinline__ int chunks_of(int n) { return max(1, (n + CHUNK - 1) / CHUNK); }

template <int THREADS>
__device__ __forceinline__ void add_lengths(const AttendArgs& a, int* cum, int* sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int before = 0;
    for (int b0 = 0; b0 < a.B; b0 += THREADS) {
        const int b = b0 + tid;
        int x = b < a.B ? chunks_of(length_of(a.pool, b)) : 0;
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
struct Deal {
    int total, per_cta, runs;       // chunks in all; warps of a CTA that get a run, runs in all
    __device__ __forceinline__ Deal(int chunks, int ctas, int warps) {
        total = chunks;
        per_cta = min(warps, (total + ctas - 1) / ctas);
        runs = per_cta * ctas;
    }
    // First chunk of run w; of run w + 1: its end.
    __device__ __forceinline__ int start(int w) const {
        const int each = (unsigned)total / (unsigned)runs;
        return w * each + min(w, total - each * runs);
    }
};
// A run's part of one unit.
struct Part {
    int b, unit, first, last, chunks;   // sequence; unit of all; chunks of the unit: [first, last) of `chunks`
    // The part that begins with chunk `at`, of a run that ends with `end`; b: where to begin looking.
    __device__ __forceinline__ void find(const int* cum, int units, int b0, int at, int end) {
        b = b0;
        while (at >= cum[b + 1] * units) ++b;
        chunks = cum[b + 1] - cum[b];
        const int rest = at - cum[b] * units, u = (unsigned)rest / (unsigned)chunks;
        unit = b * units + u;
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

// Row of q, out and lse [B,T,H*G] that row r of a unit stands for; -1 behind the last.
__device__ __forceinline__ long long row_of(const AttendArgs& a, int unit, int r, int* query) {
    const int group = unit % a.groups, bh = unit / a.groups, h = bh % a.pool.H, b = bh / a.pool.H, R = group * a.rows + r;
    const int t = (unsigned)R / (unsigned)a.G;
    *query = t;
    if (r >= a.rows || t >= a.T) return -1;
    return ((long long)b * a.T + t) * (a.pool.H * a.G) + h * a.G + R - t * a.G;
}

// ---------------------------------------------------------------- a warp's run
// ONE: a step's tokens are in one page.
template <int F, int D, int NT, bool ONE>
struct Run {
    using S = Shape<F, D, NT>;
    static constexpr int U = S::U, KW = S::KW, KS = S::KS, PAGES = ONE ? 1 : U;
    const AttendArgs& a;
    int g, t;
    uint32_t q[KS][NT][2];
    float acc[KS][NT][4], m[NT][2], l[NT][2];
    uint32_t k[U][KW], v[U][KW], ke[U], ve[U], ks[U][2], vs[U][4];

    __device__ __forceinline__ Run(const AttendArgs& args, int lane) : a(args), g(lane >> 2), t(lane & 3) {}

    // Token of k index i of a tile's row: rows g and g + 8 of K, k = 2t, 2t + 1, 2t + 8, 2t + 9 of V: a lane's four of V lie side by side.
    __device__ __forceinline__ int k_token(int half) const { return 4 * (g >> 1) + (g & 1) + 2 * half; }

    // Channels of the first operand's k = 2t, 2t + 1, 2t + 8, 2t + 9 in product s: this one and the next three.
    __device__ __forceinline__ int k_channel(int s) const {
        if constexpr (F == AKV_PAGE_FP16) return (s >> 1) * 32 + t * 8 + (s & 1) * 4;
        else if constexpr (F == AKV_PAGE_E4M3) return (s >> 2) * 64 + t * 16 + (s & 3) * 4;
        else return t * (D / 4) + s * 4;
    }
    // Channel of rows g (half 0) and g + 8 (half 1) of output tile i.
    __device__ __forceinline__ int v_channel(int i, int half) const {
        if constexpr (F == AKV_PAGE_FP16) return (i >> 2) * 64 + g * 8 + (i & 3) * 2 + half;
        else if constexpr (F == AKV_PAGE_E4M3) return g * (D / 8) + 2 * i + half;
        // (8 channels of a word: even ones of the two halves first)
        else return g * (D / 8) + (i >> 2) * 8 + 2 * (i & 3) + half;
    }

    __device__ __forceinline__ void begin(int unit) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            int query;
            const long long row = row_of(a, unit, 8 * nt + g, &query);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                uint2 w = make_uint2(0, 0);
                if (row >= 0) w = *reinterpret_cast<const uint2*>(a.q + row * D + k_channel(s));
                q[s][nt][0] = w.x;
                q[s][nt][1] = w.y;
            }
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < KS; ++i) acc[i][nt][0] = acc[i][nt][1] = acc[i][nt][2] = acc[i][nt][3] = 0.f;
        }
    }

    // Pages of a step's tiles; -1 where there is none or nothing of the sequence in it.
    __device__ __forceinline__ void look(int (&page)[PAGES], int b, int at, int n) const {
#pragma unroll
        for (int u = 0; u < PAGES; ++u) {
            page[u] = -1;
            if (at + 16 * u < n) {
                const int x = __ldg(a.pool.table + (unsigned)b * (unsigned)a.pool.width + ((at + 16 * u) >> a.pool.shift));
                if ((unsigned)x < (unsigned)a.pool.n_pages) page[u] = x;
            }
        }
    }
    static __device__ __forceinline__ bool missing(const int (&page)[PAGES], int u) { return page[ONE ? 0 : u] < 0; }
    // First row of the pool of a tile (of some page where there is none: what is read from it is not used).
    __device__ __forceinline__ unsigned tile_row(const int (&page)[PAGES], int u, int h, int at) const {
        const int from = ONE ? at : at + 16 * u;
        return (((unsigned)max(page[ONE ? 0 : u], 0) * (unsigned)a.pool.H + h) << a.pool.shift) + (from & ((1 << a.pool.shift) - 1)) + (ONE ? 16 * u : 0);
    }
    // (Addresses are a tensor's, the step's row's and the lane's; tiles and tokens are constants behind them.)
    static __device__ __forceinline__ const uint8_t* place(const void* base, unsigned row, int size, int mine) {
        return static_cast<const uint8_t*>(base) + (unsigned long long)row * size + mine;
    }
    __device__ __forceinline__ void load_k(const int (&page)[PAGES], int h, int at) {
        constexpr int PIECE = S::ROW >= 64 ? 16 : 8;
        const uint8_t *p = nullptr, *pe = nullptr, *pv = nullptr, *ps = nullptr;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!ONE || u == 0) {
                const unsigned row = tile_row(page, u, h, at);
                p = place(a.pool.kc, row, S::ROW, k_token(0) * S::ROW + t * PIECE);
                if constexpr (F != AKV_PAGE_FP16) {
                    pe = place(a.pool.ke, row, 1, 4 * (g >> 1));
                    pv = place(a.pool.ve, row, 1, 4 * (g >> 1));
                }
                if constexpr (F == AKV_PAGE_E2M1) ps = place(a.pool.ks, row, D / 16, k_token(0) * (D / 16) + t * (D / 64));
            }
            const int tile = ONE ? 16 * u : 0;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint8_t* x = p + (tile + 2 * half) * S::ROW;
                if constexpr (S::ROW >= 64) {
#pragma unroll
                    for (int c = 0; c < S::ROW / 64; ++c) {
                        const uint4 w = stream16(x + c * 64);
#pragma unroll
                        for (int i = 0; i < 4; ++i) k[u][half * (KW / 2) + 4 * c + i] = u4w(w, i);
                    }
                } else {
                    const uint2 w = stream8(x);
                    k[u][half * 2] = w.x;
                    k[u][half * 2 + 1] = w.y;
                }
                if constexpr (F == AKV_PAGE_E2M1) {
                    const uint8_t* y = ps + (tile + 2 * half) * (D / 16);
                    ks[u][half] = D == 128 ? load2(y) : load1(y);
                }
            }
            if constexpr (F != AKV_PAGE_FP16) {
                ke[u] = load4(pe + tile);
                ve[u] = load4(pv + tile);
            }
        }
    }
    __device__ __forceinline__ void load_v(const int (&page)[PAGES], int h, int at) {
        constexpr int PIECE = S::ROW >= 128 ? 16 : S::ROW / 8;
        const uint8_t *p = nullptr, *ps = nullptr;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!ONE || u == 0) {
                const unsigned row = tile_row(page, u, h, at);
                p = place(a.pool.vc, row, S::ROW, 4 * t * S::ROW + g * PIECE);
                if constexpr (F == AKV_PAGE_E2M1) ps = place(a.pool.vs, row, D / 16, 4 * t * (D / 16) + (D == 128 ? g : g >> 1));
            }
            const int tile = ONE ? 16 * u : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t* x = p + (tile + i) * S::ROW;
                if constexpr (S::ROW >= 128) {
#pragma unroll
                    for (int c = 0; c < S::ROW / 128; ++c) {
                        const uint4 w = stream16(x + c * 128);
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[u][i * (KW / 4) + 4 * c + j] = u4w(w, j);
                    }
                } else if constexpr (S::ROW == 64) {
                    const uint2 w = stream8(x);
                    v[u][i * 2] = w.x;
                    v[u][i * 2 + 1] = w.y;
                } else {
                    v[u][i] = stream4(x);
                }
                if constexpr (F == AKV_PAGE_E2M1) vs[u][i] = load1(ps + (tile + i) * (D / 16));
            }
        }
    }

    // Scores of a step's tokens, s[u][nt]: rows k_token(0) (first two) and k_token(1) by query rows 2t, 2t + 1.
    __device__ __forceinline__ void scores(float (&s)[U][NT][4]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[u][nt][0] = s[u][nt][1] = s[u][nt][2] = s[u][nt][3] = 0.f;
            constexpr int H = KW / 2;
            if constexpr (F == AKV_PAGE_FP16) {
#pragma unroll
                for (int i = 0; i < KS; ++i)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma(s[u][nt], k[u][2 * i], k[u][H + 2 * i], k[u][2 * i + 1], k[u][H + 2 * i + 1], q[i][nt][0], q[i][nt][1]);
            } else if constexpr (F == AKV_PAGE_E4M3) {
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t x[2], y[2];
                    e4m3_word(x, k[u][i]);
                    e4m3_word(y, k[u][H + i]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma(s[u][nt], x[0], y[0], x[1], y[1], q[i][nt][0], q[i][nt][1]);
                }
            } else {
                const uint32_t s0 = e4m3_halves(ks[u][0]), s1 = e4m3_halves(ks[u][1]);
#pragma unroll
                for (int w = 0; w < H; ++w) {
                    // (8 channels of a word: two products; 16 have a scale)
                    const uint32_t f0 = __byte_perm(s0, s0, D == 128 && w >= 2 ? 0x3232 : 0x1010), f1 = __byte_perm(s1, s1, D == 128 && w >= 2 ? 0x3232 : 0x1010);
                    uint32_t x[4], y[4];
                    e2m1_word(x, k[u][w]);
                    e2m1_word(y, k[u][H + w]);
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma(s[u][nt], hmul2_bits(x[2 * i], f0), hmul2_bits(y[2 * i], f1), hmul2_bits(x[2 * i + 1], f0), hmul2_bits(y[2 * i + 1], f1),
                                q[2 * w + i][nt][0], q[2 * w + i][nt][1]);
                }
            }
        }
    }

    // Scores to weights of the values, in place, and the running maximum and sum with them.  seen(nt, c): tokens below it are seen by the row; page:
    // -1 where the tile's tokens are not there.  ALL: every row sees the whole step.  (An exponent of -128 comes out as a factor of
    // -infinity: times the row's zeros NaN, as it should.)
    template <bool ALL>
    __device__ __forceinline__ void soften(float (&s)[U][NT][4], const uint32_t (&ke)[U], const uint32_t (&ve)[U], const int (&page)[PAGES], int at,
                                           const int (&seen)[NT][2]) {
        float top[NT][2], f[U][2], unit[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float e = 0.f;
                f[u][half] = a.scale2;
                unit[u][half] = LIFT;
                if constexpr (F != AKV_PAGE_FP16) {
                    const int i = (g & 1) + 2 * half, x = exponent_byte(ve[u], i);
                    f[u][half] = a.scale2 * __int_as_float((exponent_byte(ke[u], i) + 127) << 23);
                    unit[u][half] = __int_as_float((x + 127 + 15) << 23);
                    if (x == EXP_NAN) unit[u][half] = NAN;
                    e = (float)max(x, -40);           // (a row of NaN has no exponent; -35 is the least there is)
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float& x = s[u][nt][2 * half + c];
                        if (!ALL) {
                            x *= f[u][half];
                            if (missing(page, u) || at + 16 * u + k_token(half) >= seen[nt][c]) x = -INFINITY;
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
                        const bool gone = !ALL && (missing(page, u) || at + 16 * u + k_token(half) >= seen[nt][c]);
                        const float p = ex2(ALL ? fmaf(x, f[u][half], -base) : x - base);
                        l[nt][c] += p;                              // (of what is not seen: 0)
                        x = gone ? 0.f : p * unit[u][half];
                    }
            }
    }

    // Values of a step that lie behind the sequence, or nowhere: zeros, whatever is there.
    __device__ __forceinline__ void clear_v(const int (&page)[PAGES], int at, int n) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (missing(page, u) || at + 16 * u + 4 * t + i >= n) {
#pragma unroll
                    for (int j = 0; j < KW / 4; ++j) v[u][i * (KW / 4) + j] = 0;
                    if constexpr (F == AKV_PAGE_E2M1) vs[u][i] = 0;
                }
    }

    // fn(i, a0, a1, a2, a3): the first operand of output tile i, of the values of tile u.
    template <class Fn>
    __device__ __forceinline__ void tiles(int u, Fn fn) {
        constexpr int W = KW / 4;              // words of a token
        if constexpr (F == AKV_PAGE_FP16) {
#pragma unroll
            for (int i = 0; i < KS; ++i)
                fn(i, __byte_perm(v[u][i], v[u][W + i], 0x5410), __byte_perm(v[u][i], v[u][W + i], 0x7632),
                   __byte_perm(v[u][2 * W + i], v[u][3 * W + i], 0x5410), __byte_perm(v[u][2 * W + i], v[u][3 * W + i], 0x7632));
        } else if constexpr (F == AKV_PAGE_E4M3) {
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint32_t x = __byte_perm(v[u][i >> 1], v[u][W + (i >> 1)], i & 1 ? 0x7362 : 0x5140);
                const uint32_t y = __byte_perm(v[u][2 * W + (i >> 1)], v[u][3 * W + (i >> 1)], i & 1 ? 0x7362 : 0x5140);
                uint32_t p[2], r[2];
                e4m3_word(p, x);
                e4m3_word(r, y);
                fn(i, p[0], p[1], r[0], r[1]);
            }
        } else {
            const uint32_t s0 = e4m3_halves(__byte_perm(vs[u][0], vs[u][1], 0x0040)), s1 = e4m3_halves(__byte_perm(vs[u][2], vs[u][3], 0x0040));
#pragma unroll
            for (int w = 0; w < W; ++w) {
                constexpr uint32_t LOW = 0x0F0F0F0Fu;
                // two tokens' nibbles of one channel in a byte: even channels, odd ones
                const uint32_t e0 = (v[u][w] & LOW) | ((v[u][W + w] << 4) & ~LOW), o0 = ((v[u][w] >> 4) & LOW) | (v[u][W + w] & ~LOW);
                const uint32_t e1 = (v[u][2 * W + w] & LOW) | ((v[u][3 * W + w] << 4) & ~LOW), o1 = ((v[u][2 * W + w] >> 4) & LOW) | (v[u][3 * W + w] & ~LOW);
                uint32_t x0[4], y0[4], x1[4], y1[4];
                e2m1_word(x0, e0);
                e2m1_word(y0, o0);
                e2m1_word(x1, e1);
                e2m1_word(y1, o1);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    fn(4 * w + i, hmul2_bits(x0[i], s0), hmul2_bits(y0[i], s0), hmul2_bits(x1[i], s1), hmul2_bits(y1[i], s1));
            }
        }
    }
    __device__ __forceinline__ void add_values(const float (&s)[U][NT][4]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint32_t hi[NT][2], lo[NT][2];
            second_operand(s[u], hi, lo);
            tiles(u, [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma(acc[i][nt], a0, a1, a2, a3, hi[nt][0], hi[nt][1]);
                    mma(acc[i][nt], a0, a1, a2, a3, lo[nt][0], lo[nt][1]);
                }
            });
        }
    }
    __device__ __forceinline__ void second_operand(const float (&s)[NT][4], uint32_t (&hi)[NT][2], uint32_t (&lo)[NT][2]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float x = s[nt][2 * half], y = s[nt][2 * half + 1];
                const uint32_t h = halves_bits(x, y);
                const float2 back = halves_floats(h);
                hi[nt][half] = transposed(h);
                lo[nt][half] = transposed(halves_bits(x - back.x, y - back.y));
            }
    }
    // The same where some values are not finite (fp16 pages alone: elsewhere codes are).  0 * inf would be NaN: every query's product is formed by
    // itself, without the newest tokens that it does not see, and the second halves' without what is not finite.
    __device__ __forceinline__ void add_odd_values(const float (&s)[U][NT][4], int at, int n, const int (&seen)[NT][2]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint32_t hi[NT][2], lo[NT][2];
            second_operand(s[u], hi, lo);
#pragma unroll 1
            for (int limit = n - a.T + 1; limit <= n; ++limit) {
                bool there[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) there[i] = at + 16 * u + 4 * t + i < limit;
                const uint32_t m01 = (there[0] ? 0xFFFFu : 0u) | (there[1] ? 0xFFFF0000u : 0u), m23 = (there[2] ? 0xFFFFu : 0u) | (there[3] ? 0xFFFF0000u : 0u);
                tiles(u, [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float c[4] = {0.f, 0.f, 0.f, 0.f};
                        mma(c, a0 & m01, a1 & m01, a2 & m23, a3 & m23, hi[nt][0], hi[nt][1]);
                        mma(c, finite(a0 & m01), finite(a1 & m01), finite(a2 & m23), finite(a3 & m23), lo[nt][0], lo[nt][1]);
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            if (seen[nt][x & 1] == limit) acc[i][nt][x] += c[x];
                    }
                });
            }
        }
    }
    static __device__ __forceinline__ uint32_t finite(uint32_t w) {
        if ((w & 0x7C00u) == 0x7C00u) w &= 0xFFFF0000u;
        return (w & 0x7C000000u) == 0x7C000000u ? w & 0xFFFFu : w;
    }
    __device__ __forceinline__ bool odd_values() const {
        uint32_t x[2] = {0, 0};                  // (0 as long as all are finite, then NaN)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < KW; ++i) x[i & 1] = hfma2_bits(v[u][i], 0, x[i & 1]);
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
    }
    __device__ __forceinline__ void write(int unit) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                int query;
                const long long row = row_of(a, unit, 8 * nt + 2 * t + c, &query);
                if (row < 0) continue;
                const float inv = l[nt][c] == 0.f ? 0.f : 1.f / (l[nt][c] * LIFT);
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const __half2 h = __floats2half2_rn(acc[i][nt][c] * inv, acc[i][nt][2 + c] * inv);
                    *reinterpret_cast<__half2*>(a.out + row * D + v_channel(i, 0)) = h;
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
                float* row = to + (8 * nt + 2 * t + c) * (D + 4);
#pragma unroll
                for (int i = 0; i < KS; ++i)
                    *reinterpret_cast<float2*>(row + v_channel(i, 0)) = make_float2(acc[i][nt][c], acc[i][nt][2 + c]);
                if (g == 0) *reinterpret_cast<float2*>(row + D) = make_float2(m[nt][c], l[nt][c]);
            }
    }
};

// Joins rows of `count` records (lane: D / 32 channels): fn(i) = row of the i-th.  Then to a record, or to out and lse.
template <int D, class Fn>
__device__ __forceinline__ void join_row(const AttendArgs& a, int unit, int r, int count, int lane, Fn fn, float* record) {
    constexpr int N = D / 32;
    float top = -INFINITY;
    for (int i = 0; i < count; ++i) top = fmaxf(top, fn(i)[D]);
    const float base = top == -INFINITY ? 0.f : top;
    float o[N], sum = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) o[c] = 0.f;
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
        const float* x = fn(i);
        const float f = ex2(x[D] - base);
        sum = fmaf(f, x[D + 1], sum);
#pragma unroll
        for (int c = 0; c < N; ++c) o[c] = fmaf(f, x[N * lane + c], o[c]);
    }
    if (record) {
#pragma unroll
        for (int c = 0; c < N; ++c) record[N * lane + c] = o[c];
        if (lane == 0) {
            record[D] = top;
            record[D + 1] = sum;
        }
        return;
    }
    int query;
    const long long row = row_of(a, unit, r, &query);
    if (row < 0) return;
    const float inv = sum == 0.f ? 0.f : 1.f / (sum * LIFT);
#pragma unroll
    for (int c = 0; c < N; c += 2)
        *reinterpret_cast<__half2*>(a.out + row * D + N * lane + c) = __floats2half2_rn(o[c] * inv, o[c + 1] * inv);
    if (a.lse && lane == 0) a.lse[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * LN2;
}

template <int F, int D, int NT, bool ONE>
__global__ void __launch_bounds__(32 * Shape<F, D, NT>::WARPS, 1) attend_kernel(AttendArgs a) {
    using S = Shape<F, D, NT>;
    constexpr int WARPS = S::WARPS, U = S::U, PAGES = ONE ? 1 : U;
    extern __shared__ __align__(16) float records[];           // [warp][2][rows][D + 4]: of a run's first part and of its last
    int* cum = reinterpret_cast<int*>(records + WARPS * 2 * S::RECORD);
    __shared__ int sums[WARPS], s_unit[2 * WARPS];             // (s_unit: unit of each record, -1 where there is none)
    pdl_turn();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    add_lengths<32 * WARPS>(a, cum, sums);
    const int units = a.pool.H * a.groups;
    const Deal deal(cum[a.B] * units, gridDim.x, WARPS);
    const int me = blockIdx.x * deal.per_cta + warp;
    int at = 0, end = 0;
    if (warp < deal.per_cta) {
        at = deal.start(me);
        end = deal.start(me + 1);
    }
    if (lane < 2) s_unit[2 * warp + lane] = -1;
    __syncwarp();
    if (at < end) {
        Run<F, D, NT, ONE> run(a, lane);
        Part part;
        part.find(cum, units, sequence_with(cum, a.B, units, at), at, end);
        int n = length_of(a.pool, part.b), h = part.unit / a.groups % a.pool.H;
        int token = part.first * CHUNK, stop = min(n, part.last * CHUNK), page[PAGES];
        run.look(page, part.b, token, n);
        run.load_k(page, h, token);
        run.load_v(page, h, token);
        int seen[NT][2];
        bool fresh = true;
        for (;;) {
            if (fresh) {
                run.begin(part.unit);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        int query;
                        seen[nt][c] = row_of(a, part.unit, 8 * nt + 2 * run.t + c, &query) < 0 ? 0 : n - a.T + 1 + query;
                    }
            }
            // the step behind this one: the unit's next, or the first of the next unit
            const Part was = part;
            const int was_token = token, was_n = n;
            int was_page[PAGES];
#pragma unroll
            for (int u = 0; u < PAGES; ++u) was_page[u] = page[u];
            token += S::TOKENS;
            fresh = token >= stop;
            if (fresh) {
                at += part.last - part.first;
                if (at < end) {
                    part.find(cum, units, part.b, at, end);
                    n = length_of(a.pool, part.b);
                    h = part.unit / a.groups % a.pool.H;
                    token = part.first * CHUNK;
                    stop = min(n, part.last * CHUNK);
                }
            }
            const bool more = !fresh || at < end;
            if (more) run.look(page, part.b, token, n);
            float s[U][NT][4];
            run.scores(s);
            uint32_t ke[U], ve[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                ke[u] = run.ke[u];
                ve[u] = run.ve[u];
            }
            if (more) run.load_k(page, h, token);
            bool all = was_token + S::TOKENS <= was_n - a.T + 1;
#pragma unroll
            for (int u = 0; u < PAGES; ++u) all = all && was_page[u] >= 0;
            if (all) {
                run.template soften<true>(s, ke, ve, was_page, was_token, seen);
            } else {
                run.template soften<false>(s, ke, ve, was_page, was_token, seen);
                run.clear_v(was_page, was_token, was_n);
            }
            if (F == AKV_PAGE_FP16 && __any_sync(0xFFFFFFFFu, run.odd_values())) run.add_odd_values(s, was_token, was_n, seen);
            else run.add_values(s);
            if (more) run.load_v(page, h, token);
            if (fresh) {
                run.close();
                if (was.whole()) {
                    run.write(was.unit);
                } else {
                    const int slot = 2 * warp + (was.first == 0);   // (a run has one part that begins in front of it, at most)
                    run.record(records + slot * S::RECORD);
                    if (lane == 0) s_unit[slot] = was.unit;
                }
                if (!more) break;
            }
        }
    }
    __syncthreads();
    // Records of one unit lie in a row (slots without one aside).  A unit that begins and ends in this CTA is written, of another one
    // record is left: slot 0 of the CTA's two where it began in front of it.
    const int begin = deal.start(blockIdx.x * deal.per_cta), finish = deal.start((blockIdx.x + 1) * deal.per_cta);
    int groups = 0;
    for (int i = 0; i < 2 * WARPS;) {
        const int unit = s_unit[i];
        if (unit < 0) {
            ++i;
            continue;
        }
        int j = i, count = 0;
        while (j < 2 * WARPS && (s_unit[j] == unit || s_unit[j] < 0)) count += s_unit[j++] == unit;
        const int b = unit / units, chunks = cum[b + 1] - cum[b], from = cum[b] * units + (unit - b * units) * chunks;
        const bool before = from < begin, whole = !before && from + chunks <= finish;
        for (int r = 0; r < 8 * NT; ++r) {
            if ((groups + r) % WARPS != warp) continue;
            int list = 0;               // bits: the unit's slots
            for (int x = i; x < j; ++x) list |= (s_unit[x] == unit) << x;
            float* record = whole ? nullptr : a.part + ((long long)(2 * blockIdx.x + !before) * 8 * NT + r) * (D + 4);
            join_row<D>(a, unit, r, count, lane, [&](int x) { return records + __fns(list, 0, x + 1) * S::RECORD + r * (D + 4); }, record);
        }
        groups += 8 * NT;
        i = j;
    }
}

// One CTA per border between two CTAs of attend_kernel: the first inside a unit joins its records.
template <int D, int NT, int WARPS>
__global__ void __launch_bounds__(256) join_kernel(AttendArgs a, int ctas) {
    extern __shared__ int cum[];
    __shared__ int sums[8];
    // (what this kernel follows waited for everything in front of it: lens may be read)
    add_lengths<256>(a, cum, sums);
    const int units = a.pool.H * a.groups, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Deal deal(cum[a.B] * units, ctas, WARPS);
    const int border = blockIdx.x + 1, at = deal.start(border * deal.per_cta);
    pdl_turn();
    if (at >= deal.total) return;
    const int b = sequence_with(cum, a.B, units, at), chunks = cum[b + 1] - cum[b], u = (at - cum[b] * units) / chunks;
    const int unit = b * units + u, from = cum[b] * units + u * chunks;
    if (from == at || from < deal.start((border - 1) * deal.per_cta)) return;
    int last = border;              // CTA with the unit's end
    while (deal.start((last + 1) * deal.per_cta) < from + chunks) ++last;
    for (int r = warp; r < 8 * NT; r += 8)
        join_row<D>(a, unit, r, last - border + 2, lane, [&](int i) {
            return a.part + ((long long)(2 * (border - 1 + i) + (i == 0)) * 8 * NT + r) * (D + 4);
        }, nullptr);
}

struct Plan {
    int nt, groups, rows, ctas;
    long long bytes;
};
Plan plan_of(int rows, int D) {
    Plan p;
    p.nt = rows <= 8 ? 1 : 2;
    p.groups = (rows + 15) / 16;
    p.rows = (rows + p.groups - 1) / p.groups;
    p.ctas = sm_count();
    p.bytes = 2ll * p.ctas * 8 * p.nt * (D + 4) * 4;
    return p;
}

template <int F, int D, int NT, bool ONE>
int launch(const AttendArgs& a, const Plan& p, bool joined, cudaStream_t st) {
    using S = Shape<F, D, NT>;
    const int smem = S::SMEM + (a.B + 1) * 4;
    static thread_local int set_for = -1;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && set_for != dev) {
        // (the most it is ever launched with)
        e = cudaFuncSetAttribute(attend_kernel<F, D, NT, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM + 4097 * 4);
        if (e == cudaSuccess) set_for = dev;
    }
    if (e != cudaSuccess) return cuda_status(e, "paged_attention");
    launch_chained(attend_kernel<F, D, NT, ONE>, dim3(p.ctas), dim3(32 * S::WARPS), smem, st, a);
    const int rc = cuda_status(cudaGetLastError(), "paged_attention launch");
    if (rc != AKV_OK || !joined || p.ctas == 1) return rc;
    launch_chained(join_kernel<D, NT, S::WARPS>, dim3(p.ctas - 1), dim3(256), (a.B + 1) * 4, st, a, p.ctas);
    return cuda_status(cudaGetLastError(), "paged_attention join launch");
}
template <int F, int D, int NT>
int launch_pages(const AttendArgs& a, const Plan& p, bool joined, cudaStream_t st) {
    if constexpr (Shape<F, D, NT>::U > 1)
        if (Shape<F, D, NT>::TOKENS > 1 << a.pool.shift) return launch<F, D, NT, false>(a, p, joined, st);
    return launch<F, D, NT, true>(a, p, joined, st);
}
template <int F>
int launch_format(const AttendArgs& a, const Plan& p, int D, bool joined, cudaStream_t st) {
    if (D == 128) return p.nt == 1 ? launch_pages<F, 128, 1>(a, p, joined, st) : launch_pages<F, 128, 2>(a, p, joined, st);
    return p.nt == 1 ? launch_pages<F, 64, 1>(a, p, joined, st) : launch_pages<F, 64, 2>(a, p, joined, st);
}

}  // namespace
}  // namespace akv

using namespace akv;

extern "C" {

long long akv_paged_scratch_bytes(const akv_pool* pool, int bsz, int width, int group, int tokens) {
    if (!pool || bsz <= 0 || width <= 0 || group <= 0 || tokens <= 0 || group > 64 || tokens > 64 || group * tokens > 64 ||
        (pool->head_dim != 64 && pool->head_dim != 128))
        return -1;
    return plan_of(group * tokens, pool->head_dim).bytes;
}

int akv_paged_attention(const akv_pool* pool, const void* q, const void* pages, const void* lens, void* out, void* lse, void* scratch,
                        long long scratch_bytes, int bsz, int width, int group, int tokens, float scale, void* stream) {
    set_error("");
    AttendArgs a = {};
    int rc = fill_pool("paged_attention", pool, pages, lens, bsz, width, &a.pool);
    if (rc != AKV_OK) return rc;
    AKV_REQUIRE(q && out && scratch, AKV_ERR_NULL, "paged_attention: null pointer");
    AKV_REQUIRE(group > 0 && tokens > 0 && group <= 64 && tokens <= 64 && group * tokens <= 64, AKV_ERR_SHAPE,
                "paged_attention: %d new tokens of %d query heads per KV head (at most 64 rows)", tokens, group);
    AKV_REQUIRE(aligned16(q) && aligned16(out) && aligned16(scratch) && (reinterpret_cast<uintptr_t>(lse) & 3u) == 0, AKV_ERR_ALIGN,
                "paged_attention: q, out and scratch must be 16-byte aligned, lse 4-byte");
    const int D = pool->head_dim;
    const Plan p = plan_of(group * tokens, D);
    AKV_REQUIRE(scratch_bytes >= p.bytes, AKV_ERR_SHAPE, "paged_attention: scratch of %lld bytes is too small", scratch_bytes);
    AKV_REQUIRE((long long)pool->n_pages * pool->n_kv_heads * pool->page_size <= 1ll << 32 && (long long)bsz * width < INT_MAX, AKV_ERR_OVERFLOW,
                "paged_attention: a pool of more than 2^32 rows");
    const long long most = ((long long)width * pool->page_size + CHUNK - 1) / CHUNK * bsz * pool->n_kv_heads * p.groups;
    AKV_REQUIRE(most < INT_MAX, AKV_ERR_OVERFLOW, "paged_attention: too many chunks of %d tokens", CHUNK);
    a.q = static_cast<const __half*>(q);
    a.out = static_cast<__half*>(out);
    a.lse = static_cast<float*>(lse);
    a.part = static_cast<float*>(scratch);
    a.B = bsz;
    a.T = tokens;
    a.G = group;
    a.groups = p.groups;
    a.rows = p.rows;
    a.scale2 = scale * LOG2E;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool joined = (long long)width * pool->page_size > CHUNK;      // (units of one chunk are nobody else's)
    if (pool->format == AKV_PAGE_FP16) return launch_format<AKV_PAGE_FP16>(a, p, D, joined, st);
    if (pool->format == AKV_PAGE_E4M3) return launch_format<AKV_PAGE_E4M3>(a, p, D, joined, st);
    return launch_format<AKV_PAGE_E2M1>(a, p, D, joined, st);
}

}  // extern "C"
