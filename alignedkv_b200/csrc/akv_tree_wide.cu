// Attention of drafted tokens where more than 16 query rows share a KV head: the fifth-generation tensor cores.
//
// CTA = one SM, a contiguous run of 128-token tiles as in akv_tree.cu; a unit is up to 256 query rows of a (batch, KV head).
//   warp  17      copies the planes of a tile (K or V: 32 KB at head size 128) into a ring, three bulk copies for 64 tokens
//   warps 8..15   decode: four warps for 64 tokens' bytes, to fp16 operands in the same place - they take as much - by way of registers
//   warp  16      issues the products: S = Q K^T (128 rows x 128 tokens), O += P V
//   warps 0..7    two softmax groups of 128 threads, a thread per query row: S from tensor memory, P back into its place
// Everything comes in twos: S, O, P and a softmax group per slot.  With up to 128 rows the slots take the tiles in turn (each
// with an output of its own, joined at the end), with more (a slot has no more) each has half of the rows and takes every tile.  While
// one slot's softmax runs, the other's products do.
// K planes run along tokens and V planes along channels - along the n of either product, not along its sum: the operand tiles
// are "MN-major", rows of 64 elements (128 bytes), so that a decoded piece of 16 elements is two 16-byte stores.  Only the
// tail's keys (fp16 rows of channels) are K-major.
// Tensor memory: columns 0..255 S (P in the same columns as fp16), 256..511 O.
// What bounds it: up to 128 rows the planes' way into the operands (16 x 8 x 8190 tokens, 48 rows: 130 us; the copies alone took 90
// when the whole took 125, HBM's floor is 83: decode, products and softmax share the SM's shared memory with them); 256 rows (4 x 8 x
// 8192: 69 us) the chain of a slot - when they took 66: 1.3 us of softmax, bound by exponentials, and 1.1 us from P to the next S - and
// 25 us of a call's start, of the records and of the merge.
#include <limits.h>

#include "akv_tree.cuh"

namespace akv {

__device__ unsigned int g_tree_wait_gave_up = 0;     // set when a bounded wait ran out (never expected)
unsigned int tree_error_flag(cudaError_t* e) {
    unsigned int v = 0;
    *e = cudaMemcpyFromSymbol(&v, g_tree_wait_gave_up, sizeof(v));
    return v;
}
cudaError_t tree_error_clear() {
    const unsigned int v = 0;
    return cudaMemcpyToSymbol(g_tree_wait_gave_up, &v, sizeof(v));
}

namespace {

constexpr int SOFT = 8, DECODE = 8, THREADS = 32 * (SOFT + DECODE + 2);
// A row's reference maximum moves only when a score exceeds it by 2^SLACK: probabilities are at most 2^(WIDE_LIFT + SLACK) in fp16.
// (The largest is then rounded like the others; with the reference always at the maximum it would be a power of two, and outputs that two
// tokens share a little nearer - and the outputs so far would be read and scaled again in most tiles of a warp's 32 rows.)
constexpr float WIDE_LIFT = 7.f, SLACK = 8.f;

template <int D>
struct Plan {
    static constexpr int RING = D == 128 ? 5 : 8;
    static constexpr int TILE_BYTES = TILE * D * 2, Q_HALF = 16384, Q_BYTES = Q_HALF * (D / 64);
    // Two places for queries: of the two row groups, or of one group and, with one group, of the segment behind.  With one group the
    // slots' outputs are joined (128 rows x 64 channels at a time) where the queries of the segment that ends were.
    static constexpr int JOIN_BYTES = 128 * 64 * 4, Q_PLACE = Q_BYTES > JOIN_BYTES ? Q_BYTES : JOIN_BYTES;
    static constexpr int RING_AT = 0, Q_AT = RING * TILE_BYTES, Q2_AT = Q_AT + Q_PLACE;
    static constexpr int XM_AT = Q2_AT + Q_PLACE, XL_AT = XM_AT + 512, XR_AT = XL_AT + 512;
    // barriers, 8 bytes each, then the tensor memory's address, the flag that a wait gave up, odd values of the last segments
    static constexpr int BAR_AT = XR_AT + 512, RAW = 0, FULL = RING, EMPTY = 2 * RING, S_FULL = 3 * RING, P_FULL = S_FULL + 2,
                         O_FULL = P_FULL + 2, Q_FULL = O_FULL + 2, BARS = Q_FULL + 1;
    static constexpr int SEGMENTS = 8, BYTES = BAR_AT + 8 * BARS + 8 + 4 * SEGMENTS + 1024;      // (1024: the base is aligned up)
};
static_assert(Plan<128>::BYTES <= 232448 && Plan<64>::BYTES <= 232448, "shared memory of a block");

__device__ __forceinline__ void bar_init(uint32_t a, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(a), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t a) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(a) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t a, uint32_t parity) {
    uint32_t ok;
    // (a waiting thread sleeps: polls of its own would take issue slots from those that work, 66 us against 64 at 256 rows x 8192 tokens)
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(a), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded (about a second); once one has given up, none waits any more and the outputs become NaN.
__device__ __noinline__ void bar_wait_slow(uint32_t a, uint32_t parity, volatile int* dead) {
    unsigned long long t0 = 0;
    for (unsigned spin = 0; !bar_try(a, parity); ++spin) {
        if (*dead) return;
        if ((spin & 63) == 63) {
            unsigned long long t;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
            if (t0 == 0) t0 = t;
            else if (t - t0 > 1000000000ull) {
                *dead = 1;
                atomicOr(&g_tree_wait_gave_up, 8u);
                return;
            }
        }
    }
}
__device__ __forceinline__ void bar_wait(uint32_t a, uint32_t parity, volatile int* dead) {
    if (__builtin_expect(!bar_try(a, parity), 0)) bar_wait_slow(a, parity, dead);
}

__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_shared() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
// Shared-memory operand with 128-byte swizzle, as the two words of its descriptor: the upper is the same for all (groups of eight - rows
// if K-major, of the sum's indices if MN-major - lie 1024 bytes apart), the lower has the address and, MN-major, `lead`: the bytes
// between pieces of 64 elements.
constexpr uint32_t OPERAND_HI = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t operand(uint32_t at, uint32_t lead) { return at >> 4 | (lead >> 4) << 16; }
// True in one lane of a whole warp, in a form in which the compiler still knows the warp to be whole.
__device__ __forceinline__ bool elect() {
    uint32_t x;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(x));
    return x != 0;
}
// D (fp32, tensor memory) = A B (+ D): A, B fp16 in shared memory, or A in tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 x, y;\nmov.b64 x, {%1, %5};\nmov.b64 y, {%2, %5};\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(OPERAND_HI) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\n.reg .b64 y;\nmov.b64 y, {%2, %5};\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(OPERAND_HI) : "memory");
}
// fp16 x fp16 -> fp32, 128 rows, n columns; K-major, or MN-major if so.
__device__ __forceinline__ constexpr uint32_t instruction(int n, bool b_mn, bool a_mn = false) {
    return 1u << 4 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (128u >> 4) << 24;
}
// 32 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld(uint32_t (&v)[32], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
                 "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                   "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]),
                   "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
                   "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(at) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
}
// 16 columns from each of four places, with one wait.
__device__ __forceinline__ void tmem_ld4(uint32_t (&v)[4][16], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%64];\n"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%65];\n"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47}, [%66];\n"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%67];\n"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(v[0][0]), "=r"(v[0][1]), "=r"(v[0][2]), "=r"(v[0][3]), "=r"(v[0][4]), "=r"(v[0][5]), "=r"(v[0][6]), "=r"(v[0][7]),
          "=r"(v[0][8]), "=r"(v[0][9]), "=r"(v[0][10]), "=r"(v[0][11]), "=r"(v[0][12]), "=r"(v[0][13]), "=r"(v[0][14]), "=r"(v[0][15]),
          "=r"(v[1][0]), "=r"(v[1][1]), "=r"(v[1][2]), "=r"(v[1][3]), "=r"(v[1][4]), "=r"(v[1][5]), "=r"(v[1][6]), "=r"(v[1][7]),
          "=r"(v[1][8]), "=r"(v[1][9]), "=r"(v[1][10]), "=r"(v[1][11]), "=r"(v[1][12]), "=r"(v[1][13]), "=r"(v[1][14]), "=r"(v[1][15]),
          "=r"(v[2][0]), "=r"(v[2][1]), "=r"(v[2][2]), "=r"(v[2][3]), "=r"(v[2][4]), "=r"(v[2][5]), "=r"(v[2][6]), "=r"(v[2][7]),
          "=r"(v[2][8]), "=r"(v[2][9]), "=r"(v[2][10]), "=r"(v[2][11]), "=r"(v[2][12]), "=r"(v[2][13]), "=r"(v[2][14]), "=r"(v[2][15]),
          "=r"(v[3][0]), "=r"(v[3][1]), "=r"(v[3][2]), "=r"(v[3][3]), "=r"(v[3][4]), "=r"(v[3][5]), "=r"(v[3][6]), "=r"(v[3][7]),
          "=r"(v[3][8]), "=r"(v[3][9]), "=r"(v[3][10]), "=r"(v[3][11]), "=r"(v[3][12]), "=r"(v[3][13]), "=r"(v[3][14]), "=r"(v[3][15])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t (&v)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
                 "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                   "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
                   "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]),
                   "r"(v[30]), "r"(v[31]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                   "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void soft_sync() {
    __syncwarp();
    asm volatile("bar.sync 1, %0;\n" ::"n"(32 * SOFT) : "memory");
}

__device__ __forceinline__ void bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// ---------------------------------------------------------------- the run of a CTA, piece by piece
// Segment: consecutive tiles t0 .. t0 + c - 1 of one unit.
struct Segment {
    int unit, bh, b, h, super, t0, c;
    __device__ __forceinline__ void at(const TreeArgs& p, int tile, int last) {
        unit = (unsigned)tile / (unsigned)p.tiles;
        t0 = tile - unit * p.tiles;
        c = min(p.tiles - t0, last - tile);
        bh = (unsigned)unit / (unsigned)p.rt;
        super = unit - bh * p.rt;
        b = (unsigned)bh / (unsigned)p.H;
        h = bh - b * p.H;
    }
};
// Operand tile q (0 .. 2c - 1) of a segment, in the order in which the products need them: with `ahead` scores under way,
// K(0 .. ahead - 1), then V(i), K(i + ahead).
__device__ __forceinline__ int tile_of(int q, int c, int ahead, bool& value) {
    ahead = min(ahead, c);
    if (q < ahead) {
        value = false;
        return q;
    }
    const int r = q - ahead, pairs = 2 * (c - ahead);
    value = r >= pairs || !(r & 1);
    return r >= pairs ? (c - ahead) + (r - pairs) : value ? r >> 1 : (r >> 1) + ahead;
}

// What a plane tile's mask leaves of it: a padded batch has tiles of all tokens and of none, and few others.  By a warp.
enum Masked { ALL, SOME, NONE };
__device__ __forceinline__ Masked mask_of(const __half* mask, int count, int lane) {
    bool zero = true, gone = true;
#pragma unroll
    for (int e = 0; e < TILE; e += 32) {
        if (lane + e >= count) continue;
        const uint32_t x = reinterpret_cast<const uint16_t*>(mask)[lane + e];
        zero = zero && !(x & 0x7FFFu);
        gone = gone && x == 0xFC00u;
    }
    return __all_sync(0xFFFFFFFFu, zero) ? ALL : __all_sync(0xFFFFFFFFu, gone) ? NONE : SOME;
}

// ---------------------------------------------------------------- decode
// Eight elements from their high bytes and nibbles, in the order in which two permutes a pair suffice: 0 2 1 3, 4 6 5 7.  Of K that is
// the order of the scores' columns, and V's tokens are stored in it; of V it is the order of the output's columns.
__device__ __forceinline__ constexpr int swapped(int i) { return (i & ~3) | (i & 1) << 1 | (i >> 1 & 1); }     // (its own inverse)
__device__ __forceinline__ uint4 swapped8(uint32_t h0, uint32_t h1, uint32_t m, uint32_t l) {
    const uint32_t even = (m & 0xF0F0F0F0u) | ((l >> 4) & 0x0F0F0F0Fu), odd = ((m << 4) & 0xF0F0F0F0u) | (l & 0x0F0F0F0Fu);
    return make_uint4(__byte_perm(even, h0, 0x6140), __byte_perm(odd, h0, 0x7150), __byte_perm(even, h1, 0x6342), __byte_perm(odd, h1, 0x7352));
}
// The same order for eight fp16 values.
__device__ __forceinline__ uint4 reorder8(const uint4& x) {
    return make_uint4(__byte_perm(x.x, x.y, 0x5410), __byte_perm(x.x, x.y, 0x7632), __byte_perm(x.z, x.w, 0x5410), __byte_perm(x.z, x.w, 0x7632));
}
template <class L, int D, bool KEYS>
__device__ __forceinline__ void copy_role(const TreeArgs& p, uint32_t ring_at, uint32_t ring, uint32_t bars, volatile int* dead,
                                          int first, int last, bool has_tail) {
    uint32_t buf = 0, turn = 0;
    for (int tile = first; tile < last;) {
        Segment s;
        s.at(p, tile, last);
        tile += s.c;
        for (int q = 0; q < (KEYS ? 1 : 2) * s.c; ++q) {
            bool value = false;
            const int i = s.t0 + (KEYS ? q : tile_of(q, s.c, 3 - p.groups, value));
            const uint32_t bar = bars + 8 * (L::RAW + buf);
            bar_wait(bars + 8 * (L::EMPTY + buf), (turn & 1) ^ 1, dead);
            if (has_tail && i == p.tiles - 1) {
                if (elect()) bar_arrive(bar);           // (the tail is read by the decoding warps themselves)
            } else {
                const int blocks = min(2, p.nb - 2 * i);
                const uint8_t *f = value ? p.v8 : p.k8, *m = value ? p.vm : p.km, *l = value ? p.vl : p.kl;
                const long long at = (value ? (long long)s.bh * p.L + i * TILE : ((long long)s.bh * p.nmb + 2 * i) * BLK) * D;
                const uint32_t to = ring_at + buf * L::TILE_BYTES;
                if (elect()) {
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(blocks * BLK * D * 2) : "memory");
                    bulk(to, f + at, D * BLK, bar);
                    bulk(to + D * 64, m + at / 2, D * BLK / 2, bar);
                    bulk(to + D * 96, l + at / 2, D * BLK / 2, bar);
                    if (blocks == 2) {
                        bulk(to + D * 128, f + at + D * BLK, D * BLK, bar);
                        bulk(to + D * 192, m + (at + D * BLK) / 2, D * BLK / 2, bar);
                        bulk(to + D * 224, l + (at + D * BLK) / 2, D * BLK / 2, bar);
                    }
                }
            }
            __syncwarp();
            if (++buf == ring) {
                buf = 0;
                ++turn;
            }
        }
    }
}

// A thread's share of a tile: of one region (four warps each) U = D / 32 pieces of 16 elements, quarter lane % 4 of rows of 64.  Where
// pieces lie, as bytes and as operand: e0, e1, e0 + t, e1 + t and f0, f1, f0 + 4096, f1 + 4096, whatever the tile is - K: channels k,
// 64 + k, 32 + k, 96 + k (k = 8 warp + lane / 4 of 32); V: tokens k, k, 32 + k, 32 + k and both their channel halves, of neighbouring
// lanes different ones (neither the loads of the bytes nor the stores of the operands meet in a bank); D = 64: rows k, 32 + k.
__device__ __forceinline__ void sts128(uint32_t at, const uint4& x) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
}

// The tail's share: rows of fp16 values from the residual buffers and the drafted tensors, straight to the operand.  Whether V has
// values that are not finite (zeros in the operand, see add_odd).
template <int D>
__device__ __noinline__ bool tail_share(const TreeArgs& p, int b, int h, bool value, uint32_t slot, int warp, int lane) {
    const int region = warp >> 2, k = (warp & 3) * 8 + (lane >> 2), qd = lane & 3, x = ((2 * qd) ^ (k & 7)) << 4;
    const __half *rest = value ? p.restv : p.restk, *drafted = value ? p.vd : p.kd;
    const int side = D == 128 ? (lane >> 2 ^ lane >> 3) & 1 : 0;
    auto half_of = [&](int u) { return D == 128 ? (side ^ u) & 1 : 0; };
    auto row_at = [&](int u) { return (D == 128 ? u >> 1 : u) * 32 + k; };
    uint4 v[D / 32][2];                                // (all requested before the first is used: one round trip)
#pragma unroll
    for (int u = 0; u < D / 32; ++u) {
        const int y = region * BLK + row_at(u), d = y - p.rest;
        v[u][0] = v[u][1] = make_uint4(0, 0, 0, 0);
        if (y < p.tail) {
            const __half* src = d < 0 ? rest + ((long long)(b * BLK + y) * p.H + h) * D : drafted + ((long long)(b * p.T + d) * p.H + h) * D;
            const uint4* from = reinterpret_cast<const uint4*>(src + half_of(u) * 64 + qd * 16);
            v[u][0] = __ldg(from);
            v[u][1] = __ldg(from + 1);
        }
    }
    bool odd = false;
#pragma unroll
    for (int u = 0; u < D / 32; ++u) {
        const int half = half_of(u), row = row_at(u);
        const uint32_t at = slot + (value ? region * D * 128 + half * 8192 : region * 8192 + half * 16384) + row * 128 + x;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            uint4 y = v[u][e];
            if (value) {
                y = make_uint4(finite_halves(y.x, odd), finite_halves(y.y, odd), finite_halves(y.z, odd), finite_halves(y.w, odd));
                y = reorder8(y);
            }
            sts128(at ^ (16 * e), y);
        }
    }
    return odd;
}

template <class L, int D, bool KEYS>
__device__ __forceinline__ void decode_role(const TreeArgs& p, uint32_t ring_at, uint32_t ring, uint32_t bars, volatile int* dead,
                                            volatile int* odd, int first, int last, bool has_tail, int warp, int lane) {
    constexpr int U = D / 32;
    const int region = warp >> 2, k = (warp & 3) * 8 + (lane >> 2), qd = lane & 3;
    const uint32_t side = D == 128 ? (lane >> 2 ^ lane >> 3) & 1 : 0;
    const uint32_t to = region * D * 128 + k * 128 + (((2 * qd) ^ (k & 7)) << 4);
    uint32_t buf = 0, turn = 0;
    int index = 0;
    for (int tile = first; tile < last; ++index) {
        Segment s;
        s.at(p, tile, last);
        tile += s.c;
#pragma unroll 1
        for (int q = 0; q < (KEYS ? 1 : 2) * s.c; ++q) {
            bool value = false;
            const int i = s.t0 + (KEYS ? q : tile_of(q, s.c, 3 - p.groups, value));
            const uint32_t slot = ring_at + buf * L::TILE_BYTES;
            const int some = p.nb * BLK - i * TILE;    // (the tail's: none, or an odd block's)
            const Masked left = value && p.mask && some > 0 ? mask_of(p.mask + s.b * p.mask_stride + i * TILE, some, lane) : ALL;
            bar_wait(bars + 8 * (L::RAW + buf), turn & 1, dead);
            if (has_tail && i == p.tiles - 1) {
                if (tail_share<D>(p, s.b, s.h, value, slot, warp, lane) && !KEYS) odd[index % L::SEGMENTS] = index + 1;
            } else {
                const int kr = value ? swapped(k) : k;             // (V's tokens are stored in the order of the scores' columns)
                const bool by_half = D == 128 && value;
                const uint32_t at = slot + region * D * 128;
                const uint32_t e0 = by_half ? kr * 128 + side * 64 + qd * 16 : kr * 64 + qd * 16;
                const uint32_t e1 = by_half ? e0 ^ 64 : D == 64 ? e0 + 2048 : e0 + 4096, t = by_half ? 4096 : 2048;
                uint32_t w[U][8];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t e = (u & 1 ? e1 : e0) + (u >> 1) * t;
                    const uint4 h = lds128(at + e);
                    const uint2 m = lds64(at + D * 64 + e / 2), l = lds64(at + D * 96 + e / 2);
                    w[u][0] = h.x; w[u][1] = h.y; w[u][2] = h.z; w[u][3] = h.w;
                    w[u][4] = m.x; w[u][5] = m.y; w[u][6] = l.x; w[u][7] = l.y;
                }
                __syncwarp();                          // the region's bytes are in registers
                asm volatile("bar.sync %0, 128;\n" ::"r"(2 + region) : "memory");
                const uint32_t f0 = slot + to + (by_half ? side * 8192 : 0), f1 = slot + to + (by_half ? (side ^ 1) * 8192 : D == 64 ? 4096 : 8192);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t f = (u & 1 ? f1 : f0) + (u >> 1) * 4096;
                    sts128(f, swapped8(w[u][0], w[u][1], w[u][4], w[u][6]));
                    sts128(f ^ 16, swapped8(w[u][2], w[u][3], w[u][5], w[u][7]));
                }
                if (some < TILE || left != ALL) {
                    // (a token that does not exist or is masked away counts as zero, whatever there is: 0 * NaN would be NaN)
                    const uint16_t* mask = left == SOME ? reinterpret_cast<const uint16_t*>(p.mask) + s.b * p.mask_stride + i * TILE : nullptr;
#pragma unroll 1
                    for (int u = 0; u < U; ++u) {
                        const int tok = region * BLK + (value ? (D == 128 ? u >> 1 : u) * 32 + kr : 0);
                        if (tok >= some || left == NONE || (mask && mask[tok] == 0xFC00u)) {
                            const uint32_t f = (u & 1 ? f1 : f0) + (u >> 1) * 4096;
                            sts128(f, make_uint4(0, 0, 0, 0));
                            sts128(f ^ 16, make_uint4(0, 0, 0, 0));
                        }
                    }
                }
            }
            fence_shared();
            __syncwarp();
            if (lane == 0) bar_arrive(bars + 8 * (L::FULL + buf));
            if (++buf == ring) {
                buf = 0;
                ++turn;
            }
        }
    }
}

// ---------------------------------------------------------------- products
// The whole warp goes through this, one lane issues: addresses and descriptors are then the same for all lanes and come from uniform
// registers (by one lane alone a product took about 100 cycles to issue, and the issuing thread bound the kernel).
template <int D>
__device__ __forceinline__ void product_role(const TreeArgs& p, uint32_t base, uint32_t bars, uint32_t tmem, volatile int* dead,
                                             int first, int last) {
    using L = Plan<D>;
    uint32_t buf = 0, turn = 0, k_at = 0, k_buf = 0, v_at = 0, v_buf = 0;
    uint32_t items0 = 0, items1 = 0, seg = 0;          // of each slot so far
    const bool one = p.groups == 1;
    // the next operand tile: they come in the order in which they are first used
    auto take = [&](uint32_t& at, uint32_t& of) {
        bar_wait(bars + 8 * (L::FULL + buf), turn & 1, dead);
        at = base + L::RING_AT + buf * L::TILE_BYTES;
        of = buf;
        if (++buf == L::RING) {
            buf = 0;
            ++turn;
        }
    };
    for (int tile = first; tile < last; ++seg) {
        Segment s;
        s.at(p, tile, last);
        tile += s.c;
        bar_wait(bars + 8 * L::Q_FULL, seg & 1, dead);
        const int n_items = p.groups * s.c, tail_from = s.t0 + s.c == p.tiles ? n_items - p.groups : n_items;
#pragma unroll 1
        for (int n = -2; n < n_items; ++n) {           // output of item n, scores of item n + 2
            const uint32_t slot = n & 1;
            if (n >= 0) {
                bar_wait(bars + 8 * (L::P_FULL + slot), (slot ? items1 : items0) & 1, dead);
                if (one || !slot) take(v_at, v_buf);
                fence_after();
                const uint32_t v = operand(v_at, 8192), o = tmem + 256 + slot * 128, pr = tmem + slot * TILE;
                if (elect()) {
#pragma unroll
                    for (int kk = 0; kk < TILE / 16; ++kk)
                        mma_ts(o, pr + kk * 8, v + (kk >> 2) * (D * 128 >> 4) + (kk & 3) * (2048 >> 4), instruction(D, true), n >= 2 || kk > 0);
                    commit(bars + 8 * (L::O_FULL + slot));
                    if (one || slot) commit(bars + 8 * (L::EMPTY + v_buf));
                }
                __syncwarp();
                if (slot) ++items1;
                else ++items0;
            }
            if (n + 2 >= n_items) continue;
            if (one || !slot) take(k_at, k_buf);
            // (S takes P's place: the product that reads P has to be over, that of the segment before too)
            const uint32_t before = slot ? items1 : items0;
            if (before) bar_wait(bars + 8 * (L::O_FULL + slot), (before - 1) & 1, dead);
            fence_after();
            // 16 channels: of Q and of the tail's keys 32 bytes of rows of 64 (K-major), of K's planes 16 rows of 64 tokens
            const bool tail = n + 2 >= tail_from;
            const uint32_t q = operand(base + ((one ? seg & 1 : slot) ? L::Q2_AT : L::Q_AT), 16), k = operand(k_at, tail ? 16 : D * 128);
            const uint32_t near = tail ? 32 >> 4 : 2048 >> 4, far = tail ? 16384 >> 4 : 8192 >> 4;
            const uint32_t idesc = tail ? instruction(TILE, false) : instruction(TILE, true), d = tmem + slot * TILE;
            if (elect()) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    mma_ss(d, q + (kk >> 2) * (16384 >> 4) + (kk & 3) * (32 >> 4), k + (kk >> 2) * far + (kk & 3) * near, idesc, kk > 0);
                commit(bars + 8 * (L::S_FULL + slot));
                if (one || slot) commit(bars + 8 * (L::EMPTY + k_buf));
            }
            __syncwarp();
        }
    }
}

// ---------------------------------------------------------------- softmax
// A CTA's part of a unit: four channels of all rows side by side, as the lanes of a warp have and write them (row after row, no two
// lanes' stores shared a line: 75.5 us against 70.6 at 256 rows x 8192 tokens), behind them the rows' maxima and their sums of the
// probabilities, as they are and as they entered their product.  As in
// akv_tree.cu, slot 0 is of a run's first unit, slot 1 of its last.
struct Record {
    float* at;
    int rows, D, row;
    __device__ __forceinline__ Record(const TreeArgs& p, int D, int index, int row) :
        at(p.part + (size_t)index * p.rowsu * (D + 4)), rows(p.rowsu), D(D), row(row) {}
    __device__ __forceinline__ float4* quad(int q) const { return reinterpret_cast<float4*>(at) + q * rows + row; }
    __device__ __forceinline__ float4* stats() const { return reinterpret_cast<float4*>(at + rows * D) + row; }
    __device__ __forceinline__ float& operator[](int c) const { return reinterpret_cast<float*>(quad(c >> 2))[c & 3]; }
};

template <int D>
__device__ __forceinline__ void softmax_role(const TreeArgs& p, uint8_t* smem, uint32_t base, uint32_t bars, uint32_t tmem,
                                             volatile int* dead, volatile int* odd, int first, int last, int warp, int lane) {
    const int slot = warp >> 2, idx = (warp & 3) * 32 + lane, R = p.T * p.G, group = p.groups == 2 ? slot : 0;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_at = tmem + lanes + slot * TILE, o_at = tmem + lanes + 256 + slot * 128;
    const float scale2 = fabsf(p.scale2);          // (the queries take the sign)
    const uint32_t sign = p.scale2 < 0.f ? 0x80008000u : 0u;
    float* xm = reinterpret_cast<float*>(smem + Plan<D>::XM_AT);
    float* xl = reinterpret_cast<float*>(smem + Plan<D>::XL_AT);
    float* xr = reinterpret_cast<float*>(smem + Plan<D>::XR_AT);
    // Queries of the segment that begins with `tile`, 16-byte piece c of a row's half at c ^ (row & 7): a warp's 32 rows (with one group
    // either slot's warp takes half of their pieces), neighbouring pieces by neighbouring lanes and all on their way at once (a row
    // a lane, by way of registers or not, took 4 us at the start of 256 rows).  Then they are handed over.
    const int per = p.groups == 1 ? D / 16 : D / 8, i0 = p.groups == 1 ? slot * per : 0;             // (steps of 32 pieces)
    auto query_place = [&](int index, int i) {
        const int row = (warp & 3) * 32 + i * 32 / (D / 8) + lane / (D / 8), c = lane % (D / 8);
        return base + ((p.groups == 2 ? group : index & 1) ? Plan<D>::Q2_AT : Plan<D>::Q_AT) + row * 128 + (c >> 3) * Plan<D>::Q_HALF +
               (((c & 7) ^ (row & 7)) << 4);
    };
    auto request_queries = [&](int tile, int index) {
        Segment s;
        s.at(p, tile, last);
        const int of_unit = group * p.rowsg + idx, r = s.super * p.rowsu + of_unit;
        const int mine = idx < p.rowsg && of_unit < p.rowsu && r < R ? row_of(p, s.b, s.h, r) : -1;
#pragma unroll 4
        for (int i = i0; i < i0 + per; ++i) {
            const int row = __shfl_sync(0xFFFFFFFFu, mine, i * 32 / (D / 8) + lane / (D / 8));
            copy16(query_place(index, i), p.q + (long long)max(row, 0) * D + 8 * (lane % (D / 8)), row >= 0);
        }
        cp_async_commit();
    };
    auto hand_queries_over = [&](int index) {
        cp_async_wait<0>();
        if (sign) {
#pragma unroll 1
            for (int i = i0; i < i0 + per; ++i) {
                const uint4 x = lds128(query_place(index, i));
                sts128(query_place(index, i), make_uint4(x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign));
            }
        }
        fence_shared();
        __syncwarp();
        if (lane == 0) bar_arrive(bars + 8 * Plan<D>::Q_FULL);
    };
    uint32_t done = 0;
    int seg = 0;
    request_queries(first, 0);
    hand_queries_over(0);
    for (int tile = first; tile < last; ++seg) {
        Segment s;
        s.at(p, tile, last);
        tile += s.c;
        const int of_unit = group * p.rowsg + idx, r = s.super * p.rowsu + of_unit;
        const bool mine = idx < p.rowsg && of_unit < p.rowsu && r < R;
        const bool busy = __any_sync(0xFFFFFFFFu, mine);
        soft_sync();                                   // (the join of the segment before has been read)
        const bool with_tail = s.t0 + s.c == p.tiles;
        unsigned long long seen = 0;
        if (with_tail && mine) {
            const uint8_t* row = p.tree + s.b * p.tree_stride + (unsigned)r / (unsigned)p.G * p.T;
#pragma unroll 16
            for (int d = 0; d < p.T; ++d) seen |= (unsigned long long)(row[d] != 0) << d;
        }
        const __half* mask = p.mask ? p.mask + s.b * p.mask_stride : nullptr;
        float ref = -INFINITY, l = 0.f, lr = 0.f;      // (lr: the sum of the rounded probabilities)
        const int n_items = p.groups * s.c;
        bool any = false;
        for (int n = slot; n < n_items; n += 2, ++done) {
            const int i = s.t0 + (p.groups == 1 ? n : n >> 1), cached = p.nb * BLK - i * TILE;
            const bool tail = i == p.tiles - 1;
            const Masked left = mask && !tail ? mask_of(mask + i * TILE, cached, lane) : ALL;
            bar_wait(bars + 8 * (Plan<D>::S_FULL + slot), done & 1, dead);
            __syncwarp();
            fence_after();
            if (left == NONE) {
                const uint32_t zeros[16] = {0};
#pragma unroll
                for (int c = 0; c < TILE / 2; c += 16) tmem_st16(s_at + c, zeros);
                tmem_st_wait();
                any = true;
            } else if (busy) {
                // edges: scores to base 2 go back to where they came from; elsewhere they stay products until the exponential
                const bool plain = !tail && left == ALL && cached >= TILE;
                const float mul = plain ? scale2 : 1.f;
                uint32_t v[32];
                if (!plain) {
                    // tokens that are there for this row, a bit each (a block that is missing: 64 columns in any order)
                    const int count = tail ? p.rest : cached;
                    unsigned long long there = ~0ull, above = cached >= TILE ? there : 0;
                    if (tail) {
                        there = seen << p.rest | ((1ull << p.rest) - 1);
                        above = p.rest ? seen >> (64 - p.rest) : 0;
                    }
#pragma unroll 1
                    for (int c = 0; c < TILE; c += 32) {
                        const int tok = c + (tail ? lane : swapped(lane));
                        const uint32_t bits = (uint32_t)((c & 64 ? above : there) >> (c & 32));
                        float add = 0.f;
                        if (mask && tok < count) add = __half2float(mask[min(i * TILE, p.nb * BLK) + tok]) * LOG2E;
                        __syncwarp();
                        tmem_ld(v, s_at + c);
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float a = __shfl_sync(0xFFFFFFFFu, add, j);
                            v[j] = __float_as_uint((bits >> j & 1) && a != -INFINITY ? fmaf(__uint_as_float(v[j]), scale2, a) : -INFINITY);
                        }
                        tmem_st32(s_at + c, v);
                    }
                    tmem_st_wait();
                }
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                for (int c = 0; c < TILE; c += 32) {
                    tmem_ld(v, s_at + c);
#pragma unroll
                    for (int j = 0; j < 32; ++j) tops[j & 3] = fmaxf(tops[j & 3], __uint_as_float(v[j]));
                }
                const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * mul;
                const bool up = top > ref + SLACK;           // (-inf: the first score that is there)
                if (__any_sync(0xFFFFFFFFu, up)) {
                    const float to = fmaxf(ref, top), keep = ref == -INFINITY ? 0.f : ex2(ref - to);
                    ref = to;
                    l *= keep;
                    lr *= keep;
                    if (any) {
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            tmem_ld(v, o_at + c);
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * keep);
                            tmem_st32(o_at + c, v);
                        }
                    }
                }
                const float off = (ref == -INFINITY ? 0.f : ref) - WIDE_LIFT;
                float sums[4] = {0.f, 0.f, 0.f, 0.f}, rounded[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                for (int c = 0; c < TILE; c += 32) {
                    tmem_ld(v, s_at + c);
                    uint32_t h[16];
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float a = ex2(fmaf(__uint_as_float(v[j]), mul, -off)), b = ex2(fmaf(__uint_as_float(v[j + 1]), mul, -off));
                        sums[j & 2] += a;
                        sums[(j & 2) + 1] += b;
                        h[j / 2] = pack_half2(a, b);
                        rounded[j & 2] = plus_low(rounded[j & 2], h[j / 2]);
                        rounded[(j & 2) + 1] = plus_high(rounded[(j & 2) + 1], h[j / 2]);
                    }
                    tmem_st16(s_at + c / 2, h);
                }
                l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
                lr += (rounded[0] + rounded[1]) + (rounded[2] + rounded[3]);
                tmem_st_wait();
                any = true;
            }
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(bars + 8 * (Plan<D>::P_FULL + slot));
        }
        // (this slot's products with the queries are over - with one group the next ones have a place of their own - while its last
        // output is still under way)
        if (tile < last) request_queries(tile, seg + 1);
        // ---- the segment's result: with one group the slots' two, joined
        const bool have = n_items > slot;
        if (have) bar_wait(bars + 8 * (Plan<D>::O_FULL + slot), (done - 1) & 1, dead);
        if (tile < last) hand_queries_over(seg + 1);
        __syncwarp();
        fence_after();
        float f0 = 1.f, f1 = 0.f;
        if (p.groups == 1) {
            if (slot) {
                xm[idx] = have ? ref : -INFINITY;
                xl[idx] = have ? l : 0.f;
                xr[idx] = have ? lr : 0.f;
            }
            soft_sync();
            if (!slot && n_items > 1) {
                const float to = fmaxf(ref, xm[idx]);
                f0 = ref == -INFINITY ? 0.f : ex2(ref - to);
                f1 = xm[idx] == -INFINITY ? 0.f : ex2(xm[idx] - to);
                // (a sum that is not a number stays one: 0 * NaN)
                l = f0 * l + f1 * xl[idx];
                lr = f0 * lr + f1 * xr[idx];
                ref = to;
            }
        }
        const bool whole = s.c == p.tiles, odd_tail = with_tail && odd[seg % Plan<D>::SEGMENTS] == seg + 1;
        if (*dead) l = lr = __int_as_float(0x7FC00000);
        const float inv = lr == 0.f ? 0.f : 1.f / lr;
        const int rec_slot = s.unit != (unsigned)first / (unsigned)p.tiles;
        const Record rec(p, D, 2 * blockIdx.x + rec_slot, of_unit);
        float4* join = reinterpret_cast<float4*>(smem + (seg & 1 ? Plan<D>::Q2_AT : Plan<D>::Q_AT));              // [16 channel quads][128 rows]
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            if (p.groups == 1 && c % 64 == 0) {
                if (c > 0) soft_sync();
                if (slot && have && busy) {
#pragma unroll 1
                    for (int e = 0; e < 64; e += 32) {
                        uint32_t v[32];
                        __syncwarp();
                        tmem_ld(v, o_at + c + e);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            join[(e / 4 + j) * 128 + idx] = make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 2]),
                                                                        __uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 3]));
                    }
                }
                soft_sync();
            }
            if ((p.groups == 1 && slot) || !busy) continue;
            uint32_t v[32];
            __syncwarp();
            tmem_ld(v, o_at + c);
            float o[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __uint_as_float(v[swapped(j)]);
            if (p.groups == 1 && n_items > 1) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float4 x = join[((c & 63) / 4 + j) * 128 + idx];
                    o[4 * j] = fmaf(o[4 * j], f0, x.x * f1);
                    o[4 * j + 1] = fmaf(o[4 * j + 1], f0, x.y * f1);
                    o[4 * j + 2] = fmaf(o[4 * j + 2], f0, x.z * f1);
                    o[4 * j + 3] = fmaf(o[4 * j + 3], f0, x.w * f1);
                }
            }
            if (!mine) continue;
            if (whole) {
                uint4* dst = reinterpret_cast<uint4*>(p.out + (long long)row_of(p, s.b, s.h, r) * D + c);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    dst[j] = make_uint4(pack_half2(o[8 * j] * inv, o[8 * j + 1] * inv), pack_half2(o[8 * j + 2] * inv, o[8 * j + 3] * inv),
                                        pack_half2(o[8 * j + 4] * inv, o[8 * j + 5] * inv), pack_half2(o[8 * j + 6] * inv, o[8 * j + 7] * inv));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    *rec.quad(c / 4 + j) = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            }
        }
        if (mine && !(p.groups == 1 && slot)) {
            if (odd_tail) {
                const float off = (ref == -INFINITY ? 0.f : ref) - WIDE_LIFT;
                if (whole) add_odd(p, s.b, s.h, r, D, off, inv, p.out + (long long)row_of(p, s.b, s.h, r) * D);
                else add_odd(p, s.b, s.h, r, D, off, 1.f, rec);
            }
            if (!whole) {
                *rec.stats() = make_float4(ref, l, lr, 0.f);
            } else if (p.lse) {
                p.lse[row_of(p, s.b, s.h, r)] = l == 0.f ? -INFINITY : (ref - WIDE_LIFT + log2f(l)) * LN2;
            }
        }
        fence_before();
    }
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1) tree_wide_kernel(const __grid_constant__ TreeArgs p) {
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const uint32_t base = smem_u32(smem), bars = base + Plan<D>::BAR_AT;
    using L = Plan<D>;
    uint32_t* slot_tmem = reinterpret_cast<uint32_t*>(smem + L::BAR_AT + 8 * L::BARS);
    volatile int* dead = reinterpret_cast<volatile int*>(slot_tmem + 1);
    volatile int* odd = dead + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
#pragma unroll 1
        for (int i = 0; i < L::RING; ++i) {
            bar_init(bars + 8 * (L::RAW + i), 1);
            bar_init(bars + 8 * (L::FULL + i), DECODE);
            bar_init(bars + 8 * (L::EMPTY + i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(bars + 8 * (L::S_FULL + i), 1);
            bar_init(bars + 8 * (L::P_FULL + i), SOFT / 2);
            bar_init(bars + 8 * (L::O_FULL + i), 1);
        }
        bar_init(bars + 8 * L::Q_FULL, SOFT);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        *dead = 0;
#pragma unroll 1
        for (int i = 0; i < L::SEGMENTS; ++i) odd[i] = 0;
    }
    // (the memory is taken once the kernel in front is over: it might want some, and this one would hold it while it waits)
    pdl_enter();
    __syncwarp();
    if (warp == SOFT + DECODE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(slot_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(slot_tmem);
    const int first = run_start(p, blockIdx.x), last = run_start(p, blockIdx.x + 1);
    if (warp < SOFT) {
        softmax_role<D>(p, smem, base, bars, tmem, dead, odd, first, last, warp, lane);
    } else if (warp < SOFT + DECODE) {
        decode_role<L, D, false>(p, base + L::RING_AT, L::RING, bars, dead, odd, first, last, true, warp - SOFT, lane);
    } else if (warp == SOFT + DECODE) {
        product_role<D>(p, base, bars, tmem, dead, first, last);
    } else {
        copy_role<L, D, false>(p, base + L::RING_AT, L::RING, bars, dead, first, last, true);
    }
    __syncwarp();
    __syncthreads();
    if (*dead) {
        // (never expected) products may still run: time for them to end before their memory is released
#pragma unroll 1
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        __syncthreads();
    }
    fence_after();
    if (warp == SOFT + DECODE)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
}

// A thread per row and four channels: the records of the runs that share its unit, in the order of the tokens, four under way at a time.
template <int D>
__global__ void __launch_bounds__(2 * D) tree_wide_merge_kernel(const __grid_constant__ TreeArgs p) {
    pdl_trigger();
    constexpr int STEP = 4;
    const int q = threadIdx.x >> 3, row = blockIdx.x * 8 + (threadIdx.x & 7);   // row: unit * rowsu + row of the unit
    const int unit = (unsigned)row / (unsigned)p.rowsu, of_unit = row - unit * p.rowsu;
    const int bh = (unsigned)unit / (unsigned)p.rt, b = (unsigned)bh / (unsigned)p.H, h = bh - b * p.H;
    const int r = (unit - bh * p.rt) * p.rowsu + of_unit;
    const int w0 = run_with(p, unit * p.tiles), w1 = run_with(p, unit * p.tiles + p.tiles - 1);
    const long long to = row_of(p, b, h, r);
    const int skip = run_start(p, w0) < unit * p.tiles;                        // (the first run of the unit's may have begun before it)
    pdl_wait();
    // (a whole unit has been written by its run)
    if ((unsigned)unit >= (unsigned)p.total / (unsigned)p.tiles || r >= p.T * p.G || w0 == w1) return;
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f, lr = 0.f, top = -INFINITY;
#pragma unroll 1
    for (int w = w0; w <= w1; w += STEP) {
        float4 ml[STEP];
        float4 o[STEP];
#pragma unroll
        for (int k = 0; k < STEP; ++k) {
            const Record rec(p, D, 2 * (w + k) + (w + k == w0 ? skip : 0), of_unit);
            ml[k] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
            o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (w + k > w1) continue;
            ml[k] = *rec.stats();
            o[k] = *rec.quad(q);
        }
        float t = top;
#pragma unroll
        for (int k = 0; k < STEP; ++k) t = fmaxf(t, ml[k].x);
        const float base = t == -INFINITY ? 0.f : t, keep = ex2(top - base);
        top = t;
        l *= keep;
        lr *= keep;
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] *= keep;
#pragma unroll
        for (int k = 0; k < STEP; ++k) {
            const float f = ex2(ml[k].x - base);
            l = fmaf(f, ml[k].y, l);
            lr = fmaf(f, ml[k].z, lr);
            acc[0] = fmaf(f, o[k].x, acc[0]);
            acc[1] = fmaf(f, o[k].y, acc[1]);
            acc[2] = fmaf(f, o[k].z, acc[2]);
            acc[3] = fmaf(f, o[k].w, acc[3]);
        }
    }
    const float inv = lr == 0.f ? 0.f : 1.f / lr;
    *reinterpret_cast<uint2*>(p.out + to * D + 4 * q) = make_uint2(pack_half2(acc[0] * inv, acc[1] * inv), pack_half2(acc[2] * inv, acc[3] * inv));
    if (p.lse && q == 0) p.lse[to] = l == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) - WIDE_LIFT + log2f(l)) * LN2;
}

// ---------------------------------------------------------------- weights
// weights[t] += sum over the rows of exp(s_t - lse): keys alone, and the product the other way round: S^T = K Q^T, a tile's 128 tokens
// by up to 128 rows, so that a thread has a token and adds its rows up by itself, whatever their number: no warp has to wait for
// another's, and the order is always the same.  Copy and decode as above, the ring as deep as the queries leave room for; two score
// slots, the tiles in turn.  One row is bound by HBM (8 x 32 x 4096 tokens: 51 us, 5.4 TB/s of 6.5); 128 rows (4 x 8 x 8190: 30 us)
// by the threads' chain of loads and exponentials (5 us less without), the rest is the start and the end of a run of 14 tiles.
template <int D>
struct KeysPlan {
    static constexpr int RING = D == 128 ? 6 : 8, TILE_BYTES = TILE * D * 2, SEGMENTS = 8;
    static constexpr int RAW = 0, FULL = RING, EMPTY = 2 * RING, S_FULL = 3 * RING, S_FREE = S_FULL + 2, Q_FULL = S_FREE + 2, BARS = Q_FULL + 1;
    // A product of 128 channels is eight steps into one fp32 sum, and each of them cuts off what does not fit: 4.3e-6 of the weights at
    // scores of 25, all to one side.  Rows go in groups of 128, and a group's steps into as many sums as a slot's 256 columns have room
    // for, added up (and rounded) by the threads: 1.9e-6 with four, 2.2e-6 with two (a plain fp32 product: 1.6e-6), for 2 us of 50.
    static constexpr int GROUP = 128, MOST_SUMS = 4;
    static __device__ __forceinline__ int lg_steps(int columns) {             // log2 of the steps into one sum
        int lg = 0;
        while ((D / 16 >> lg) > MOST_SUMS || (D / 16 >> lg) * columns > 256) ++lg;
        return lg;
    }
    static constexpr int ROWS = 512, OFF_AT = 512, Q_AT = OFF_AT + ROWS * 4 + 512;          // barriers and words; -lse of the rows; queries
    static_assert(8 * BARS + 8 + ROWS / 32 * 4 <= OFF_AT && Q_AT % 1024 == 0, "layout");
    static __host__ __device__ int padded(int rows) { return (rows + 15) & ~15; }
    static __host__ __device__ int ring_at(int rows) { return (Q_AT + padded(rows) * D * 2 + 1023) & ~1023; }
    static __host__ __device__ int depth(int rows) {
        const int fit = (232448 - 1024 - ring_at(rows)) / TILE_BYTES;
        return fit < RING ? fit : RING;
    }
    static __host__ __device__ int bytes(int rows) { return 1024 + ring_at(rows) + depth(rows) * TILE_BYTES; }
};

// exp(score - lse) of a token's first n rows, added to four interleaved sums: 16 rows of SUMS = 4 or 32 of 2 at a time.
template <int SUMS>
__device__ __forceinline__ void add_rows(float (&sum)[4], uint32_t s_at, uint32_t columns, int n, const float* off, const uint32_t* absent,
                                         float scale, float add) {
    constexpr int ROWS = 64 / SUMS;
    const uint32_t pair = SUMS == 4 ? 2 * columns : 16;
#pragma unroll 1
    for (int c = 0; c < n; c += ROWS) {
        uint32_t v[4][16];
        __syncwarp();
        tmem_ld4(v, s_at + c, s_at + columns + c, s_at + pair + c, s_at + columns + pair + c);
        float x[ROWS];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            x[e] = __uint_as_float(v[0][e]) + __uint_as_float(v[1][e]);
            const float y = __uint_as_float(v[2][e]) + __uint_as_float(v[3][e]);
            if constexpr (SUMS == 4) x[e] += y;
            else x[16 + e] = y;
        }
        if (const uint32_t none = absent[c >> 5] >> (c & 16)) {
            // (no weight from these, whatever their scores are: 0 - inf)
#pragma unroll
            for (int e = 0; e < ROWS; ++e) x[e] = none >> e & 1 ? 0.f : x[e];
        }
        // (one rounding of the small difference: scores of 25 are half of 2e-6 off themselves)
#pragma unroll
        for (int e = 0; e < ROWS / 4; ++e) {
            const float4 o = reinterpret_cast<const float4*>(off + c)[e];
            sum[0] += ex2(fmaf(fmaf(x[4 * e], scale, o.x), LOG2E, add));
            sum[1] += ex2(fmaf(fmaf(x[4 * e + 1], scale, o.y), LOG2E, add));
            sum[2] += ex2(fmaf(fmaf(x[4 * e + 2], scale, o.z), LOG2E, add));
            sum[3] += ex2(fmaf(fmaf(x[4 * e + 3], scale, o.w), LOG2E, add));
        }
    }
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1)
weights_wide_kernel(const __grid_constant__ TreeArgs p, float* __restrict__ weights, int row0, int rows) {
    using L = KeysPlan<D>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const uint32_t base = smem_u32(smem), bars = base;
    uint32_t* slot_tmem = reinterpret_cast<uint32_t*>(smem + 8 * L::BARS);
    volatile int* dead = reinterpret_cast<volatile int*>(slot_tmem + 1);
    uint32_t* absent = slot_tmem + 2;              // a bit per row: it sees nothing, or there is none
    float* off = reinterpret_cast<float*>(smem + L::OFF_AT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = L::depth(rows), ring_at = base + L::ring_at(rows), q_half = L::padded(rows) * 128;
    const int groups = (rows + L::GROUP - 1) / L::GROUP;
    const bool has_tail = p.rest > 0;
    if (threadIdx.x == 0) {
#pragma unroll 1
        for (int i = 0; i < L::RING; ++i) {
            bar_init(bars + 8 * (L::RAW + i), 1);
            bar_init(bars + 8 * (L::FULL + i), DECODE);
            bar_init(bars + 8 * (L::EMPTY + i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(bars + 8 * (L::S_FULL + i), 1);
            bar_init(bars + 8 * (L::S_FREE + i), SOFT / 2);
        }
        bar_init(bars + 8 * L::Q_FULL, SOFT);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        *dead = 0;
    }
    pdl_enter();
    __syncwarp();
    if (warp == SOFT + DECODE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(slot_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(slot_tmem);
    const int first = run_start(p, blockIdx.x), last = run_start(p, blockIdx.x + 1);
    if (warp < SOFT) {
        const int slot = warp >> 2, idx = (warp & 3) * 32 + lane;
        const uint32_t s_at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + slot * 256;
        uint32_t done = 0;
        for (int tile = first; tile < last;) {
            Segment s;
            s.at(p, tile, last);
            tile += s.c;
            soft_sync();                               // (all products with the queries before are over: their scores have been read)
            // (all at once: as loads, one after the other, they took 5 us of a call with 128 rows)
#pragma unroll 4
            for (int i = threadIdx.x; i < L::padded(rows) * (D / 8); i += 32 * SOFT) {
                const int r = i / (D / 8), c = i % (D / 8);
                copy16(base + L::Q_AT + (c >> 3) * q_half + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                       p.q + (long long)(r < rows ? row_of(p, s.b, s.h, row0 + r) : 0) * D + 8 * c, r < rows);
            }
            cp_async_commit();
#pragma unroll
            for (int r = threadIdx.x; r < L::ROWS; r += 32 * SOFT) {
                const float x = r < rows ? p.lse[row_of(p, s.b, s.h, row0 + r)] : -INFINITY;
                const uint32_t none = __ballot_sync(0xFFFFFFFFu, x == -INFINITY);
                off[r] = x == -INFINITY ? x : -x;
                if (lane == 0) absent[r >> 5] = none;
            }
            cp_async_wait<0>();
            fence_shared();
            soft_sync();                               // (`off` is everybody's)
            if (lane == 0) bar_arrive(bars + 8 * L::Q_FULL);
            for (int j = slot; j < s.c; j += 2) {
                const int i = s.t0 + j;
                const bool tail = has_tail && i == p.tiles - 1;
                const int at = tail ? p.nb * BLK : i * TILE, tok = tail ? idx : swapped(idx);
                const int count = tail ? p.rest : min(TILE, p.nb * BLK - at);
                float add = 0.f, sum[4] = {0.f, 0.f, 0.f, 0.f};
                if (p.mask && tok < count) add = __half2float(p.mask[s.b * p.mask_stride + at + tok]);
                const bool gone = tok >= count || add == -INFINITY;
                add *= LOG2E;
                float* to = weights + (long long)s.bh * p.L + at + tok;
                const float before = gone ? 0.f : *to;         // (on its way while the scores are)
                for (int g = 0; g < groups; ++g, ++done) {
                    bar_wait(bars + 8 * (L::S_FULL + slot), done & 1, dead);
                    __syncwarp();
                    fence_after();
                    const int n = min(L::GROUP, rows - L::GROUP * g), columns = L::padded(n), sums = D / 16 >> L::lg_steps(columns);
                    if (!__all_sync(0xFFFFFFFFu, gone)) {
                        const float* o = off + L::GROUP * g;
                        const uint32_t* none = absent + L::GROUP / 32 * g;
                        if (sums == 4) add_rows<4>(sum, s_at, columns, n, o, none, p.scale, add);
                        else add_rows<2>(sum, s_at, columns, n, o, none, p.scale, add);
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(bars + 8 * (L::S_FREE + slot));
                }
                if (!gone) {
                    float x = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    if (*dead) x = __int_as_float(0x7FC00000);
                    *to = before + x;
                }
            }
        }
    } else if (warp < SOFT + DECODE) {
        decode_role<L, D, true>(p, ring_at, ring, bars, dead, nullptr, first, last, has_tail, warp - SOFT, lane);
    } else if (warp == SOFT + DECODE) {
        uint32_t buf = 0, turn = 0, items0 = 0, items1 = 0, seg = 0, k_at[2] = {0, 0}, k_buf[2] = {0, 0};
        for (int tile = first; tile < last; ++seg) {
            Segment s;
            s.at(p, tile, last);
            tile += s.c;
            bar_wait(bars + 8 * L::Q_FULL, seg & 1, dead);
            // a pair of tiles, one for each slot, and of them the row groups one after the other
#pragma unroll 1
            for (int j0 = 0; j0 < s.c; j0 += 2) {
                for (int g = 0; g < groups; ++g) {
                    const int columns = L::padded(min(L::GROUP, rows - L::GROUP * g)), lg = L::lg_steps(columns), first_step = (1 << lg) - 1;
                    const uint32_t idesc_n = (uint32_t)(columns >> 3) << 17;
#pragma unroll
                    for (int slot = 0; slot < 2; ++slot) {
                        if (j0 + slot >= s.c) continue;
                        if (g == 0) {
                            bar_wait(bars + 8 * (L::FULL + buf), turn & 1, dead);
                            k_at[slot] = ring_at + buf * L::TILE_BYTES;
                            k_buf[slot] = buf;
                            if (++buf == ring) {
                                buf = 0;
                                ++turn;
                            }
                        }
                        bar_wait(bars + 8 * (L::S_FREE + slot), ((slot ? items1 : items0) & 1) ^ 1, dead);
                        fence_after();
                        const bool tail = has_tail && s.t0 + j0 + slot == p.tiles - 1;
                        const uint32_t q = operand(base + L::Q_AT + g * (L::GROUP * 128), 16), d = tmem + slot * 256, half = q_half >> 4;
                        if (tail) {
                            const uint32_t k = operand(k_at[slot], 16), idesc = instruction(0, false) | idesc_n;
                            if (elect()) {
#pragma unroll
                                for (int kk = 0; kk < D / 16; ++kk)
                                    mma_ss(d + (kk >> lg) * columns, k + (kk >> 2) * (16384 >> 4) + (kk & 3) * (32 >> 4),
                                           q + (kk >> 2) * half + (kk & 3) * (32 >> 4), idesc, kk & first_step);
                            }
                        } else {
                            const uint32_t k = operand(k_at[slot], D * 128), idesc = instruction(0, false, true) | idesc_n;
                            if (elect()) {
#pragma unroll
                                for (int kk = 0; kk < D / 16; ++kk)
                                    mma_ss(d + (kk >> lg) * columns, k + kk * (2048 >> 4), q + (kk >> 2) * half + (kk & 3) * (32 >> 4), idesc,
                                           kk & first_step);
                            }
                        }
                        if (elect()) {
                            commit(bars + 8 * (L::S_FULL + slot));
                            if (g == groups - 1) commit(bars + 8 * (L::EMPTY + k_buf[slot]));
                        }
                        __syncwarp();
                        if (slot) ++items1;
                        else ++items0;
                    }
                }
            }
        }
    } else {
        copy_role<L, D, true>(p, ring_at, ring, bars, dead, first, last, has_tail);
    }
    __syncwarp();
    __syncthreads();
    if (*dead) {
#pragma unroll 1
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        __syncthreads();
    }
    fence_after();
    if (warp == SOFT + DECODE)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
}

}  // namespace

int launch_tree_wide(const TreeArgs& p, int D, int ctas, int units, cudaStream_t st) {
    auto kernel = D == 128 ? tree_wide_kernel<128> : tree_wide_kernel<64>;
    const int bytes = D == 128 ? Plan<128>::BYTES : Plan<64>::BYTES;
    const int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                               "tree_attention shared memory");
    if (rc != AKV_OK) return rc;
    launch_chained(kernel, dim3(ctas), dim3(THREADS), (size_t)bytes, st, p);
    if (p.tiles > 1)                                   // (units of one tile: none is shared)
        launch_chained(D == 128 ? tree_wide_merge_kernel<128> : tree_wide_merge_kernel<64>,
                       dim3((unsigned)(((long long)units * p.rowsu + 7) / 8)), dim3(2 * D), 0, st, p);
    return cuda_status(cudaGetLastError(), "tree_attention launch");
}

int launch_weights_wide(const TreeArgs& p, int D, int ctas, float* weights, cudaStream_t st) {
    auto kernel = D == 128 ? weights_wide_kernel<128> : weights_wide_kernel<64>;
    int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448), "tree_weights shared memory");
    // (more rows than the queries' place holds: one launch after the other)
    for (int row0 = 0; rc == AKV_OK && row0 < p.T * p.G; row0 += KeysPlan<128>::ROWS) {
        const int left = p.T * p.G - row0, rows = left < KeysPlan<128>::ROWS ? left : KeysPlan<128>::ROWS;
        launch_chained(kernel, dim3(ctas), dim3(THREADS), (size_t)(D == 128 ? KeysPlan<128>::bytes(rows) : KeysPlan<64>::bytes(rows)), st, p,
                       weights, row0, rows);
        rc = cuda_status(cudaGetLastError(), "tree_weights launch");
    }
    return rc;
}

}  // namespace akv
