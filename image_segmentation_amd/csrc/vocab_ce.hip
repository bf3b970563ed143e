// Softmax cross entropy over a large table of classes, with its gradient, without the [rows, classes] scores ever in memory.
//
//   z = x W^T + b,  lse_m = log sum_v exp z_mv,  loss_m = (1-e)(lse_m - z_mt) + e (lse_m - mean_v z_mv)
//   dz_mv = c_m (exp(z_mv - lse_m) - (1-e)[v = t_m] - e/V),  dx = dz W,  dW = dz^T x,  db = sum_m dz
//
// Forward: every tile of z lives in accumulators only; its epilogue leaves one (base, sum of exponentials) pair a row and tile.
// Backward: a piece of the classes at a time, z is formed again, dz of the piece goes to a workspace in bf16 (fp32: in three bf16
// terms, see mma), and two more products read it.  Rows whose target is ignored are taken out first (order kept): they cost nothing,
// and what they hold (NaN included) reaches no gradient.
//
// 2 M D V operations forward, 6 M D V backward, against (M + V) D values read: wide rows are bound by the matrix pipes.  Narrow ones are
// not: the scores' and dz's epilogues (an exponential a score) stay what they are, and dz, written once and read twice, gives D operations
// a byte to each of dx and dW -- 256 of them where this card's copy and its matrix product balance at 312.  With the scores in memory the
// plain form moves 2 to 4 bytes of each several times over and takes the sum of three library products besides.  Measured, bf16, rows (one
// in ten ignored) x D x classes, forward and gradients: 16384 x 256 x 32000 in 1.25 ms (plain 10.6; scores 350 us, dz 436, dx 281, dW 244:
// 0.69, 0.55, 0.86 and 0.99 PFLOP/s of the rows that count; dz alone is 0.94 GB, 186 us a pass at a copy's rate), 8192 x 896 x 50257 in
// 2.44 ms (plain 19.3; scores 625, dz 684, dx 625, dW 661: 0.97 to 1.06); forward alone 4096 x 448 x 65536 in 223 to 234 us (plain 2945);
// few rows are bound by the table's bytes, read three times and its gradient written once: 1 x 896 x 50257 in 110 us (3.3 TB/s).
#include <type_traits>

#include "kernels.hpp"

namespace lsam {
namespace {

using lds_p = __attribute__((address_space(3))) void*;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int ROW_BAD = -1;   // target outside [0, V): the row's loss and gradient become NaN

// Exponentials are taken as 2^(z log2e - base) with a whole-number base: one fused multiply-add an element, and bases of different tiles
// differ by exact powers of two.  Where the highest score is beyond 2^30 the rounding of z log2e to a base would be a step of 2^64 and more;
// there neighbouring fp32 scores lie 128 apart, so that all but the highest itself count nothing, and exponentials are taken as
// 2^(z - max), exactly 1 for it.  The base is 2 max then: beyond every whole-number base, in the same order, and two of them, or one of
// either kind, are as far apart as their exponentials need.  Up to 1.7e38.
constexpr float FAR_Z = 0x1p30f, FAR_BASE = 0x1p31f;
struct Base {   // 2^(z mul - sub)
    float mul, sub;
    __device__ __forceinline__ explicit Base(float base) {
        const bool far = fabsf(base) > FAR_BASE;
        mul = far ? 1.f : LOG2E;
        sub = far ? 0.5f * base : base;
    }
    static __device__ __forceinline__ float of(float mx) { return fabsf(mx) > FAR_Z ? 2.f * mx : __builtin_ceilf(mx * LOG2E); }
};
constexpr float MASK = 1e38f;       // finite biases beyond it count as that: their scores' bases stay finite
constexpr float Z_SCALE = 0x1p-30f; // sums of scores are kept in units of 2^30: neither masks nor many classes leave the range

// ---------------------------------------------------------------------------------------------------------------------
// The product: Out[j][i] = sum_k A(i, k) B(j, k), i contiguous in Out.  An operand is stored "KC" ([i][k], k contiguous) or
// transposed ([k][i]).  Tile IT x JT, k-tiles of 128 bytes, two LDS stages filled by LDS-DMA.
// ---------------------------------------------------------------------------------------------------------------------
enum Mode { STATS, DZ, ACC, OUT, PART };   // PART: OUT in fp32

// The gradients of the scores are held in units of one number for all rows, `unit` times the incoming gradient (over n), chosen so that
// what dominates them -- the target's entry of a row that is not learned yet -- is exactly -1 under MEAN and SUM.  Rounded to bf16 at its
// own size, (1 - e) g / n, that entry would be off by the same fraction in every row, and the fraction would come through the sums
// whole.  The factor is applied to the fp32 sums; without rows every sum is 0 and stays it, whatever 1 / n is.
// Rounded all the same, once, where the operands are bf16: the matrix pipes multiply what they are given, and a second term would double
// both products.  Every entry is off by up to 2^-9 of itself, and dx and dW in L2 by 0.0019 to 0.0021 where their own rounding alone makes
// 0.0017 (a single row of two classes, where nothing averages: 0.0037 against 0.0027).  db is summed from the values before it.
struct Grad {
    const float* gout;
    int reduction;
    float unit;
    __device__ __forceinline__ float factor(int n) const {
        if (n == 0) return 0.f;
        return reduction == LSAM_REDUCE_NONE ? unit : reduction == LSAM_REDUCE_MEAN ? gout[0] * unit / (float)n : gout[0] * unit;
    }
};

struct CeArgs {
    const void* A; long lda;   // elements
    const void* B; long ldb;
    int I, J, K;               // limits; J (STATS, DZ, ACC) or K (OUT, PART) is further limited by *n
    const int* n;              // number of rows that count (device)
    // STATS / DZ
    const float* bias;         // [I] or null
    const int* tgt;            // [rows]
    int i_base;                // class of column 0
    float smooth_z;            // != 0: the sum of z over the classes is wanted too
    float* part;               // STATS: planes [tiles_i][rows_cap] of (base, sum of exponentials, sum of z in units of 1 / Z_SCALE)
    float* zt;                 // STATS: z of the target
    const float* base2;        // DZ: the row's base and its sum of exponentials
    const float* sum;
    const int* idx;
    float sm, keep;            // DZ: the subtrahends of every class and of the target, in units of the row's coefficient
    Grad grad;                 // DZ, OUT
    float* dbp;                // DZ: [tiles_j][I_cap] partial column sums or null
    long dbp_ld;
    int rows_cap;
    // outputs
    void* out; long ldo;       // DZ: bf16; OUT: the operands' type; ACC, PART: fp32
    int cols, vec;             // OUT: columns of a row; rows take whole vectors
    long split_stride;         // elements between the splits' outputs
    int splits, accumulate;
    long plane_a, plane_b, plane_out;   // fp32 operands: bytes between the three bf16 planes of A, of B and of DZ's output
};

__device__ __forceinline__ void mma(const uint4& a, const uint4& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// fp32 operands go through the bf16 matrix pipes as three terms, x = x0 + x1 + x2 exactly: 8 bits of the 24 each, whatever is left being
// rounded to the nearest 8.  |x1| <= 2^-9 |x|, |x2| <= 2^-18 |x|, so of the nine products the three left out, x1 y2, x2 y1 and x2 y2, come
// to at most 2^-25 |x y|: half of what rounding one fp32 product costs.  Six bf16 products at 16 times the fp32 instructions' rate; of a
// k-tile the small ones go first.  A k-tile holds all three planes of both operands, so that each is fetched and read once for its six
// products.  (2011 x 252 x 10007 forward and gradient: 303 to 317 us; 416 with
// fp32 matrix instructions, 357 with k run through once a product.)

// One operand's tile in LDS.  KC: R rows of KE values, 16-byte chunk c of row r at c ^ (r & 7) (KE = 32, four chunks: c ^ (r / 4 & 3)), so
// that sixteen rows' reads of one chunk fall on different banks.  Transposed: KE rows of R values, read
// with the transposing LDS load (16 lanes take 4 k-rows x 16 columns), whose 8 rows of a half wave must fall on different banks: 32-byte
// column pair p of row k at p ^ h(k), h = k's bits 0, 1, 3.
// DMA instruction q (of NI a wave) fills 1 KB; from one q to the next a lane's source moves by a fixed number of rows, and its chunk
// within the row stays, so one offset and one first k describe them all.  Rows of a KC tile behind the limit lie behind the
// descriptor's last byte and read zeros; every other chunk that must not be read gets an offset that does.
template <bool KC, int R, int NW, int KE> struct Tile {
    static constexpr int RB = R * 2, KB = KE * 2, BYTES = R * KB;
    static constexpr int NI = BYTES / 1024 / NW;               // DMA instructions a wave and stage
    static constexpr int ROWS = NW * 1024 / (KC ? KB : RB);    // rows from one of them to the next
    static_assert(KE == 64 || KE == 32, "chunks of a KC row");
    static_assert(BYTES % (1024 * NW) == 0 && NW * 1024 % (KC ? KB : RB) == 0 && ROWS % 16 == 0, "a lane's chunk stays");
    static __device__ __forceinline__ int swizzle(int c, int row) { return KE == 64 ? c ^ (row & 7) : c ^ ((row >> 2) & 3); }
    unsigned vo;   // byte offset of this lane's first chunk in the k-tile's slab
    int ke, col;   // its first k; transposed: its first column in the tile
    __device__ __forceinline__ void init(int wave, int lane, long ld) {
        const int b = wave * 1024 + lane * 16;
        if constexpr (KC) {
            const int row = b / KB, c = swizzle((b % KB) >> 4, row);
            vo = (unsigned)((long)row * ld * 2 + c * 16);
            ke = c * 8;
            col = 0;
        } else {
            const int k = b / RB, c = ((b % RB) >> 4) ^ (2 * ((k & 3) | (((k >> 3) & 1) << 2)));
            vo = (unsigned)((long)k * ld * 2 + c * 16);
            ke = k;
            col = c * 8;
        }
    }
    // k-tile slab: KC advances KE values along the rows, transposed KE rows
    static __device__ __forceinline__ const char* slab(const void* base, long ld, int r0, long k0) {
        const char* p = static_cast<const char*>(base);
        return KC ? p + ((long)r0 * ld + k0) * 2 : p + (k0 * ld + r0) * 2;
    }
    static __device__ __forceinline__ long step(long ld) { return KC ? KB : KE * ld * 2; }
    // DMA instruction q of a k-tile of which `left` k and `rows` rows (columns, transposed) exist
    __device__ __forceinline__ void issue(const char* slab_p, char* dst, int wave, int left, int q, long ld, int rows) const {
        const int bytes = KC ? rows * (int)ld * 2 : 0x7FFFFFFF;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(slab_p), 0, bytes, 0x00020000);
        unsigned vo = this->vo;
        asm volatile("" : "+v"(vo));   // the NI offsets are not held across the loop
        const bool ok = KC ? ke < left : ke < left - q * ROWS && col < rows;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_p)(dst + (wave + NW * q) * 1024), 16,
                                                 ok ? vo + (unsigned)(q * ROWS * 2) * (unsigned)ld : 0xFFFFFFFFu, 0, 0, 0);
    }
    // the fragment of 16-wide tile t, k-step ks (0, 1): lane (g, lr) holds column 16 t + lr, its share of the step's k
    static __device__ __forceinline__ uint4 read(const char* s, int t, int ks, int g, int lr) {
        if constexpr (KC) return *reinterpret_cast<const uint4*>(s + (t * 16 + lr) * KB + (swizzle(ks * 4 + g, lr) << 4));
        using s4 = __attribute__((ext_vector_type(4))) short;
        using s4p = __attribute__((address_space(3))) s4*;
        const int h = (lr >> 2) | ((g & 1) << 2);
        const char* a = s + (ks * 32 + 8 * g + (lr >> 2)) * RB + (lr & 3) * 8 + ((t ^ h) << 5);
        const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4p)a), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4p)(a + 4 * RB));
        const uint2 x = __builtin_bit_cast(uint2, lo), y = __builtin_bit_cast(uint2, hi);
        return make_uint4(x.x, x.y, y.x, y.y);
    }
};

// over the 16 lanes that share lane >> 4, four values side by side: a sum's result can be moved across lanes three instructions later
__device__ __forceinline__ void row16_sum(float (&v)[4]) {
#define ROW16(ctrl)                                                                                                                             \
    _Pragma("unroll") for (int r = 0; r < 4; ++r) v[r] +=                                                                                       \
        __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v[r]), ctrl, 0xf, 0xf, true));
    ROW16(0x128) ROW16(0x124) ROW16(0x122) ROW16(0x121)
#undef ROW16
}

// The scores' products (short k, long epilogue) are persistent: a workgroup takes every gridDim-th tile, and the DMA runs two k-tiles
// ahead across the border of two tiles, so that the next tile's operands arrive under this one's epilogue.  Lane (g, lr) of wave
// (wi, wj) ends up with Out[j][i] at j = j0 + (wj TJ + y) 16 + lr, i = i0 + (wi TI + x) 16 + 4 g + r in register r of accumulator (x, y).
// X3: operands of three planes.
// A fragment read feeds TJ (TI) products and the barrier stands once a k-tile, so the 256-wide tile waits for the matrix pipes, not for
// LDS: 4096^3 at 1200 TF/s with both operands stored along k, 1205 with both transposed (library product: 1300).
template <bool X3, bool AKC, bool BKC, int MODE, int WI, int WJ, int TI, int TJ>
__global__ __launch_bounds__(64 * WI * WJ, 2) void ce_gemm_kernel(const CeArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)   // the host pass needs the launch stub only, and cannot form the LDS builtins
    constexpr int NW = WI * WJ, IT = WI * TI * 16, JT = WJ * TJ * 16;
    constexpr bool OPQ = !AKC && !BKC, ROWS_K = MODE == OUT || MODE == PART, SCORES = MODE == STATS || MODE == DZ;
    constexpr bool MORE = SCORES;   // more than one tile a workgroup
    static_assert(64 * NW >= IT && 64 * NW >= JT, "a thread a column and a row of the tile");
    constexpr int PL = X3 ? 3 : 1, KE = X3 ? 32 : 64;   // planes of an operand; k of a k-tile
    using TA = Tile<AKC, IT, NW, KE>;
    using TB = Tile<BKC, JT, NW, KE>;
    // two stages of either operand, each a variable of its own: what the compiler can tell apart it does not make a read wait for
    __shared__ __attribute__((aligned(1024))) char sa0[PL * TA::BYTES];
    __shared__ __attribute__((aligned(1024))) char sa1[PL * TA::BYTES];
    __shared__ __attribute__((aligned(1024))) char sb0[PL * TB::BYTES];
    __shared__ __attribute__((aligned(1024))) char sb1[PL * TB::BYTES];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = wave % WI, wj = wave / WI, g = lane >> 4, lr = lane & 15;
    const int n = __builtin_amdgcn_readfirstlane(*p.n);   // in a scalar register, like all that the tile loop counts by
    const int J = ROWS_K ? p.J : min(p.J, n), K = ROWS_K ? min(p.K, n) : p.K;
    const int tiles_i = (p.I + IT - 1) / IT, tiles_j = (J + JT - 1) / JT, tiles = tiles_i * tiles_j * p.splits;
    const int kt_all = (K + KE - 1) / KE, per_split = (kt_all + p.splits - 1) / p.splits;

    // Tile order: runs of 8 j-tiles against one i-tile.  An XCD's workgroups take neighbours, which share operands in its L2.
    struct At { int i0, j0, it, jt, split; };
    auto at = [&](int id) __attribute__((always_inline)) {
        At t;
        int ti = tiles_i, tj = tiles_j;
        asm volatile("" : "+s"(ti), "+s"(tj));   // the divisions' reciprocals are not kept in registers across the k-loop
        t.split = 0;
        if constexpr (!SCORES) {
            t.split = id / (ti * tj);
            id -= t.split * ti * tj;
        }
        const int per = 8 * ti, grp = id / per, in = id - grp * per, gj = min(8, tj - grp * 8);
        t.it = in / gj;
        t.jt = grp * 8 + in - t.it * gj;
        t.i0 = t.it * IT;
        t.j0 = t.jt * JT;
        return t;
    };
    // k-tiles of a tile: an even number, so that every tile begins in the same stage; those behind its share of k read zeros
    const int kts = (max(1, min(per_split, kt_all)) + 1) & ~1;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    if (id >= tiles) return;
    TA ta;
    TB tb;
    ta.init(wave, lane, p.lda);
    tb.init(wave, lane, p.ldb);
    constexpr int NP = PL * (TA::NI + TB::NI);
    // Where the DMA is: the next k-tile to fetch, `fin` k-tiles into a tile.  It runs on into the workgroup's next tile.
    struct Slab { const char *pa, *pb; int left, ra, rb; };   // slabs; k left; rows (columns) of the tile that exist
    Slab f, fnext;
    int fin = 0;
    auto enter = [&](int id) __attribute__((always_inline)) {
        Slab f;
        const At t = at(id);
        const int kt0 = min(t.split * per_split, kt_all);
        f.pa = TA::slab(p.A, p.lda, t.i0, (long)kt0 * KE);
        f.pb = TB::slab(p.B, p.ldb, t.j0, (long)kt0 * KE);
        f.left = min(K, (kt0 + per_split) * KE) - kt0 * KE;
        f.ra = min(IT, p.I - t.i0);
        f.rb = min(JT, J - t.j0);
        return f;
    };
    auto advance = [&] __attribute__((always_inline)) {
        // choices by masks: a branch in the k-loop splits the blocks that its registers are planned over, and they spill
        f.pa += TA::step(p.lda);
        f.pb += TB::step(p.ldb);
        f.left -= KE;
        if constexpr (MORE) {
            const long m = -(long)(++fin == kts);
            auto sel = [&](auto a, auto b) { return (decltype(a))(((long)b & m) | ((long)a & ~m)); };
            f.pa = sel(f.pa, fnext.pa);
            f.pb = sel(f.pb, fnext.pb);
            f.left = sel(f.left, fnext.left);
            f.ra = sel(f.ra, fnext.ra);
            f.rb = sel(f.rb, fnext.rb);
            fin &= ~(int)m;
        }
    };
    // the DMA, two k-tiles ahead, leaves tile r for r + 1 while r is multiplied, and r + 1 for r + 2 where a tile is two k-tiles
    auto follow = [&](int id) __attribute__((always_inline)) {
        const bool more = id < tiles;
        fnext = enter(more ? id : 0);
        fnext.left = more ? fnext.left : 0;   // no such tile: nothing is fetched
    };
    f = enter(id);
    follow(id + gridDim.x);
    auto issue = [&](const Slab& t, char* sa, char* sb, int q) __attribute__((always_inline)) {   // DMA instruction q
        constexpr int NA = PL * TA::NI;
        if (q < NA) ta.issue(t.pa + q / TA::NI * p.plane_a, sa + q / TA::NI * TA::BYTES, wave, t.left, q % TA::NI, p.lda, t.ra);
        else tb.issue(t.pb + (q - NA) / TB::NI * p.plane_b, sb + (q - NA) / TB::NI * TB::BYTES, wave, t.left, (q - NA) % TB::NI, p.ldb, t.rb);
    };
    int lr_k = lr, g_k = g;
    auto rd_a = [&](const char* s, int x, int ks, int plane = 0) __attribute__((always_inline)) {
        return TA::read(s + plane * TA::BYTES, wi * TI + x, ks, g_k, lr_k);
    };
    auto rd_b = [&](const char* s, int y, int ks, int plane = 0) __attribute__((always_inline)) {
        return TB::read(s + plane * TB::BYTES, wj * TJ + y, ks, g_k, lr_k);
    };

    f32x4 acc[TI][TJ];
    // A k-step is TI rows of TJ MFMAs.  Behind row x its A fragment is replaced by the next step's (needed TI rows later), the next
    // step's B fragments arrive in a second set during the first rows.  In the second step of a k-tile, behind row 0 -- by then every
    // read of this tile has landed -- the workgroup meets: the other stage is complete, this one is free for the k-tile after next,
    // whose DMA instructions go out between the rows.
    uint4 a[TI], b0[TJ], b1[TJ];
    auto step = [&](const char* na, const char* nb, int ks, uint4 (&bc)[TJ], uint4 (&bn)[TJ], bool meet, char* fa,
                    char* fb) __attribute__((always_inline)) {
        // two transposed operands: their addresses are worked out here; held across the loop they spill (4096^3: 816 against 1100 TF/s)
        if (OPQ) asm volatile("" : "+v"(lr_k), "+v"(g_k));
#pragma unroll
        for (int x = 0; x < TI; ++x) {
#pragma unroll
            for (int y = 0; y < TJ; ++y) mma(a[x], bc[y], acc[x][y]);
            if (meet && x == 0) {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
            __builtin_amdgcn_sched_barrier(0);   // the replaced fragment's registers are taken over, not doubled
            a[x] = rd_a(na, x, ks);
#pragma unroll
            for (int y = 0; y < TJ; ++y)
                if (y / 2 == x) bn[y] = rd_b(nb, y, ks);
            if (meet) {
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    if (q * TI / NP == x) issue(f, fa, fb, q);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (meet) advance();
    };
    // X3: a k-step is the six products of the planes (2, 0) (0, 2) (1, 1) (1, 0) (0, 1) (0, 0).  A plane's fragments are replaced behind its
    // last product -- B's plane 0, wanted to the end, by a second set -- and the workgroup meets behind the first row, as above.
    uint4 a1[TI], a2[TI], q1[TJ], q2[TJ];
    auto step3 = [&](const char* na, const char* nb, uint4 (&bc)[TJ], uint4 (&bn)[TJ], char* fa, char* fb) __attribute__((always_inline)) {
        if (OPQ) asm volatile("" : "+v"(lr_k), "+v"(g_k));
        auto rows = [&](int term, uint4 (&ax)[TI], uint4 (&by)[TJ], auto behind) __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < TI; ++x) {
#pragma unroll
                for (int y = 0; y < TJ; ++y) mma(ax[x], by[y], acc[x][y]);
                if (term == 0 && x == 0) {
                    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                }
                __builtin_amdgcn_sched_barrier(0);
                behind(x);
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    if (q == term * TI + x) issue(f, fa, fb, q);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        static_assert(NP <= 6 * TI, "a DMA instruction a row");
        rows(0, a2, bc, [&](int x) __attribute__((always_inline)) { a2[x] = rd_a(na, x, 0, 2); });
        rows(1, a, q2, [&](int x) __attribute__((always_inline)) {
            if (x == TI - 1) {
#pragma unroll
                for (int y = 0; y < TJ; ++y) q2[y] = rd_b(nb, y, 0, 2);
            }
        });
        rows(2, a1, q1, [&](int x) __attribute__((always_inline)) {
            if (x < TJ) bn[x] = rd_b(nb, x, 0, 0);
        });
        rows(3, a1, bc, [&](int x) __attribute__((always_inline)) { a1[x] = rd_a(na, x, 0, 1); });
        rows(4, a, q1, [&](int x) __attribute__((always_inline)) {
            if (x == TI - 1) {
#pragma unroll
                for (int y = 0; y < TJ; ++y) q1[y] = rd_b(nb, y, 0, 1);
            }
        });
        rows(5, a, bc, [&](int x) __attribute__((always_inline)) { a[x] = rd_a(na, x, 0, 0); });
        advance();
    };
    static_assert(!X3 || TJ <= TI, "B's plane 0 is read a fragment a row");
    auto meet_lds = [&] {   // LDS writes of the epilogue only: the DMA in flight is not waited for
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    // the next tile's first operands, fetched during this one's last steps, are waited for before the epilogue's stores go out behind them
    auto landed = [&] { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };

#pragma unroll
    for (int q = 0; q < NP; ++q) issue(f, sa0, sb0, q);
    advance();
#pragma unroll
    for (int q = 0; q < NP; ++q) issue(f, sa1, sb1, q);
    advance();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    auto first = [&](const char* na, const char* nb) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < TI; ++x) a[x] = rd_a(na, x, 0);
#pragma unroll
        for (int y = 0; y < TJ; ++y) b0[y] = rd_b(nb, y, 0);
        if constexpr (X3) {
#pragma unroll
            for (int x = 0; x < TI; ++x) {
                a1[x] = rd_a(na, x, 0, 1);
                a2[x] = rd_a(na, x, 0, 2);
            }
#pragma unroll
            for (int y = 0; y < TJ; ++y) {
                q1[y] = rd_b(nb, y, 0, 1);
                q2[y] = rd_b(nb, y, 0, 2);
            }
        }
    };
    first(sa0, sb0);
    for (;; id += gridDim.x) {
        if (MORE) follow(id + (kts == 2 ? 2 : 1) * (int)gridDim.x);
#pragma unroll
        for (int x = 0; x < TI; ++x)
#pragma unroll
            for (int y = 0; y < TJ; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
        const At cur = at(id);
        // a thread's column and row of the tile: what the epilogue needs of them, on its way while the products are formed
        float col_b = 0.f, row_base = 0.f, row_w = 0.f, row_s = 0.f;
        int row_t = ROW_BAD;
        if constexpr (SCORES) {
            const int i = cur.i0 + tid, m = cur.j0 + tid;
            if (tid < IT) col_b = i < p.I ? (p.bias ? p.bias[i] : 0.f) : -INFINITY;   // classes that do not exist: masked
            if (tid < JT && m < J) {
                row_t = p.tgt[m] - p.i_base;
                if constexpr (MODE == DZ) {
                    row_base = p.base2[m];
                    row_w = row_t + p.i_base == ROW_BAD ? NAN : p.grad.reduction == LSAM_REDUCE_NONE ? p.grad.gout[p.idx[m]] : 1.f;
                    row_s = row_w / (p.grad.unit * p.sum[m]);
                }
            }
        }
        for (int kt = 0; kt < kts; kt += 2) {
            if constexpr (X3) {
                step3(sa1, sb1, b0, b1, sa0, sb0);
                step3(sa0, sb0, b1, b0, sa1, sb1);
            } else {
                step(sa0, sb0, 1, b0, b1, false, nullptr, nullptr);
                step(sa1, sb1, 0, b1, b0, true, sa0, sb0);
                step(sa1, sb1, 1, b0, b1, false, nullptr, nullptr);
                step(sa0, sb0, 0, b1, b0, true, sa1, sb1);
            }
        }

        // opaque copies: nothing of an epilogue's addresses is worked out ahead of the k-loop, where every register is taken
        int lr_e = lr, g_e = g, tid_e = tid;
        asm volatile("" : "+v"(lr_e), "+v"(g_e), "+v"(tid_e));
        const int i0 = cur.i0, j0 = cur.j0, ib = i0 + wi * TI * 16 + 4 * g_e, jb = j0 + wj * TJ * 16 + lr_e;
        if constexpr (SCORES) {
            __shared__ __attribute__((aligned(16))) float col[IT];   // read four at a time, like red written
            __shared__ float rbase[JT], rw[JT], rs[JT];
            __shared__ int rt[JT];
            __shared__ __attribute__((aligned(16))) float red[MODE == STATS ? WI * 3 * JT : WJ * IT];
            // a class masked with the type's lowest value; -inf and NaN stay what they are
            if (fabsf(col_b) > MASK && fabsf(col_b) != INFINITY) col_b = copysignf(MASK, col_b);
            if (tid_e < IT) col[tid_e] = col_b;
            if (tid_e < JT) {
                rt[tid_e] = row_t;
                if constexpr (MODE == DZ) {
                    rbase[tid_e] = j0 + tid_e < J ? row_base : 3e38f;   // rows that do not exist: exponentials 0
                    rw[tid_e] = row_w;
                    rs[tid_e] = row_s;
                }
            }
            meet_lds();
            if (p.bias || i0 + IT > p.I) {
#pragma unroll
                for (int x = 0; x < TI; ++x) {
                    const f32x4 b = *reinterpret_cast<const f32x4*>(col + (wi * TI + x) * 16 + 4 * g_e);
#pragma unroll
                    for (int y = 0; y < TJ; ++y) acc[x][y] += b;
                }
            }
            if constexpr (MODE == STATS) {
#pragma unroll
                for (int y = 0; y < TJ; ++y) {
                    const int t = rt[(wj * TJ + y) * 16 + lr_e] - ib;   // the target's place among this lane's classes
                    float mx = -INFINITY, zs = 0.f;
#pragma unroll
                    for (int x = 0; x < TI; ++x)
#pragma unroll
                        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[x][y][r]);
                    if (__any(t >= 0 && t < TI * 16)) {
#pragma unroll
                        for (int x = 0; x < TI; ++x)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (16 * x + r == t) p.zt[jb + 16 * y] = acc[x][y][r];
                    }
                    if (p.smooth_z != 0.f) {
                        if (i0 + IT > p.I) {
#pragma unroll
                            for (int x = 0; x < TI; ++x)
#pragma unroll
                                for (int r = 0; r < 4; ++r) zs = fmaf(ib + 16 * x + r < p.I ? acc[x][y][r] : 0.f, Z_SCALE, zs);
                        } else {
#pragma unroll
                            for (int x = 0; x < TI; ++x)
#pragma unroll
                                for (int r = 0; r < 4; ++r) zs = fmaf(acc[x][y][r], Z_SCALE, zs);
                        }
                        zs = group4_sum(zs);
                    }
                    const float base = Base::of(group4_max(mx));
                    Base to(base);
                    if (base == -INFINITY) to.sub = 0.f;   // every class of the tile at -inf: its exponentials are 0
                    float s = 0.f;
#pragma unroll
                    for (int x = 0; x < TI; ++x) {   // four at a time: an exponential's result can be used two instructions later
                        f32x4 e;
#pragma unroll
                        for (int r = 0; r < 4; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(acc[x][y][r], to.mul, -to.sub));
                        s += (e[0] + e[1]) + (e[2] + e[3]);
                    }
                    s = group4_sum(s);
                    if (g_e == 0) {
                        const int c = (wj * TJ + y) * 16 + lr_e;
                        red[(wi * 3 + 0) * JT + c] = base;
                        red[(wi * 3 + 1) * JT + c] = s;
                        red[(wi * 3 + 2) * JT + c] = zs;
                    }
                }
                landed();
                meet_lds();
                if (tid_e < JT && j0 + tid_e < J) {
                    const int c = tid_e;
                    float mx = red[c], s = 0.f, zs = 0.f;
#pragma unroll
                    for (int w = 1; w < WI; ++w) mx = fmaxf(mx, red[w * 3 * JT + c]);
#pragma unroll
                    for (int w = 0; w < WI; ++w) {
                        const float mw = red[w * 3 * JT + c];
                        s += red[(w * 3 + 1) * JT + c] * (mw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mw - mx));
                        zs += red[(w * 3 + 2) * JT + c];
                    }
                    const size_t o = (size_t)cur.it * p.rows_cap + j0 + c, plane = (size_t)tiles_i * p.rows_cap;
                    p.part[o] = mx;
                    p.part[plane + o] = s;
                    if (p.smooth_z != 0.f) p.part[2 * plane + o] = zs;
                }
            } else {
                bf16* out = static_cast<bf16*>(p.out);
#pragma unroll
                for (int y = 0; y < TJ; ++y) {
                    const int c = (wj * TJ + y) * 16 + lr_e, m = j0 + c;
                    const bool ok = m < J;
                    const Base to(rbase[c]);
                    const float w = rw[c], cs = rs[c], low = -w * p.sm;
                    const int t = rt[c] - ib;
#pragma unroll
                    for (int x = 0; x < TI; ++x)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[x][y][r] = fmaf(__builtin_amdgcn_exp2f(fmaf(acc[x][y][r], to.mul, -to.sub)), cs, low);
                    if (__any(t >= 0 && t < TI * 16)) {
#pragma unroll
                        for (int x = 0; x < TI; ++x)
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[x][y][r] -= 16 * x + r == t ? w * p.keep : 0.f;
                    }
                    if (y == 0) landed();
                    bf16* rowp = out + (size_t)(ok ? m : 0) * p.ldo + i0 + wi * TI * 16;
#pragma unroll
                    for (int x = 0; x < TI; x += 2) {
                        store_bf16_tile_pair(rowp + 16 * x, g_e, acc[x][y], acc[x + 1][y], ok);
                        if constexpr (X3) {
                            f32x4 u = acc[x][y], v = acc[x + 1][y];
#pragma unroll
                            for (int q = 1; q < 3; ++q) {
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    u[r] -= (float)(bf16)u[r];
                                    v[r] -= (float)(bf16)v[r];
                                }
                                store_bf16_tile_pair(rowp + q * (p.plane_out / 2) + 16 * x, g_e, u, v, ok);
                            }
                        }
                    }
                }
                if (p.dbp) {
#pragma unroll
                    for (int x = 0; x < TI; ++x) {
                        float s[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            s[r] = acc[x][0][r];
#pragma unroll
                            for (int y = 1; y < TJ; ++y) s[r] += acc[x][y][r];
                        }
                        row16_sum(s);
                        if (lr_e == 0) *reinterpret_cast<f32x4*>(red + wj * IT + (wi * TI + x) * 16 + 4 * g_e) = f32x4{s[0], s[1], s[2], s[3]};
                    }
                    meet_lds();
                    if (tid_e < IT && i0 + tid_e < p.I) {
                        float s = 0.f;
#pragma unroll
                        for (int w = 0; w < WJ; ++w) s += red[w * IT + tid_e];
                        p.dbp[(size_t)cur.jt * p.dbp_ld + i0 + tid_e] = s;
                    }
                }
            }
        } else {
            const float f = MODE == OUT ? p.grad.factor(n) : 1.f;
#pragma unroll
            for (int y = 0; y < TJ; ++y) {
                const int j = jb + 16 * y;
                if constexpr (MODE == OUT) {
                    using T = std::conditional_t<X3, float, bf16>;
                    T* row = static_cast<T*>(p.out) + (size_t)min(j, J - 1) * p.ldo;
                    if (!X3 && p.vec) {   // every lane takes part in the exchange of a tile pair
                        bf16* rowp = static_cast<bf16*>(p.out) + (size_t)min(j, J - 1) * p.ldo + i0 + wi * TI * 16;
#pragma unroll
                        for (int x = 0; x < TI; x += 2)
                            store_bf16_tile_pair(rowp + 16 * x, g_e, acc[x][y] * f, acc[x + 1][y] * f, j < J && i0 + (wi * TI + x) * 16 + 8 * g_e < p.I);
                    } else if (j < J) {
#pragma unroll
                        for (int x = 0; x < TI; ++x) {
                            const int i = ib + 16 * x;
                            const f32x4 v = acc[x][y] * f;
                            if (X3 && p.vec) {
                                if (i < p.cols) store4(row + i, v);
                            } else {
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    if (i + r < p.cols) row[i + r] = from_f<T>(v[r]);
                            }
                        }
                    }
                } else {
                    if (j >= J) continue;
#pragma unroll
                    for (int x = 0; x < TI; ++x) {
                        const int i = ib + 16 * x;
                        if (i >= p.I) continue;
                        float* o = static_cast<float*>(p.out) + cur.split * p.split_stride + (size_t)j * p.ldo + i;
                        f32x4 v = acc[x][y] * f;
                        if (MODE == ACC && p.accumulate) v += load4(o);
                        store4(o, v);
                    }
                }
            }
        }
        if (!MORE || id + (int)gridDim.x >= tiles) break;
        if constexpr (MODE == DZ) meet_lds();
        first(sa0, sb0);   // read here: held through the epilogue they cost 48 registers
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing may land in this workgroup's LDS after it
#endif
}

// ---------------------------------------------------------------------------------------------------------------------
// Row selection: the rows whose target is not ignored, in order.  A workgroup takes 8192 rows; with more than one, a first launch counts
// each one's rows and the second adds up those in front of its own.
// ---------------------------------------------------------------------------------------------------------------------
struct CeState {   // what the forward leaves for the backward
    int* n;        // rows that count
    int* idx;      // [M] compact row -> row
    int* pos;      // [M] row -> compact row, -1 where ignored
    int* tgt;      // [M] compact; ROW_BAD outside [0, V)
    float* base2;  // [M] compact: lse = base2 / log2(e) + ln(sum), or base2 / 2 + ln(sum) where |base2| > FAR_BASE
    float* sum;
    char* xc;      // bf16 [M][Dp] compact rows, columns padded with zeros; fp32: three planes
};

constexpr int ROWS_WG = 8192;

__global__ __launch_bounds__(1024) void ce_count_kernel(const long long* __restrict__ target, int M, long long ignore, int* __restrict__ counts) {
    __shared__ int wsum[16];
    const int tid = threadIdx.x, b = blockIdx.x * ROWS_WG;
    int cnt = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int m = b + j * 1024 + tid;
        cnt += __popcll(__ballot(m < M && target[m < M ? m : M - 1] != ignore));
    }
    if ((tid & 63) == 0) wsum[tid >> 6] = cnt;
    __syncthreads();
    if (tid == 0) {
        int s = 0;
        for (int w = 0; w < 16; ++w) s += wsum[w];
        counts[blockIdx.x] = s;
    }
}

// Rows of `src` (through idx, or all of them) to bf16 [rows][Dp], columns D.. filled with zeros; fp32 to three planes, `plane` elements apart.
template <typename T> struct Gather {
    const T* src; long ld;
    const int* idx;
    int D, Dp, vec;
    bf16* dst; long plane;
    __device__ __forceinline__ void run(int rows, long first, long step) const {
        const int cpr = Dp / 8;
        for (long id = first; id < (long)rows * cpr; id += step) {
            const int r = (int)(id / cpr), c = (int)(id - (long)r * cpr) * 8;
            const T* s = src + (idx ? idx[r] : r) * ld + c;
            T e[8];
            if (vec) __builtin_memcpy(e, __builtin_assume_aligned(s, 16), sizeof(e));
            else {
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = c + j < D ? s[j] : from_f<T>(0.f);
            }
            bf16* o = dst + (size_t)r * Dp + c;
#pragma unroll
            for (int q = 0; q < (sizeof(T) == 4 ? 3 : 1); ++q) {
                bf16x8 v;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] = (bf16)e[j];
                    if constexpr (sizeof(T) == 4) e[j] -= (float)v[j];
                }
                *reinterpret_cast<bf16x8*>(o + q * plane) = v;
            }
        }
    }
};
template <typename T> __global__ __launch_bounds__(256) void ce_gather_kernel(const Gather<T> g, const int* __restrict__ n, int rows) {
    g.run(n ? min(rows, *n) : rows, (long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256);
}

// `take`: the one workgroup gathers the rows too
template <typename T>
__global__ __launch_bounds__(1024) void ce_rows_kernel(const long long* __restrict__ target, int M, int V, long long ignore, CeState st,
                                                       const int* __restrict__ counts, float* __restrict__ loss_none, int take, const Gather<T> g) {
    __shared__ int part[8][16], front[8 * 16], before;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x * ROWS_WG;
    if (wave == 0) {   // rows that count in front of this workgroup's
        int s = 0;
        for (int i = lane; i < (int)blockIdx.x; i += 64) s += counts[i];
        for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
        if (lane == 0) before = s;
    }
    long long t[8];
    unsigned long long mask[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int m = b + j * 1024 + tid;
        t[j] = m < M ? target[m] : ignore;
        mask[j] = __ballot(t[j] != ignore);
        if (lane == 0) part[j][wave] = __popcll(mask[j]);
    }
    __syncthreads();
    if (wave == 0) {   // exclusive sums over the 128 groups of 64 rows
        const int a = (&part[0][0])[2 * lane], c = (&part[0][0])[2 * lane + 1];
        int inc = a + c;
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(inc, o);
            if (lane >= o) inc += v;
        }
        front[2 * lane] = inc - a - c;
        front[2 * lane + 1] = inc - c;
        if (lane == 63 && blockIdx.x == gridDim.x - 1) *st.n = before + inc;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int m = b + j * 1024 + tid;
        if (m >= M) continue;
        if (t[j] != ignore) {
            const int r = before + front[j * 16 + wave] + __popcll(mask[j] & ((1ull << lane) - 1));
            st.idx[r] = m;
            st.tgt[r] = t[j] >= 0 && t[j] < V ? (int)t[j] : ROW_BAD;
            st.pos[m] = r;
        } else {
            st.pos[m] = -1;
            if (loss_none) loss_none[m] = 0.f;
        }
    }
    if (take) {
        __syncthreads();
        g.run(before + front[127] + part[7][15], tid, 1024);
    }
}

// 16 rows a workgroup, 64 threads a row: joins the tiles' (base, sum) pairs; the loss of the row.  With one workgroup the sum over
// the rows too.  The logarithm of the sum and the target's score are subtracted in 64 bits: a learned row's loss is their small difference.
__global__ __launch_bounds__(1024) void ce_loss_kernel(const float* __restrict__ part, const float* __restrict__ zt, int tiles, int cap, int V,
                                                       float smooth, CeState st, float* __restrict__ row_loss, float* __restrict__ loss,
                                                       int reduction) {
    __shared__ float sb[64][17], ss[64][17], sz[64][17];
    __shared__ double sl[16];
    const int tid = threadIdx.x, c = tid & 15, sl_ = tid >> 4, n = *st.n;
    const int r = blockIdx.x * 16 + c;
    const size_t plane = (size_t)tiles * cap;
    float b = -INFINITY, s = 0.f, z = 0.f;
    if (r < n) {
        for (int t = sl_; t < tiles; t += 64) {
            const size_t o = (size_t)t * cap + r;
            const float bt = part[o], v = part[plane + o];
            const float nb = fmaxf(b, bt);
            s = (b == -INFINITY ? s : s * exp2f(b - nb)) + (bt == -INFINITY ? v : v * exp2f(bt - nb));
            b = nb;
            if (smooth != 0.f) z += part[2 * plane + o];
        }
    }
    sb[sl_][c] = b; ss[sl_][c] = s; sz[sl_][c] = z;
    __syncthreads();
    if (tid < 16) {
        double out = 0.;
        if (r < n) {
            float B = -INFINITY, S = 0.f, Z = 0.f;
            for (int k = 0; k < 64; ++k) B = fmaxf(B, sb[k][c]);
            for (int k = 0; k < 64; ++k) {
                S += ss[k][c] * (sb[k][c] == -INFINITY ? 1.f : exp2f(sb[k][c] - B));
                Z += sz[k][c];
            }
            st.base2[r] = B;
            st.sum[r] = S;
            const double L = (double)LOG2E, top = fabsf(B) > FAR_BASE ? 0.5 * (double)B : (double)B / L, rest = log2((double)S) / L;
            if (st.tgt[r] == ROW_BAD) out = (double)NAN;
            else out = (top - (double)zt[r] + rest) * (1. - (double)smooth) + (smooth != 0.f ? (double)smooth * (top - (double)Z / Z_SCALE / V + rest) : 0.);
            if (reduction == LSAM_REDUCE_NONE) loss[st.idx[r]] = (float)out;
            else row_loss[r] = (float)out;
        }
        sl[c] = out;
    }
    if (gridDim.x == 1 && reduction != LSAM_REDUCE_NONE) {
        __syncthreads();
        if (tid == 0) {
            double a = 0.;
            for (int k = 0; k < 16; ++k) a += sl[k];
            loss[0] = (float)(reduction == LSAM_REDUCE_MEAN ? a / (double)n : a);
        }
    }
}

__global__ __launch_bounds__(1024) void ce_sum_kernel(const float* __restrict__ row_loss, const int* __restrict__ np, float* __restrict__ loss,
                                                      int reduction) {
    __shared__ double part[1024];
    const int n = *np;
    double a = 0.;
    for (int r = threadIdx.x; r < n; r += 1024) a += (double)row_loss[r];
    part[threadIdx.x] = a;
    __syncthreads();
    for (int o = 512; o; o >>= 1) {
        if ((int)threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) loss[0] = (float)(reduction == LSAM_REDUCE_MEAN ? part[0] / (double)n : part[0]);
}

// out[m] = factor * (sum of the splits' rows), or zeros where the row was ignored; `lanes` threads share a sum of many splits where
// there are few sums (6 x 592 of 512 splits: 4 us, 20 with a thread a sum; 2011 x 252 of 16: 23 and 16).  Workgroups from `first_db` on: the bias gradient, the row tiles'
// column sums in their order.
struct Finish {
    const float* acc; long stride; int splits;
    const int *pos, *n;
    int M, D, Dp;
    Grad grad;
    void* out; long ldo;
    int first_db, V, rows_tile;
    const float* dbp; float* db;
    int lanes;
};
template <typename T> __global__ __launch_bounds__(256) void ce_finish_kernel(const Finish p) {
    __shared__ f32x4 sh[256];
    const int n = *p.n, tid = threadIdx.x;
    const float f = p.grad.factor(n);
    if ((int)blockIdx.x >= p.first_db) {
        const int v = ((int)blockIdx.x - p.first_db) * 256 + tid, tiles = (n + p.rows_tile - 1) / p.rows_tile;
        if (v >= p.V) return;
        float s = 0.f;
#pragma unroll 8
        for (int t = 0; t < tiles; ++t) s += p.dbp[(size_t)t * p.V + v];
        p.db[v] = tiles ? s * f : 0.f;
        return;
    }
    const int cpr = p.Dp / 4, per = 256 / p.lanes, lane = tid / per;
    const long total = (long)p.M * cpr;
    for (long base = (long)blockIdx.x * per; base < total; base += (long)p.first_db * per) {
        const long id = base + tid % per;
        const int m = (int)(id / cpr), c = (int)(id - (long)m * cpr) * 4;
        const bool on = id < total && c < p.D;
        const int r = !on ? -1 : p.pos ? p.pos[m] : m;
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
        if (r >= 0) {
            const float* a = p.acc + (size_t)r * p.Dp + c;
#pragma unroll 4
            for (int s = lane; s < p.splits; s += p.lanes) v += load4(a + s * p.stride);
        }
        if (p.lanes > 1) {
            sh[tid] = v;
            __syncthreads();
            for (int o = p.lanes / 2; o; o >>= 1) {
                if (lane < o) sh[tid] += sh[tid + o * per];
                __syncthreads();
            }
            v = sh[tid % per];
            __syncthreads();
        }
        if (!on || lane) continue;
        v *= f;
        T* o = static_cast<T*>(p.out) + (size_t)m * p.ldo + c;
        if (p.D % 4 == 0 && p.ldo % 4 == 0) store4(o, v);
        else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < p.D) o[j] = from_f<T>(v[j]);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------
// A piece's dz.  16384 x 256 x 32000 in all: 1560 us with 256 MB (what the last-level cache holds), 1475 with 512, 1337 with 1024: fewer
// passes over the fp32 sums of dx weigh more than where dz is read from.  A piece has 256 classes at least: beyond 0.7 M rows in fp32 and
// 2.1 M in bf16 that is more than this many bytes (512 or 1536 a row).
constexpr size_t DZ_CAP = (size_t)1 << 30;
constexpr int CU = 256;

struct Carve {
    char* p;
    size_t used = 0;
    template <typename U> U* take(size_t n) {
        U* r = reinterpret_cast<U*>(p + used);
        used += align_up(n * sizeof(U), 256);
        return p ? r : nullptr;
    }
};

// Tiles of 256 x 256 (8 waves of 128 x 64 or 64 x 128, one workgroup a CU) or 128 x 128 (64 x 32, two a CU).  The large one feeds the
// matrix pipes from LDS at close to their rate; the small one balances where the large leaves CUs idle.  Rounds of tiles, a small one
// costed at a quarter of a large one and half as much again (16384 x 256 x 32000 scores: 440 us against 364; weight gradient of
// 8192 x 896 x 50257: 769 against 644).  fp32: 256 x 128 (64 x 64 a wave) or 128 x 128, one workgroup a CU, a small one costed at half a
// large one and a fifth more (scores of 2011 x 252 x 10007: 64 against 66 us, of 4096 x 512 x 4096: 96 against 86).
constexpr double SMALL = 1.5, SMALL3 = 1.2;
template <typename T> struct CePlan {
    static constexpr bool X3 = sizeof(T) == 4;
    static constexpr int ES = X3 ? 6 : 2;   // bytes a value of the operands takes
    static constexpr int JL = X3 ? 128 : 256;   // rows of a large tile: three planes of 256 x 128 fill the LDS
    int M, D, V, Dp, tile_m, tiles_v, tiles_m;   // tile_m: rows of the scores' tiles
    bool pack_w, small, dx_small, dw_small;
    int piece, s_dx, s_dw;
    CePlan(int M_, int D_, int V_, bool pack) : M(M_), D(D_), V(V_), pack_w(pack) {
        Dp = (D + 7) / 8 * 8;
        const int m = M > 0 ? M : 1;
        small = smaller((long)cdiv(V, 256) * cdiv(m, JL), 1, (long)cdiv(V, 128) * cdiv(m, 128), 1);
        tile_m = small ? 128 : JL;
        tiles_v = cdiv(V, small ? 128 : 256);
        tiles_m = cdiv(m, tile_m);
        const size_t col = (size_t)m * ES * 256;
        size_t pt = DZ_CAP / col;
        if (pt < 1) pt = 1;
        if (pt > 1024) pt = 1024;   // byte offsets within a tile's rows stay within 31 bits
        const int vt = cdiv(V, 256);
        if (pt > (size_t)vt) pt = vt;
        piece = (int)pt * 256;
        // the other two products: the work of a CU is its rounds of tiles times their share of k
        auto pick = [&](int rows, int k, bool& small, int& cuts) {
            const long big = (long)cdiv(rows, Dp <= 128 ? 256 : JL) * cdiv(Dp, 256), lit = (long)cdiv(rows, 128) * cdiv(Dp, 128);
            const int sb = splits(big, k, false), sl = splits(lit, k, true);
            small = smaller(big, sb, lit, sl);
            cuts = small ? sl : sb;
        };
        pick(m, piece, dx_small, s_dx);
        pick(piece, m, dw_small, s_dw);
    }
    static bool smaller(long big, int sb, long lit, int sl) {   // tiles, cuts of k
        return (double)((big * sb + CU - 1) / CU) * (X3 ? 2 : 4) / sb > (X3 ? SMALL3 : SMALL) * (double)((lit * sl + CU - 1) / CU) / sl;
    }
    int splits(long tiles, int k, bool small) const {   // cuts of k that keep the CUs busy, at least four k-tiles (or six terms) each
        const int slots = small && !X3 ? 2 * CU : CU, least = X3 ? 64 : 256, most = k / least > 0 ? k / least : 1;
        const long s = tiles >= slots ? 1 : slots / tiles;
        return (int)(s < most ? s : most);
    }
    // Several rounds of the weight gradient's large tiles with the last one less than half full: the classes of that one go apart, their
    // k cut (8192 x 896 x 50257: 788 tiles on 256 CUs).  How many of nv classes do.
    int rest(int nv) const {
        const int td = cdiv(Dp, 256), vt = cdiv(nv, 256), over = vt * td % CU;
        if (X3 || dw_small || dw_f32() || vt * td <= CU || over == 0 || over >= CU / 2) return 0;
        const int rt = cdiv(over, td);
        return splits((long)rt * td, M, false) > 1 ? nv - (vt - rt) * 256 : 0;
    }
    bool dw_f32() const { return s_dw > 1; }   // partial sums: through fp32 and the joining kernel
    size_t dw_floats() const {   // the rest's tiles times cuts: at most CU of 65536
        return dw_f32() ? (size_t)s_dw * piece * Dp : !X3 && piece / 256 * cdiv(Dp, 256) > CU ? (size_t)CU * 65536 : 0;
    }
    size_t state(char* base, CeState* st) const {
        Carve c{base};
        CeState s;
        s.n = c.take<int>(1);
        s.idx = c.take<int>(M);
        s.pos = c.take<int>(M);
        s.tgt = c.take<int>(M);
        s.base2 = c.take<float>(M);
        s.sum = c.take<float>(M);
        s.xc = c.take<char>((size_t)M * Dp * ES);
        if (st) *st = s;
        return c.used;
    }
    struct Fwd { char* wp; float *part, *zt, *row_loss; int* counts; };
    size_t fwd(char* base, Fwd* f, bool smooth) const {
        Carve c{base};
        Fwd w;
        w.wp = c.take<char>(pack_w ? (size_t)V * Dp * ES : 0);
        w.part = c.take<float>((size_t)tiles_v * M * (smooth ? 3 : 2));
        w.zt = c.take<float>(M);
        w.row_loss = c.take<float>(M);
        w.counts = c.take<int>(M / ROWS_WG + 1);
        if (f) *f = w;
        return c.used;
    }
    struct Bwd { char *wp, *dz; float *dx, *dw, *dbp; };
    size_t bwd(char* base, Bwd* f, bool want_dx, bool want_dw, bool want_db) const {
        Carve c{base};
        Bwd w;
        w.wp = c.take<char>(pack_w ? (size_t)V * Dp * ES : 0);
        w.dz = c.take<char>((size_t)M * piece * ES);
        w.dx = c.take<float>(want_dx ? (size_t)s_dx * M * Dp : 0);
        w.dw = c.take<float>(want_dw ? dw_floats() : 0);
        w.dbp = c.take<float>(want_db ? (size_t)tiles_m * V : 0);
        if (f) *f = w;
        return c.used;
    }
};

template <bool X3, bool AKC, bool BKC, int MODE, int WI, int WJ, int TI, int TJ> int ce_gemm_run(const CeArgs& a, int a_cu, hipStream_t s) {
    constexpr int IT = WI * TI * 16, JT = WJ * TJ * 16;
    const long tiles = (long)cdiv(a.I, IT) * cdiv(a.J, JT) * a.splits, most = (long)CU * a_cu;
    const int wgs = (int)(tiles < most || !(MODE == STATS || MODE == DZ) ? tiles : most);
    ce_gemm_kernel<X3, AKC, BKC, MODE, WI, WJ, TI, TJ><<<wgs, 64 * WI * WJ, 0, s>>>(a);
    LSAM_LAUNCH_CHECK();
    return LSAM_OK;
}
// wave grids of the large tile: as many fragments of the operand that is cheaper to read.  4096^3: A transposed 64 x 128 waves 1333 TF/s
// against 1177 with 128 x 64; both transposed 1205 against 1103 the other way round
template <bool X3, bool AKC, bool BKC, int MODE> int ce_gemm(const CeArgs& a, bool small, hipStream_t s) {
    if (small) return ce_gemm_run<X3, AKC, BKC, MODE, 2, 4, 4, 2>(a, X3 ? 1 : 2, s);
    if constexpr (X3 && (!(MODE == STATS || MODE == DZ)))
        if (a.I <= 128)   // narrow rows: 128 x 256.  8000 x 128 x 8000: dx 146 us, dW 132; with 128 x 128 tiles 199 and 170
            return ce_gemm_run<X3, AKC, BKC, MODE, 2, 4, 4, 4>(a, 1, s);
    if constexpr (X3) return ce_gemm_run<X3, AKC, BKC, MODE, 4, 2, 4, 4>(a, 1, s);
    else
    if constexpr (!AKC && BKC) return ce_gemm_run<X3, AKC, BKC, MODE, 4, 2, 4, 8>(a, 1, s);
    else return ce_gemm_run<X3, AKC, BKC, MODE, 2, 4, 8, 4>(a, 1, s);
}

template <typename T> bool rows_aligned(const void* p, long ld, int D) { return D % 8 == 0 && ld % (16 / (int)sizeof(T)) == 0 && aligned16(p); }
template <typename T> bool rows_direct(const void* p, long ld, int D) {   // rows that the DMA can fetch in place
    return sizeof(T) == 2 && rows_aligned<T>(p, ld, D) && ld < (1l << 20);
}

template <typename T> Gather<T> gather_of(const void* src, long ld, const int* idx, int rows, int D, int Dp, void* dst) {
    return {static_cast<const T*>(src), ld, idx, D, Dp, rows_aligned<T>(src, ld, D), static_cast<bf16*>(dst), (long)rows * Dp};
}
template <typename T> int gather(const Gather<T>& g, const int* n, int rows, hipStream_t s) {
    const long blocks = ((long)rows * (g.Dp / 8) + 255) / 256;
    ce_gather_kernel<T><<<(int)(blocks < 8192 ? blocks : 8192), 256, 0, s>>>(g, n, rows);
    LSAM_LAUNCH_CHECK();
    return LSAM_OK;
}
}  // namespace

int ce_check(int M, int D, int V, int reduction, float smooth) {
    LSAM_REQUIRE(M >= 0 && D > 0 && V > 0, LSAM_ERR_BAD_ARG, "linear_ce: %d rows, %d columns, %d classes", M, D, V);
    // launches stay below 2^32 threads (64 a row in the loss's kernel, 512 a tile of dx): the runtime cuts a longer one short without an error
    LSAM_REQUIRE(M <= (1 << 26) - 16 && V <= (1 << 28) && D <= (1 << 18) && (long)cdiv(M, 128) * cdiv(D, 128) < (1l << 23),
                 LSAM_ERR_UNSUPPORTED, "linear_ce: %d rows, %d columns, %d classes", M, D, V);
    LSAM_REQUIRE(((long)M / 128 + 1) * ((long)V / 128 + 1) < (1l << 30), LSAM_ERR_UNSUPPORTED, "linear_ce: %d rows x %d classes", M, V);
    LSAM_REQUIRE(reduction >= 0 && reduction <= 2, LSAM_ERR_BAD_ARG, "linear_ce: reduction %d", reduction);
    LSAM_REQUIRE(smooth >= 0.f && smooth <= 1.f, LSAM_ERR_BAD_ARG, "linear_ce: label smoothing %g outside [0, 1]", (double)smooth);
    return LSAM_OK;
}

template <typename T> size_t ce_state_bytes(int M, int D) { return CePlan<T>(M, D, 1, false).state(nullptr, nullptr); }
template <typename T> size_t ce_ws_bytes(int M, int D, int V, const void* w, long ldw, float smooth, int grads) {
    const CePlan<T> pl(M, D, V, !rows_direct<T>(w, ldw, D));
    const size_t n = grads ? pl.bwd(nullptr, nullptr, grads & 1, grads & 2, grads & 4) : pl.fwd(nullptr, nullptr, smooth != 0.f);
    return n ? n : 256;   // without rows nothing is kept there, but the pointer is wanted
}

template <typename T>
int launch_linear_ce_fwd(const void* x, long ldx, const void* w, long ldw, const float* bias, const long long* target, int M, int D, int V,
                         long long ignore, float smooth, int reduction, float* loss, void* state, void* ws, size_t ws_bytes, hipStream_t s) {
    LSAM_TRY(ce_check(M, D, V, reduction, smooth));
    constexpr bool X3 = CePlan<T>::X3;
    const CePlan<T> pl(M, D, V, !rows_direct<T>(w, ldw, D));
    LSAM_REQUIRE((M == 0 || (x && target)) && w && state && ws && (loss || (M == 0 && reduction == LSAM_REDUCE_NONE)), LSAM_ERR_BAD_ARG,
                 "linear_ce: null operand");
    LSAM_REQUIRE(ldx >= D && ldw >= D && aligned16(state) && aligned16(ws), LSAM_ERR_BAD_ARG,
                 "linear_ce: row strides %ld, %ld below %d columns, or a workspace off its 16-byte alignment", ldx, ldw, D);
    CeState st;
    typename CePlan<T>::Fwd f;
    pl.state(static_cast<char*>(state), &st);
    LSAM_REQUIRE(pl.fwd(static_cast<char*>(ws), &f, smooth != 0.f) <= ws_bytes, LSAM_ERR_WORKSPACE, "linear_ce: workspace too small");
    const int wgs = M > 0 ? cdiv(M, ROWS_WG) : 1;
    if (wgs > 1) {
        ce_count_kernel<<<wgs, 1024, 0, s>>>(target, M, ignore, f.counts);
        LSAM_LAUNCH_CHECK();
    }
    const Gather<T> gx = gather_of<T>(x, ldx, st.idx, M, D, pl.Dp, st.xc);
    const bool take = wgs == 1 && (long)M * pl.Dp <= 32768;   // a launch less; a CU copies 64 KB in that time
    ce_rows_kernel<T><<<wgs, 1024, 0, s>>>(target, M, V, ignore, st, f.counts, reduction == LSAM_REDUCE_NONE ? loss : nullptr, take, gx);
    LSAM_LAUNCH_CHECK();
    if (M > 0) {
        if (!take) LSAM_TRY(gather<T>(gx, st.n, M, s));
        if (pl.pack_w) LSAM_TRY(gather<T>(gather_of<T>(w, ldw, nullptr, V, D, pl.Dp, f.wp), nullptr, V, s));
        CeArgs a{};
        a.A = pl.pack_w ? f.wp : w; a.lda = pl.pack_w ? pl.Dp : ldw;
        a.B = st.xc; a.ldb = pl.Dp;
        a.I = V; a.J = M; a.K = pl.Dp; a.n = st.n;
        a.bias = bias; a.tgt = st.tgt; a.smooth_z = smooth; a.part = f.part; a.zt = f.zt; a.rows_cap = M; a.splits = 1;
        a.plane_a = (long)V * pl.Dp * 2; a.plane_b = (long)M * pl.Dp * 2;
        LSAM_TRY((ce_gemm<X3, true, true, STATS>(a, pl.small, s)));
    }
    const int blocks = M > 0 ? cdiv(M, 16) : 1;
    if (M > 0 || reduction != LSAM_REDUCE_NONE) {
        ce_loss_kernel<<<blocks, 1024, 0, s>>>(f.part, f.zt, pl.tiles_v, M, V, smooth, st, f.row_loss, loss, reduction);
        LSAM_LAUNCH_CHECK();
    }
    if (blocks > 1 && reduction != LSAM_REDUCE_NONE) {
        ce_sum_kernel<<<1, 1024, 0, s>>>(f.row_loss, st.n, loss, reduction);
        LSAM_LAUNCH_CHECK();
    }
    return LSAM_OK;
}

template <typename T>
int launch_linear_ce_bwd(const void* w, long ldw, const float* bias, const float* gout, int M, int D, int V, float smooth, int reduction,
                         const void* state, void* dx, long lddx, void* dw, long lddw, float* db, void* ws, size_t ws_bytes, hipStream_t s) {
    LSAM_TRY(ce_check(M, D, V, reduction, smooth));
    constexpr bool X3 = CePlan<T>::X3;
    const CePlan<T> pl(M, D, V, !rows_direct<T>(w, ldw, D));
    LSAM_REQUIRE(w && state && ws && (M == 0 || gout), LSAM_ERR_BAD_ARG, "linear_ce: null operand");
    LSAM_REQUIRE(ldw >= D && (!dx || lddx >= D) && (!dw || lddw >= D) && aligned16(state) && aligned16(ws), LSAM_ERR_BAD_ARG,
                 "linear_ce: a row stride below %d columns, or a workspace off its 16-byte alignment", D);
    LSAM_REQUIRE((!dx || (aligned16(dx) && (lddx % 8 == 0 || D % 8))) && (!dw || (aligned16(dw) && (lddw % 8 == 0 || D % 8))), LSAM_ERR_BAD_ARG,
                 "linear_ce: gradients off their 16-byte alignment");
    CeState st;
    typename CePlan<T>::Bwd b;
    pl.state(static_cast<char*>(const_cast<void*>(state)), &st);
    LSAM_REQUIRE(pl.bwd(static_cast<char*>(ws), &b, dx != nullptr, dw != nullptr, db != nullptr) <= ws_bytes, LSAM_ERR_WORKSPACE,
                 "linear_ce: workspace too small");
    if (pl.pack_w) LSAM_TRY(gather<T>(gather_of<T>(w, ldw, nullptr, V, D, pl.Dp, b.wp), nullptr, V, s));
    const char* W = pl.pack_w ? b.wp : static_cast<const char*>(w);
    const long lw = pl.pack_w ? pl.Dp : ldw;
    const float keep = 1.f - smooth, unit = keep > 0.f ? keep : 1.f;
    const Grad grad{gout, reduction, unit};
    auto finish = [&](const Finish& p, long values) -> int {
        Finish q = p;
        q.lanes = p.splits >= 16 && values / 4 < 32768 ? 16 : 1;
        const long blocks = (values / 4 * q.lanes + 255) / 256;
        q.grad = grad;
        q.n = st.n;
        q.first_db = (int)(blocks < 8192 ? blocks : 8192);
        ce_finish_kernel<T><<<q.first_db + (q.db ? cdiv(V, 256) : 0), 256, 0, s>>>(q);
        LSAM_LAUNCH_CHECK();
        return LSAM_OK;
    };
    for (int v0 = 0, k = 0; v0 < V; v0 += pl.piece, ++k) {
        const int nv = V - v0 < pl.piece ? V - v0 : pl.piece;
        if (M > 0) {
            CeArgs a{};
            a.A = W + (size_t)v0 * lw * 2; a.lda = lw; a.plane_a = (long)V * pl.Dp * 2;
            a.plane_b = (long)M * pl.Dp * 2; a.plane_out = (long)M * pl.piece * 2;
            a.B = st.xc; a.ldb = pl.Dp;
            a.I = nv; a.J = M; a.K = pl.Dp; a.n = st.n;
            a.bias = bias ? bias + v0 : nullptr; a.tgt = st.tgt; a.i_base = v0;
            a.base2 = st.base2; a.sum = st.sum; a.idx = st.idx; a.grad = grad; a.sm = smooth / ((float)V * unit); a.keep = keep / unit;
            a.dbp = db ? b.dbp + v0 : nullptr; a.dbp_ld = V;
            a.out = b.dz; a.ldo = pl.piece; a.splits = 1;
            LSAM_TRY((ce_gemm<X3, true, true, DZ>(a, pl.small, s)));
        }
        if (dx && M > 0) {
            CeArgs a{};
            a.A = W + (size_t)v0 * lw * 2; a.lda = lw; a.plane_a = (long)V * pl.Dp * 2; a.plane_b = (long)M * pl.piece * 2;
            a.B = b.dz; a.ldb = pl.piece;
            a.I = pl.Dp; a.J = M; a.K = nv; a.n = st.n;
            a.out = b.dx; a.ldo = pl.Dp; a.split_stride = (long)M * pl.Dp; a.splits = pl.s_dx; a.accumulate = k > 0;
            LSAM_TRY((ce_gemm<X3, false, true, ACC>(a, pl.dx_small, s)));
        }
        if (dw) {
            // classes c0 .. c0 + nc of the piece; through fp32 where k is cut
            auto weight_grad = [&](int c0, int nc, bool f32, int cuts) -> int {
                T* o = static_cast<T*>(dw) + (size_t)(v0 + c0) * lddw;
                CeArgs a{};
                a.A = st.xc; a.lda = pl.Dp;
                a.B = b.dz + (size_t)c0 * 2; a.ldb = pl.piece; a.plane_a = (long)M * pl.Dp * 2; a.plane_b = (long)M * pl.piece * 2;
                a.I = pl.Dp; a.J = nc; a.K = M; a.n = st.n; a.splits = cuts;
                if (!f32) {
                    a.out = o; a.ldo = lddw; a.grad = grad; a.cols = D;
                    a.vec = X3 ? D % 4 == 0 && lddw % 4 == 0 : D % 8 == 0;
                    return ce_gemm<X3, false, false, OUT>(a, pl.dw_small, s);
                }
                a.out = b.dw; a.ldo = pl.Dp; a.split_stride = (long)nc * pl.Dp;
                LSAM_TRY((ce_gemm<X3, false, false, PART>(a, pl.dw_small, s)));
                return finish(Finish{b.dw, a.split_stride, cuts, nullptr, nullptr, nc, D, pl.Dp, {}, o, lddw, 0, 0, 0, nullptr, nullptr, 1},
                              (long)nc * pl.Dp);
            };
            const int rest = pl.rest(nv);
            LSAM_TRY(weight_grad(0, nv - rest, pl.dw_f32(), pl.s_dw));
            if (rest) LSAM_TRY(weight_grad(nv - rest, rest, true, pl.splits((long)cdiv(rest, 256) * cdiv(pl.Dp, 256), M, false)));
        }
    }
    if ((dx && M > 0) || db)
        LSAM_TRY(finish(Finish{b.dx, (long)M * pl.Dp, pl.s_dx, st.pos, nullptr, dx ? M : 0, D, pl.Dp, {}, dx, lddx, 0, V, pl.tile_m, b.dbp, db, 1},
                        dx ? (long)M * pl.Dp : 0));
    return LSAM_OK;
}
#define CE_INST(T)                                                                                                                          \
    template size_t ce_state_bytes<T>(int, int);                                                                                           \
    template size_t ce_ws_bytes<T>(int, int, int, const void*, long, float, int);                                                          \
    template int launch_linear_ce_fwd<T>(const void*, long, const void*, long, const float*, const long long*, int, int, int, long long,   \
                                         float, int, float*, void*, void*, size_t, hipStream_t);                                           \
    template int launch_linear_ce_bwd<T>(const void*, long, const float*, const float*, int, int, int, float, int, const void*, void*,     \
                                         long, void*, long, float*, void*, size_t, hipStream_t);
CE_INST(float)
CE_INST(bf16)
}  // namespace lsam
