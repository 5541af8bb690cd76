// ung_tiles.h -- tiles of a matrix product C[m][n] = sum_k A[m][k] B[n][k] on gfx950's matrix
// instructions, shared by the operators that make one (ung_int8.hip, ung_table_loss.hip); what
// becomes of a tile's sums is the operator's own (its `Finish`).  Not part of the public ABI.
//
// The inner length is taken in chunks of 128 bytes of a row: 128 8-bit whole numbers, 64 16-bit
// or 32 32-bit numbers.  A matrix instruction takes 16 bytes a lane in each of these types, so
// panels, fragments and loads are the same for all of them.
#pragma once

#include "ung_elements.h"

namespace ung {

using i32x4 = __attribute__((ext_vector_type(4))) int;
using fp16x8 = __attribute__((ext_vector_type(8))) _Float16;

constexpr uint32_t CHUNK = 128; // bytes of the inner length in a panel

// 16 rows of x times 16 rows of y over 64 bytes of the inner length, added to c.  A lane brings
// 16 bytes of row lane % 16 (bytes lane / 16 * 16) of each; of the result it holds row lane % 16 of y
// and rows lane / 16 * 4 + 0..3 of x.
template <class E>
struct Matrix;
template <>
struct Matrix<int8_t> {
    using Acc = i32x4;
    static __device__ inline Acc mul(u32x4 x, u32x4 y, Acc c)
    {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, x), __builtin_bit_cast(i32x4, y), c, 0, 0,
                                                     0);
    }
};
template <>
struct Matrix<bf16_t> {
    using Acc = f32x4;
    static __device__ inline Acc mul(u32x4 x, u32x4 y, Acc c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c,
                                                       0, 0, 0);
    }
};
template <>
struct Matrix<fp16_t> {
    using Acc = f32x4;
    static __device__ inline Acc mul(u32x4 x, u32x4 y, Acc c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(fp16x8, x), __builtin_bit_cast(fp16x8, y), c, 0,
                                                      0, 0);
    }
};
template <>
struct Matrix<float> {
    using Acc = f32x4;
    static __device__ inline Acc mul(u32x4 x, u32x4 y, Acc c)
    {
        const f32x4 a = __builtin_bit_cast(f32x4, x), b = __builtin_bit_cast(f32x4, y);
#pragma unroll
        for (int t = 0; t < 4; ++t)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[t], b[t], c, 0, 0, 0);
        return c;
    }
};

// One side of a product: `rows` rows of `k` elements.  Along the inner length: elements of a row
// lie side by side, rows `stride` bytes apart.  Across it: element k of all rows lies side by
// side, `stride` bytes after element k - 1 of them.  Either way these lines begin at 16-byte
// boundaries and are whole vectors of 16 bytes long, or zero up to one; stride < 2^22.
struct Operand {
    const void *p;
    uint64_t stride;
    uint64_t rows, k;
};
constexpr uint64_t MOST_STRIDE = 1ull << 22;

constexpr uint32_t OUTSIDE = 0x80000000u; // a range-checked load from here gives zeros

// A block's loads and a wave's reads of R rows of one side.  As m side (LANES) its rows are the lanes'
// own, as n side they are spread over four instructions so that a lane ends with 16 neighbouring ones.
template <class E, int R, bool ACROSS, bool LANES, int WAVES>
struct Side {
    static_assert(R / 8 % WAVES == 0 && (!ACROSS || sizeof(E) > 1), "");
    static constexpr uint32_t KE = CHUNK / sizeof(E);                         // elements of a chunk
    static constexpr uint32_t LINE = ACROSS ? R * sizeof(E) / 16 : CHUNK / 16; // vectors of a line
    static constexpr uint32_t BYTES = R * CHUNK;
    static constexpr int LOADS = R / 8 / WAVES; // of a wave, 64 vectors each

    // Position of a vector is turned by exclusive-or with a number of its line, so that lanes
    // that read different lines meet different banks.  The turn is made on the global side, as
    // loads past the registers land in lane order.
    static __device__ inline uint32_t turn(uint32_t line)
    {
        if constexpr (!ACROSS)
            return LANES ? line & 7 : (line & 3) | (line >> 2 & 4);
        else if constexpr (sizeof(E) == 4)
            return (LANES ? (line >> 2 & 3) << 2 : line >> 2 & 3) & (LINE - 1);
        else
            return (LANES ? (line & 3) << 1 | (line >> 3 & 1) << 3 : (line & 1) | (line >> 1 & 1) << 3) & (LINE - 1);
    }

    // Where the next chunk is loaded from.  A lane's offsets are made once a tile: made for every
    // chunk they cost a tenth (8192 x 8192 x 8192 bf16 1166 us, 1053; 4096 x 16384 x 768 137, 121).
    const uint8_t *from;
    uint64_t step;
    int64_t left;           // elements of the inner length from here on
    uint32_t offset[LOADS]; // rows past the end repeat the last one, vectors past it are outside
    uint32_t key[LOADS];    // the element (along) or line (across) of the chunk that a load begins with

    __device__ inline void begin(const Operand &of, uint64_t row0, uint32_t kb, uint32_t wave, uint32_t lane)
    {
        const uint32_t stride = (uint32_t)of.stride, last = (uint32_t)min(of.rows - row0, (uint64_t)R) - 1;
        from = (const uint8_t *)of.p + (ACROSS ? (uint64_t)kb * KE * of.stride + row0 * sizeof(E)
                                               : row0 * of.stride + (uint64_t)kb * CHUNK);
        step = ACROSS ? KE * of.stride : CHUNK;
        left = (int64_t)of.k - (int64_t)kb * KE;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t v = (i * WAVES + wave) * 64 + lane, line = v / LINE, at = (v % LINE ^ turn(line)) * 16;
            if constexpr (!ACROSS) {
                offset[i] = min(line, last) * stride + at;
                key[i] = at / sizeof(E);
            } else {
                offset[i] = at < (last + 1) * sizeof(E) ? line * stride + at : OUTSIDE;
                key[i] = line;
            }
        }
    }

    // The next chunk to `to`, zeros past the end; every wave of the block takes part.
    __device__ inline void load(uint8_t *to, uint32_t wave)
    {
        const __amdgpu_buffer_rsrc_t at = buffer_of(from, 0x7FFFFFFFu);
        const uint32_t there = uniform(left >= (int64_t)KE ? KE : left > 0 ? (uint32_t)left : 0u);
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            to_lds16(at, key[i] < there ? offset[i] : OUTSIDE, 0, to + (i * WAVES + wave) * 1024);
        from += step;
        left -= KE;
    }

    // A lane's 16 bytes of 16 rows for half `half` of the chunk: rows first + t * 16 + 0..15 as m
    // side; as n side row first + 16 q + 4 t + i for instruction row 4 q + i.
    static __device__ inline u32x4 fragment(const uint8_t *panel, uint32_t first, int t, int half, uint32_t lane)
    {
        const uint32_t r = lane & 15, g = lane >> 4;
        if constexpr (!ACROSS) {
            const uint32_t row = LANES ? first + t * 16 + r : first + (r >> 2) * 16 + t * 4 + (r & 3);
            return *reinterpret_cast<const u32x4 *>(panel + row * CHUNK + ((half * 4 + g) ^ (r & 7)) * 16);
        } else if constexpr (sizeof(E) == 4) {
            const uint32_t row = LANES ? first + t * 16 + r : first + (r >> 2) * 16 + t * 4 + (r & 3);
            u32x4 f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t line = half * 16 + g * 4 + i;
                f[i] = *reinterpret_cast<const uint32_t *>(panel + line * (R * 4) + (((row >> 2) ^ turn(line)) * 4 + (row & 3)) * 4);
            }
            return f;
        } else {
            // The transposing read: of 16 lanes, lane l brings the place of four neighbouring rows of
            // line l / 4, and gets the four lines of row l % 4 of place l / 4.
            using s16x4 = __attribute__((ext_vector_type(4))) short;
            using lds_s16x4 = __attribute__((address_space(3))) s16x4;
            const uint32_t place = r & 3;
            const uint32_t row = LANES ? first + t * 16 + place * 4 : first + place * 16 + t * 4;
            union {
                s16x4 h[2];
                u32x4 v;
            } f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t line = half * 32 + g * 8 + h * 4 + (r >> 2);
                const uint8_t *at = panel + line * (R * 2) + ((row >> 3) ^ turn(line)) * 16 + (row & 4) * 2;
                f.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)at);
            }
            return f.v;
        }
    }
};

// The grid of a product: tiles along both sides, and shares of the inner length, whose sums are
// joined afterwards.
struct Grid {
    uint32_t m_tiles, n_tiles, splits;
    uint64_t chunks;
    uint32_t band; // tiles of m that follow each other before the next one of n
};

// Where a block's tile lies.  An XCD takes a contiguous run of them, in bands of tiles of m, so that the
// tiles it works on at a time share panels in its L2.
struct Tile {
    uint64_t m0, n0;
    uint32_t split;
    uint32_t high, strips; // rows of a tile; waves side by side along n, 64 columns each
    uint32_t wm, wn;       // the wave's part begins at row m0 + wm and column n0 + wn
    uint32_t lane, wave;
};

constexpr int BIG = 256; // rows and columns of the largest tile
// LDS that a wave needs to turn 16 x 64 results of a size
constexpr uint32_t turn_bytes(uint32_t size) { return 16 * 64 * size; }

// A block of WM x WN waves makes a BM x (64 WN) tile, each wave BM / WM x 64 of it in 16 x 16
// matrix instructions.  Both panels of a chunk are staged in LDS by loads that bypass the
// registers, one chunk ahead.  A lane ends with results [i][j][e]: row wm + 16 i + lane % 16,
// column wn + lane / 16 * 16 + 4 j + e.  `finish` brings what it needs of the tile's rows to LDS before
// the sums (ahead), the values they begin with (start), and takes the results.  One with MORE (bytes of LDS
// for a wave) adds to a chunk's products what A's panel does not hold: of the chunks that have such elements
// in the wave's rows (holds), a second fragment of A (more) beside the panel's, in the same order.
//   256 x 256 tiles of eight waves: a wave reads 24 KB of LDS for a chunk's 4 M products where 64 x 64
// parts read 32; 8192 x 8192 x 8192 bf16 1249 TFLOP/s in bands of 16 (4: 1168), 128 x 128 tiles, two
// blocks to a CU, 1097 (the library's product 1377); without the results' stores 4096 x 16384 x 384 1065
// and 950.  Chunks of 64 bytes in three or four stages were slower (1106 and 864): a row's loads
// are then half a line of memory each.
//   The panels lie in LDS variables of their own, and the loads are without branches: so the compiler
// knows which loads a read of LDS depends on, and adds no wait of its own.
template <class E, int BM, int WM, int WN, bool A_ACROSS, bool B_ACROSS, bool ONE, class Finish>
__device__ inline void make_tile(const Operand &a, const Operand &b, const Grid &grid, uint32_t block,
                                 const Finish &finish, uint8_t *a_even, uint8_t *a_odd, uint8_t *b_even, uint8_t *b_odd,
                                 uint8_t *side)
{
    // The largest tile takes chunks in pairs (a last odd one with zeros): a loop that can end between the
    // two moves the sums from registers to others, and there are none left.
    constexpr bool PAIRS = BM == BIG;
    constexpr int WAVES = WM * WN, BN = WN * 64, TM = BM / WM / 16;
    using A = Side<E, BM, A_ACROSS, true, WAVES>;
    using B = Side<E, BN, B_ACROSS, false, WAVES>;
    Tile at;
    at.high = BM;
    at.strips = WN;
    at.lane = threadIdx.x & 63;
    at.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    at.wm = at.wave % WM * (BM / WM);
    at.wn = at.wave / WM * 64;
    uint32_t kb, kb_end;
    {
        const uint32_t tiles = grid.m_tiles * grid.n_tiles, item = xcd_run(block, tiles * grid.splits);
        uint32_t tm, tn;
        at.split = uniform(item / tiles);
        tile_of(item - at.split * tiles, grid.band, grid.m_tiles, grid.n_tiles, tm, tn);
        at.m0 = (uint64_t)uniform(tm) * BM;
        at.n0 = (uint64_t)uniform(tn) * BN;
        constexpr uint32_t UNIT = PAIRS ? 2 : 1;
        const uint32_t units = (uint32_t)((grid.chunks + UNIT - 1) / UNIT);
        const uint32_t share = units / grid.splits, longer = units % grid.splits;
        kb = UNIT * (at.split * share + min(at.split, longer));
        kb_end = kb + UNIT * (share + (at.split < longer ? 1 : 0));
    }
    A left;
    B right;
    left.begin(a, at.m0, kb, at.wave, at.lane);
    right.begin(b, at.n0, kb, at.wave, at.lane);
    auto load = [&](uint8_t *to_a, uint8_t *to_b) {
        left.load(to_a, at.wave);
        right.load(to_b, at.wave);
        __builtin_amdgcn_sched_barrier(0);
    };
    load(a_even, b_even);
    typename Matrix<E>::Acc acc[TM][4];
    finish.ahead(at, side);
    finish.start(at, acc);
    constexpr bool MORE = Finish::MORE > 0;
    static_assert(!MORE || BM < BIG, "the largest tile has no registers left for it");
    typename Finish::Next next;
    uint8_t *const own = side + BM * Finish::AHEAD + at.wave * Finish::MORE;
    if constexpr (MORE)
        finish.first(next, kb * (CHUNK / sizeof(E)), at.lane);

    auto step = [&](const uint8_t *pa, const uint8_t *pb, uint8_t *next_a, uint8_t *next_b) {
        await_loads<0>(); // loads into LDS are counted as memory loads, which a barrier alone does not await
        __builtin_amdgcn_s_barrier(); // the panels have landed; every wave is done with the others
        __builtin_amdgcn_sched_barrier(0);
        uint32_t held = 0; // of the wave's groups of 16 rows, those with more: of either half, 16 bits each
        if constexpr (MORE)
            held = finish.template holds<TM>(next, at, own);
        if constexpr (!ONE)
            load(next_a, next_b);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            u32x4 y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                y[j] = B::fragment(pb, at.wn, j, half, at.lane);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const u32x4 x = A::fragment(pa, at.wm, i, half, at.lane);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = Matrix<E>::mul(y[j], x, acc[i][j]);
            }
            if constexpr (MORE)
                if (held >> half * 16 & 0xFFFF)
#pragma unroll
                    for (int i = 0; i < TM; ++i)
                        if (held >> (half * 16 + i) & 1) {
                            const u32x4 x = finish.more(own, i, half, at.lane);
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                acc[i][j] = Matrix<E>::mul(y[j], x, acc[i][j]);
                        }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the panels are read
    };
    if constexpr (ONE) {
        step(a_even, b_even, nullptr, nullptr);
    } else if constexpr (PAIRS) {
        for (uint32_t pairs = (kb_end - kb) / 2; pairs; --pairs) {
            step(a_even, b_even, a_odd, b_odd);
            step(a_odd, b_odd, a_even, b_even);
        }
    } else {
        while (kb < kb_end) {
            step(a_even, b_even, a_odd, b_odd);
            if (++kb == kb_end)
                break;
            step(a_odd, b_odd, a_even, b_even);
            ++kb;
        }
    }
    await_loads<0>(); // the last step's loads, of the chunk past the end, land here
    __syncthreads();  // the panels are free for the finish
    finish(at, side, acc, WN == 1 ? a_even : b_even); // (turn_bytes of every wave)
}

template <class E, int BM, int WM, int WN, bool A_ACROSS, bool B_ACROSS, class Finish>
__global__ __launch_bounds__(WM * WN * 64, 2) void ung_tile_kernel(Operand a, Operand b, Grid grid, Finish finish)
{
    constexpr uint32_t HIGH = BM * CHUNK, WIDE = WN * 64 * CHUNK;
    __shared__ alignas(16) uint8_t a_even[HIGH], a_odd[HIGH], b_even[WIDE], b_odd[WIDE];
    __shared__ alignas(16) uint8_t side[BM * Finish::AHEAD + WM * WN * Finish::MORE + 16];
    make_tile<E, BM, WM, WN, A_ACROSS, B_ACROSS, false>(a, b, grid, blockIdx.x, finish, a_even, a_odd, b_even, b_odd, side);
}

// Two products in one launch, the first's tiles before the second's, for two that do not need each other
// and do not fill the chip's rounds by themselves.
template <class E, int BM, int WM, int WN, bool A_ACROSS, bool B_ACROSS, bool A2_ACROSS, bool B2_ACROSS, class Finish,
          class Finish2>
__global__ __launch_bounds__(WM * WN * 64, 2) void ung_two_products_kernel(Operand a, Operand b, Grid grid, Finish finish,
                                                                         Operand a2, Operand b2, Grid grid2,
                                                                         Finish2 finish2)
{
    constexpr uint32_t HIGH = BM * CHUNK, WIDE = WN * 64 * CHUNK;
    constexpr uint32_t SIDE = BM * Finish::AHEAD + WM * WN * Finish::MORE, SIDE2 = BM * Finish2::AHEAD + WM * WN * Finish2::MORE;
    __shared__ alignas(16) uint8_t a_even[HIGH], a_odd[HIGH], b_even[WIDE], b_odd[WIDE];
    __shared__ alignas(16) uint8_t side[(SIDE > SIDE2 ? SIDE : SIDE2) + 16];
    const uint32_t first = grid.m_tiles * grid.n_tiles * grid.splits;
    if (blockIdx.x < first)
        make_tile<E, BM, WM, WN, A_ACROSS, B_ACROSS, false>(a, b, grid, blockIdx.x, finish, a_even, a_odd, b_even, b_odd, side);
    else
        make_tile<E, BM, WM, WN, A2_ACROSS, B2_ACROSS, false>(a2, b2, grid2, blockIdx.x - first, finish2, a_even, a_odd,
                                                              b_even, b_odd, side);
}

// Products of one chunk, where the results' stores are what takes the time: half the LDS, so that four blocks
// are on a CU at different places of a tile.  100000 x 384 results of 1 to 64 16-bit numbers 20 us, two
// blocks to a CU 26.
template <class E, bool A_ACROSS, bool B_ACROSS, class Finish>
__global__ __launch_bounds__(256, 4) void ung_one_chunk_kernel(Operand a, Operand b, Grid grid, Finish finish)
{
    __shared__ alignas(16) uint8_t a_panel[128 * CHUNK], b_panel[128 * CHUNK];
    __shared__ alignas(16) uint8_t side[128 * Finish::AHEAD + 4 * Finish::MORE + 16];
    make_tile<E, 128, 2, 2, A_ACROSS, B_ACROSS, true>(a, b, grid, blockIdx.x, finish, a_panel, nullptr, b_panel, nullptr, side);
}

// ---- few rows against many ------------------------------------------------------------------

// 64 rows of the n side, a wave's, straight to registers: nothing else reads them.
template <class E>
struct Stream {
    const uint8_t *from;
    int32_t left; // bytes of a row from here on
    uint32_t offset[4], at;

    __device__ inline void begin(const Operand &of, uint64_t row0, uint32_t lane)
    {
        const uint32_t r = lane & 15, last = (uint32_t)min(of.rows - row0, (uint64_t)64) - 1;
        at = (lane >> 4) * 16;
        from = (const uint8_t *)of.p + row0 * of.stride;
        left = (int32_t)(of.k * sizeof(E));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            offset[j] = min((r >> 2) * 16 + j * 4 + (r & 3), last) * (uint32_t)of.stride + at;
    }
    // The next chunk, zeros past the end.
    __device__ inline void load(u32x4 (&y)[2][4])
    {
        const __amdgpu_buffer_rsrc_t p = buffer_of(from, 0x7FFFFFFFu);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                y[h][j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                        p, (int32_t)(at + h * 64) < left ? offset[j] + h * 64 : OUTSIDE, 0, 0));
        from += CHUNK;
        left -= CHUNK;
    }
};

// A wave's own rows of the m side, up to 16 TM of them, read by every wave from memory (its caches).
template <class E, int TM>
struct Rows {
    const uint8_t *from;
    int32_t left;
    uint32_t offset[TM], at;

    __device__ inline void begin(const Operand &of, uint32_t lane)
    {
        at = (lane >> 4) * 16;
        from = (const uint8_t *)of.p;
        left = (int32_t)(of.k * sizeof(E));
#pragma unroll
        for (int i = 0; i < TM; ++i)
            offset[i] = min(i * 16 + (lane & 15), (uint32_t)of.rows - 1) * (uint32_t)of.stride + at;
    }
    __device__ inline void load(u32x4 (&x)[2][TM])
    {
        const __amdgpu_buffer_rsrc_t p = buffer_of(from, 0x7FFFFFFFu);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < TM; ++i)
                x[h][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                        p, (int32_t)(at + h * 64) < left ? offset[i] + h * 64 : OUTSIDE, 0, 0));
        from += CHUNK;
        left -= CHUNK;
    }
};

// The same of rows that are aligned to their elements alone, and end anywhere: the chunk that a row's end
// is in comes first (zeros past the end), then the whole ones, by loads that are in range without a check.
// Loads off 4-byte boundaries are slow (100000 x 384 bf16 at an odd stride 47 us): 16-bit rows are loaded
// from the boundary before, a word more of them, and shifted when they are used.
template <class E, int ROWS>
struct Loose {
    static constexpr bool HALVES = sizeof(E) == 2;
    struct Words {
        u32x4 w;
        uint32_t next; // (16-bit rows alone)
    };
    using Chunk = Words[2][ROWS];
    const uint8_t *from;
    uint32_t left; // whole chunks
    uint32_t offset[ROWS], shift[ROWS];

    // place(i): the lane's i-th row.  `end`: the chunk of the row's end.
    template <class Place>
    __device__ inline void begin(const Operand &of, uint64_t row0, uint32_t lane, u32x4 (&end)[2][ROWS], const Place &place)
    {
        const uint32_t last = (uint32_t)min(of.rows - row0, (uint64_t)64) - 1, at = (lane >> 4) * 16;
        from = (const uint8_t *)of.p + row0 * of.stride;
        const uint32_t off = (uint32_t)(uintptr_t)from & 3;
        left = (uint32_t)(of.k * sizeof(E)) / CHUNK;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const uint32_t row = min(place(i), last) * (uint32_t)of.stride;
            offset[i] = row + at + off;
            shift[i] = offset[i] & 3;
            offset[i] -= shift[i];
#pragma unroll
            for (int h = 0; h < 2; ++h)
                end[h][i] = __builtin_bit_cast(u32x4, load_row((const E *)(from + row), (left * CHUNK + h * 64 + at) / sizeof(E), of.k));
        }
        from -= off;
    }
    // The next whole chunk, or the last again.
    __device__ inline void load(Chunk &y)
    {
        if (!left)
            return;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const uint32_t *p = reinterpret_cast<const uint32_t *>(from + offset[i] + h * 64);
                __builtin_memcpy(&y[h][i].w, p, 16);
                if constexpr (HALVES) // (the word that holds the last element)
                    y[h][i].next = p[shift[i] ? 4 : 3];
            }
        if (--left)
            from += CHUNK;
        else
            left = 1;
    }
    __device__ inline u32x4 of(const Words &y, int i) const
    {
        if constexpr (!HALVES)
            return y.w;
        else
            return u32x4{__builtin_amdgcn_alignbyte(y.w[1], y.w[0], shift[i]), __builtin_amdgcn_alignbyte(y.w[2], y.w[1], shift[i]),
                         __builtin_amdgcn_alignbyte(y.w[3], y.w[2], shift[i]),
                         __builtin_amdgcn_alignbyte(y.next, y.w[3], shift[i])};
    }
};

// Up to 16 TM rows of a against all of b, where reading b is what takes the time: a wave takes 64 rows of
// b and no more, past LDS and without barriers, the next two chunks' loads under way while two are
// multiplied.  Results as ung_tile_kernel's.  LOOSE: rows need no alignment (100000 x 384 bf16 at an odd
// stride 25.6 us, copied to rows of whole vectors first 51.5; at whole vectors 19.7 as they are.  float32
// 36, 95 and 32; 100000 x 100 bf16 13, 26, and 9 where they are 104).
// Blocks y: shares of the inner length, `each` chunks long.
template <class E, int TM, bool LOOSE, class Finish>
__global__ __launch_bounds__(64) void ung_few_rows_kernel(Operand a, Operand b, uint32_t each, Finish finish)
{
    __shared__ alignas(16) uint8_t own[turn_bytes(4)];
    __shared__ alignas(16) uint8_t side[16 * TM * Finish::AHEAD + 16];
    Tile at = {};
    at.high = 16 * TM;
    at.strips = 1;
    at.lane = threadIdx.x;
    at.n0 = (uint64_t)xcd_run(blockIdx.x, gridDim.x) * 64;
    if (gridDim.y > 1) {
        const uint64_t first = (uint64_t)blockIdx.y * each * CHUNK;
        a.p = (const uint8_t *)a.p + first;
        b.p = (const uint8_t *)b.p + first;
        a.k = b.k = min(b.k - first / sizeof(E), (uint64_t)each * CHUNK / sizeof(E));
        at.split = blockIdx.y;
    }
    typename Matrix<E>::Acc acc[TM][4];
    auto multiply = [&](const auto &y, const auto &x) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = Matrix<E>::mul(y(h, j), x(h, i), acc[i][j]);
    };
    const uint32_t bytes = (uint32_t)(b.k * sizeof(E)), r = at.lane & 15;
    if constexpr (LOOSE) {
        Loose<E, 4> right;
        Loose<E, TM> left;
        typename Loose<E, 4>::Chunk y[2];
        typename Loose<E, TM>::Chunk x[2];
        u32x4 y_end[2][4], x_end[2][TM];
        right.begin(b, at.n0, at.lane, y_end, [&](int j) { return (r >> 2) * 16 + j * 4 + (r & 3); });
        left.begin(a, 0, at.lane, x_end, [&](int i) { return i * 16 + r; });
        right.load(y[0]);
        left.load(x[0]);
        finish.ahead(at, side);
        finish.start(at, acc);
        multiply([&](int h, int j) { return y_end[h][j]; }, [&](int h, int i) { return x_end[h][i]; });
        auto step = [&](int now) {
            right.load(y[now ^ 1]);
            left.load(x[now ^ 1]);
            multiply([&](int h, int j) { return right.of(y[now][h][j], j); }, [&](int h, int i) { return left.of(x[now][h][i], i); });
        };
        for (uint32_t chunks = bytes / CHUNK; chunks; --chunks) {
            step(0);
            if (!--chunks)
                break;
            step(1);
        }
    } else {
        u32x4 y[2][2][4], x[2][2][TM];
        Stream<E> right;
        Rows<E, TM> left;
        right.begin(b, at.n0, at.lane);
        left.begin(a, at.lane);
        right.load(y[0]);
        left.load(x[0]);
        finish.ahead(at, side);
        finish.start(at, acc);
        auto step = [&](int now) {
            right.load(y[now ^ 1]);
            left.load(x[now ^ 1]);
            multiply([&](int h, int j) { return y[now][h][j]; }, [&](int h, int i) { return x[now][h][i]; });
        };
        for (uint32_t pairs = ((bytes + CHUNK - 1) / CHUNK + 1) / 2; pairs; --pairs) { // (a last odd one with zeros)
            step(0);
            step(1);
        }
    }
    __syncthreads();
    finish(at, side, acc, own);
}

// A finish that needs nothing ahead and adds nothing, and sums that begin at 0.
struct Plainly {
    static constexpr uint32_t AHEAD = 0; // bytes of LDS for a row
    static constexpr uint32_t MORE = 0;  // and for a wave
    struct Next {};
    __device__ inline void ahead(const Tile &, uint8_t *) const {}
    template <class Acc, int TM>
    __device__ inline void start(const Tile &, Acc (&acc)[TM][4]) const
    {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[i][j] = Acc{0, 0, 0, 0};
    }
};

// ---- storing a tile's results ------------------------------------------------------------

// A wave's 16 x 64 results (row r, columns g * 16 + 0..15 of each lane 16 g + r) to `to`, rows
// `stride` elements apart, of which `rows` and `cols` are there.  16-bit vectors go out as they lie where
// `vectors`; the others are turned in LDS first, so that a store's lanes write neighbouring elements.
// `own`: turn_bytes of LDS of the wave's own; a block's are no more than its larger panel.
template <class T>
__device__ inline void store_rows(T *to, uint64_t stride, uint32_t rows, uint64_t cols, bool vectors,
                                  const Vec<T> (&o)[16 / Vec<T>::N], uint8_t *own, uint32_t lane)
{
    constexpr int N = Vec<T>::N;
    constexpr uint32_t V = 64 / N; // vectors of a row; their positions are turned by its number
    const uint32_t r = lane & 15, g = lane >> 4;
    if (sizeof(T) == 2 && vectors && cols >= 64) {
        if (r < rows)
#pragma unroll
            for (int x = 0; x < 16 / N; ++x)
                store_loose(to + r * stride + g * 16 + x * N, o[x]);
        return;
    }
    auto place = [&](uint32_t row, uint32_t v) { return own + (row * V + (v ^ (row & (V - 1)))) * 16; };
#pragma unroll
    for (uint32_t x = 0; x < 16 / N; ++x)
        *reinterpret_cast<Vec<T> *>(place(r, g * (16 / N) + x)) = o[x];
    wave_lds_fence();
    if (vectors && cols >= 64) {
        const uint32_t y0 = lane / V, x = lane % V; // V lanes hold a row
#pragma unroll
        for (uint32_t y = 0; y < 16; y += N)
            if (y + y0 < rows)
                store_loose(to + (y + y0) * stride + x * N, *reinterpret_cast<const Vec<T> *>(place(y + y0, x)));
    } else if (lane < cols) {
#pragma unroll 4
        for (uint32_t y = 0; y < rows; ++y)
            to[y * stride + lane] = *reinterpret_cast<const T *>(place(y, lane / N) + lane % N * sizeof(T));
    }
    wave_lds_fence();
}

} // namespace ung
