// Products over the rows of a block in bf16 (what fgl_row_product.hip forms, which see) where there are enough rows to keep the weights on the CUs:
// C[m, n] = A[m, k] B[k, n], or act(A B + bias) + residual.
//
// Split: as in fgl_split_product.hip a workgroup keeps its 32 NT columns of B in LDS, in the order in which the lanes take them, and its waves go over the rows
// of A, here in tiles of 64 or 32, each by itself: no barrier after the first.  A lane reads its one or two rows of A straight to registers, 64 k (a line of 128 bytes
// a row) ahead.  Lines are read whole: in pieces of 32 k, with twice as many on their way, 87 K x 256 x 512 took 61 us for 53.
//
// What bounds it: for short k and few columns the pass over A and C (2.4 M x 64 x 100 164 us, 4.8 TB/s), beyond that the loads' latency, with as many rows on their way as the
// registers hold: the matrix cores are busy for a seventh to a fifth of the time (87 K x 512 x 256 45 us, 0.51 PFLOP/s, 21 %; 87 K x 256 x 512 with relu 64 us, 14 %; the old kernel of fgl_row_product.hip 67).
//
// k past the end: a lane's eight k begin where they would or eight before the end of the row, and those that an eight before has are zero on both sides.
// Rows past the end repeat the last one and are not stored, nor are columns past the end, which repeat the last one too.  No access leaves the operands.
#include "fgl_common.hpp"
#include "fgl_kernels.hpp"
#include "fgl_row_product.hpp"
#include "fgl_split.hpp"

namespace fgl {

constexpr int kBpLds = 158 * 1024;
typedef uint32_t BpU4 __attribute__((ext_vector_type(4), aligned(2)));

// Steps of 16 k that are on their way together: 64 k, a line of 128 bytes a row, or a whole row of up to 128 k where the accumulators leave the registers.  (Rows of 200 bytes in two
// loads are read twice: the lines between the two have left the L2 by the second, which comes behind a tile's epilogue.  2.4 M x 100 x 64: 911 MB read, 279 us with silu and its slopes, 252 so.)
constexpr int bp_steps(int k, int nt) { return nt <= 2 && k > 64 && k <= 128 ? 8 : 4; }
__device__ __host__ __forceinline__ int bp_chunks(int k, int steps) { return (k + 16 * steps - 1) / (16 * steps); }
// Where the eight k of number `oct` are read
__device__ __forceinline__ int bp_first(int oct, int k) { return 8 * oct + 8 <= k ? 8 * oct : k - 8; }

// Of a row's last S steps, how many are whole whatever the row
constexpr int bp_whole(int steps) { return steps == 8 ? 4 : 0; }

// Clears what of a row's last S steps, from number `step` on, an eight before has: infinite, it would make a zero of B's image no number.  One step at most has
// both, of which a lane's eight are those from `again` on.
template <int VA, int S>
__device__ __forceinline__ void bp_own(SpU4 (&a)[VA][S], int step, int half, int k)
{
    const int mixed = k / 16 - step;
#pragma unroll
    for (int s = bp_whole(S); s < S; ++s) {
        if (s < mixed) continue;
        if (s > mixed) {
#pragma unroll
            for (int i = 0; i < VA; ++i) a[i][s] = SpU4{};
            continue;
        }
        int oct = 2 * (step + s) + half;
        asm volatile("" : "+v"(oct));  // (what is made of it is not kept over the rows)
        const int again = 8 * oct - bp_first(oct, k);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t own = again <= 2 * j ? 0xFFFFFFFFu : again == 2 * j + 1 ? 0xFFFF0000u : 0u;
#pragma unroll
            for (int i = 0; i < VA; ++i) a[i][s][j] &= own;
        }
    }
}

// (the lanes' columns: fgl_split_product.hip)
__device__ __forceinline__ int bp_column(int vl, int t, int i) { return ((t >> vl) << (5 + vl)) + (i << vl) + (t & ((1 << vl) - 1)); }

// B's columns from col0 on -> img[step * NT + tile][lane], a step being 16 k
template <int NT, bool BT, int THREADS>
__device__ __forceinline__ void bp_stage(const RowProductSide& x, int octs, int col0, int n, int vl, SpU4* img)
{
    constexpr int kCols = 32 * NT, kBatch = 8;  // (so many loads a thread on their way; the accumulators' registers are free yet)
    const uint16_t* b = static_cast<const uint16_t*>(x.b);
    const int items = octs * kCols;
    // A transposed B is read along its rows, a line of 128 bytes by eight lanes, another one along its columns.
    auto place = [&](int at, int& oct, int& c) {
        if constexpr (BT) {
            oct = at / (8 * kCols) * 8 + at % 8;
            c = at / 8 % kCols;
        } else {
            oct = at / kCols;
            c = at % kCols;
        }
    };
    for (int first = (int)threadIdx.x; first < items; first += THREADS * kBatch) {
        SpU4 v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            int oct, c;
            place(first + i * THREADS < items ? first + i * THREADS : items - 1, oct, c);
            const int col = col0 + c < n ? col0 + c : n - 1, k0 = bp_first(oct, x.k);
            if constexpr (BT) {
                const BpU4 w = *reinterpret_cast<const BpU4*>(b + (int64_t)col * x.ldb + k0);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = w[j];
            } else {
                const uint16_t* p = b + (int64_t)k0 * x.ldb + col;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i][j] = (uint32_t)p[2 * j * x.ldb] | (uint32_t)p[(2 * j + 1) * x.ldb] << 16;
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int at = first + i * THREADS;
            if (at >= items) break;
            int oct, c;
            place(at, oct, c);
            const int k0 = bp_first(oct, x.k), own = 8 * oct;
            if (k0 != own) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (k0 + 2 * j < own) v[i][j] &= 0xFFFF0000u;
                    if (k0 + 2 * j + 1 < own) v[i][j] &= 0x0000FFFFu;
                }
            }
            const int t = (c >> (5 + vl) << vl) + (c & ((1 << vl) - 1)), lane = (c >> vl) & 31;
            img[((oct / 2) * NT + t) * kWave + oct % 2 * 32 + lane] = v[i];
        }
    }
}

template <int VA, int NT, int V>
__device__ __forceinline__ void bp_then(const RowProductArgs& g, int64_t row0, int col0, const SpF32x16 (&acc)[VA][NT])
{
    int lane = lane_id();
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int q = 0; q < NT / V; ++q) {
        const int col = col0 + 32 * V * q + lane % 32 * V;
        float add[V];
#pragma unroll
        for (int t = 0; t < V; ++t) {
            add[t] = 0.0f;
            if (g.bias != nullptr && col + t < g.n) add[t] = __uint_as_float((uint32_t)static_cast<const uint16_t*>(g.bias)[col + t] << 16);
        }
#pragma unroll
        for (int i = 0; i < VA; ++i) rp_then<uint16_t, V>(g, row0 + 32 * i, lane / 32, col, [&](int t, int r) { return acc[i][q * V + t][r] + add[t]; });
    }
}

// Behind matrix instructions, before their results are read.  (All of them operands of the one statement, so that none is read before it.)
template <int VA, int NT>
__device__ __forceinline__ void bp_wait(SpF32x16 (&a)[VA][NT])
{
    if constexpr (VA == 2 && NT == 4)
        asm volatile("s_nop 15\n\ts_nop 15" : "+v"(a[0][0]), "+v"(a[0][1]), "+v"(a[0][2]), "+v"(a[0][3]), "+v"(a[1][0]), "+v"(a[1][1]), "+v"(a[1][2]), "+v"(a[1][3]));
    else if constexpr (VA == 2 && NT == 2) asm volatile("s_nop 15\n\ts_nop 15" : "+v"(a[0][0]), "+v"(a[0][1]), "+v"(a[1][0]), "+v"(a[1][1]));
    else if constexpr (VA == 2) asm volatile("s_nop 15\n\ts_nop 15" : "+v"(a[0][0]), "+v"(a[1][0]));
    else if constexpr (NT == 4) asm volatile("s_nop 15\n\ts_nop 15" : "+v"(a[0][0]), "+v"(a[0][1]), "+v"(a[0][2]), "+v"(a[0][3]));
    else if constexpr (NT == 2) asm volatile("s_nop 15\n\ts_nop 15" : "+v"(a[0][0]), "+v"(a[0][1]));
    else asm volatile("s_nop 15\n\ts_nop 15" : "+v"(a[0][0]));
}

// Waves a SIMD: as the accumulators' and the rows' registers allow
constexpr int bp_waves(int va, int nt, int steps) { return va == 1 ? (nt >= 4 || steps == 8 ? 3 : 4) : nt >= 4 || steps == 8 ? 2 : nt == 2 ? 3 : 4; }

// V: neighbouring columns a lane stores, S: bp_steps
template <int VA, int NT, int W, bool BT, int V, int S>
__global__ __launch_bounds__(W * kWave, bp_waves(VA, NT, S)) void bf16_product_kernel(const RowProductArgs g)
{
    extern __shared__ SpU4 s_img[];
    const int lane = lane_id(), half = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    const unsigned per_group = 8u * (unsigned)g.tiles_n;
    const int64_t rb = (int64_t)(blockIdx.x / per_group) * 8 + blockIdx.x % per_group % 8;
    const int col0 = (int)(blockIdx.x % per_group / 8) * 32 * NT;
    const int64_t row_tiles = (g.m + 32 * VA - 1) / (32 * VA), stride = g.row_blocks * W;
    if (rb * W >= row_tiles) return;  // (uniform over the workgroup: no row tile for it)
    const int k = g.side[0].k, chunks = bp_chunks(k, S);
    const bool ragged = k % (16 * S) != 0;
    const int64_t lda = g.side[0].lda;
    int64_t tile = rb * W + wave, ahead = tile;
    int at = 0;
    const uint16_t* p[VA];
    auto rows_of = [&](int64_t t) {
#pragma unroll
        for (int i = 0; i < VA; ++i) {
            const int64_t row = t * (32 * VA) + 32 * i + lane % 32;
            p[i] = static_cast<const uint16_t*>(g.side[0].a) + (row < g.m ? row : g.m - 1) * lda;
        }
    };
    rows_of(ahead);
    auto load = [&](SpU4 (&a)[VA][S]) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int k0 = bp_first(2 * S * at + 2 * s + half, k);
#pragma unroll
            for (int i = 0; i < VA; ++i) {
                const BpU4 u = *reinterpret_cast<const BpU4*>(p[i] + k0);
#pragma unroll
                for (int j = 0; j < 4; ++j) a[i][s][j] = u[j];
            }
        }
        if (++at == chunks) {
            at = 0;
            if (ahead + stride < row_tiles) ahead += stride;
            rows_of(ahead);
        }
    };
    SpU4 cur[VA][S], next[VA][S];
    load(cur);
    bp_stage<NT, BT, W * kWave>(g.side[0], 2 * S * chunks, col0, g.n, V == 4 ? 2 : V == 2 ? 1 : 0, s_img);
    __syncthreads();
    if (tile >= row_tiles) return;  // (uniform over the wave; no barrier follows)
    for (;;) {
        SpF32x16 acc[VA][NT];
#pragma unroll
        for (int i = 0; i < VA; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[i][t] = SpF32x16{};
        const SpU4* img = s_img + lane;
        for (int c = 0; c < chunks; ++c) {
            load(next);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                if (s == bp_whole(S) && ragged && c == chunks - 1) bp_own<VA, S>(cur, S * c, half, k);
                SpU4 b[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) b[t] = img[(s * NT + t) * kWave];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < VA; ++i)
                        acc[i][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Bf16x8, cur[i][s]), __builtin_bit_cast(Bf16x8, b[t]), acc[i][t], 0, 0, 0);
            }
            img += S * NT * kWave;
#pragma unroll
            for (int i = 0; i < VA; ++i)
#pragma unroll
                for (int s = 0; s < S; ++s) cur[i][s] = next[i][s];
        }
        // The sums may be read so many cycles after the last product; a branch lies between the two, across which the compiler was seen not to keep them.
        bp_wait(acc);
        const int64_t row0 = tile * (32 * VA);
        bp_then<VA, NT, V>(g, row0, col0, acc);
        tile += stride;
        if (tile >= row_tiles) return;
    }
}

static size_t bp_lds(int k, int nt) { return (size_t)bp_chunks(k, bp_steps(k, nt)) * bp_steps(k, nt) * nt * kWave * sizeof(SpU4); }

static int bp_tiles(int k, int n)
{
    if (n > 64 && bp_lds(k, 4) <= (size_t)kBpLds) return 4;
    return n > 32 && bp_lds(k, 2) <= (size_t)kBpLds ? 2 : 1;
}

// Whether that is ahead of fgl_row_product.hip's kernel, which has nothing to stage first: from 3.3 M outputs on, columns padded to 32 and 128 at least, and for a short k, of which
// that kernel reads little again, 100 K rows.  (us, that kernel / this, B transposed: 256 x 256 8192 rows 8.5 / 10.4, 12 K 14 / 11, 80 K 41 / 30; 100 x 256 8192 5.1 / 6.8, 20 K
// 10.3 / 8.7, 80 K 28 / 16; 512 x 256 8192 14 / 21, 20 K 41 / 22; 256 x 512 4000 10 / 10, 20 K 31 / 20; 256 x 47 12 K 6 / 9, 40 K 14 / 12; 602 x 64 12 K 8 / 12, 20 K 17 / 12; 64 x 64 80 K
// 8.1 / 8.4; not transposed: 256 x 256 12 K 9 / 11, 20 K 15 / 11; 512 x 256 12 K 15 / 21, 20 K 26 / 21; 256 x 47 40 K 12 / 13, 80 K 20 / 17; 2.4 M x 64 x 100 172 / 162.)
bool bf16_product_pays(const RowProductArgs& g)
{
    const int k = g.side[0].k;
    const int64_t columns = ceil_div(g.n, 32) * 32;
    return k >= 16 && bp_lds(k, 1) <= (size_t)kBpLds && g.m * (columns < 128 ? 128 : columns) >= 3300000 && (k >= 96 || g.m >= 100000);
}

template <int VA, int NT, int W, bool BT, int S>
static int launch_bf16_product(RowProductArgs g, hipStream_t stream)
{
    const size_t lds = bp_lds(g.side[0].k, NT);
    g.tiles_n = (int)ceil_div(g.n, 32 * NT);
    int64_t per_cu = kBpLds / (int64_t)lds;
    if (per_cu > bp_waves(VA, NT, S) * 4 / W) per_cu = bp_waves(VA, NT, S) * 4 / W;
    const uint64_t starts = (uintptr_t)g.c | (uintptr_t)g.then.residual | (uintptr_t)g.then.slope | (uint64_t)(g.ldc | g.then.ldr | g.then.lds | g.n) * 2;
    const int v = NT >= 4 && starts % 8 == 0 ? 4 : NT >= 2 && starts % 4 == 0 ? 2 : 1;
    g.row_blocks = sp_row_blocks(ceil_div(g.m, 32 * VA), W, (int)per_cu, g.tiles_n);
    const int64_t blocks = ceil_div(g.row_blocks, 8) * 8 * g.tiles_n;
    FGL_REQUIRE(blocks <= 0x7FFFFFFF, "row_product: grid too large");
    const dim3 grid((unsigned)blocks), block(W * kWave);
    if (v == 4) hipLaunchKernelGGL((bf16_product_kernel<VA, NT, W, BT, NT >= 4 ? 4 : 1, S>), grid, block, lds, stream, g);
    else if (v == 2) hipLaunchKernelGGL((bf16_product_kernel<VA, NT, W, BT, NT >= 2 ? 2 : 1, S>), grid, block, lds, stream, g);
    else hipLaunchKernelGGL((bf16_product_kernel<VA, NT, W, BT, 1, S>), grid, block, lds, stream, g);
    FGL_CHECK_LAUNCH("bf16_product_kernel");
    return FGL_OK;
}

// Rows of a wave's tile, 32 or 64.  64 read an operand of B for two products, but more of them than the chip has waves are another whole round, and a round of them is longer: what
// the two take is counted in rows for each SIMD, 32 allowed to be a tenth behind (87 K x 512 x 256: 44.7 us where 64 take 61.9, with a residual 47.8 / 66.3; but 256 x 512, alike in
// rows, 58.2 / 53.5 and with relu 68.9 / 58.5).  Up to 128 k the pass over memory is what counts, and more waves are ahead (2.4 M x 64 x 100 164 / 170).
static bool bp_short_tiles(const RowProductArgs& g, int nt)
{
    const int steps = bp_steps(g.side[0].k, nt);
    auto rows = [&](int va) {
        const int64_t waves = 4 * 256 * bp_waves(va, nt, steps), tiles = ceil_div(g.m, 32 * va) * ceil_div(g.n, 32 * nt);
        return ceil_div(tiles, waves) * bp_waves(va, nt, steps) * va;
    };
    return (nt == 4 && g.side[0].k <= 128) || rows(1) * 11 <= rows(2) * 10;
}

template <bool BT>
static int launch_bf16_product_any(const RowProductArgs& g, hipStream_t stream)
{
    const int k = g.side[0].k, nt = bp_tiles(k, g.n);
    const size_t lds = bp_lds(k, nt);
    const bool one_a_cu = lds * 2 > (size_t)kBpLds, small = bp_short_tiles(g, nt);
    if (nt == 4) {
        if (!small) return one_a_cu ? launch_bf16_product<2, 4, 8, BT, 4>(g, stream) : launch_bf16_product<2, 4, 4, BT, 4>(g, stream);
        if (lds * 3 <= (size_t)kBpLds) return launch_bf16_product<1, 4, 4, BT, 4>(g, stream);
        return one_a_cu ? launch_bf16_product<1, 4, 12, BT, 4>(g, stream) : launch_bf16_product<1, 4, 6, BT, 4>(g, stream);
    }
    auto of = [&](auto tall) {
        constexpr int VA = decltype(tall)::value;
        if (bp_steps(k, nt) == 8) return nt == 2 ? launch_bf16_product<VA, 2, 4, BT, 8>(g, stream) : launch_bf16_product<VA, 1, 4, BT, 8>(g, stream);
        if (nt == 2) return one_a_cu ? launch_bf16_product<VA, 2, 8, BT, 4>(g, stream) : launch_bf16_product<VA, 2, 4, BT, 4>(g, stream);
        return one_a_cu ? launch_bf16_product<VA, 1, 8, BT, 4>(g, stream) : launch_bf16_product<VA, 1, 4, BT, 4>(g, stream);
    };
    return small ? of(std::integral_constant<int, 1>{}) : of(std::integral_constant<int, 2>{});
}

int bf16_product(const RowProductArgs& g, bool b_transposed, hipStream_t stream)
{
    return b_transposed ? launch_bf16_product_any<true>(g, stream) : launch_bf16_product_any<false>(g, stream);
}

}  // namespace fgl
