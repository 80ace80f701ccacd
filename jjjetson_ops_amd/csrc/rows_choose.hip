// The kernel of a float product by its sizes, and what its workspaces hold.  Host code only.
#include "rows_mm.hpp"

namespace jjo {

int64_t rows_output_rows(RowsMode mode, const RowsMm &p) {
    return mode == kRowsWeight ? (int64_t)p.Q * p.halves * std::max(p.n_experts, 1) : p.Q;
}

int64_t rows_part_bytes(RowsMode mode, const RowsMm &p) {
    return p.slices == 1 ? 0 : 4LL * p.slices * rows_output_rows(mode, p) * p.P * (mode == kRowsSwiglu ? 2 : 1);
}

// An estimate of each tile's time, the cheapest wins.  A launch is rounds of as many workgroups as the 256 CUs hold
// (the device's own number would change the workspace): two of the small tiles a CU, one of the large; a round takes
// `fixed` and one[] or two[] for each stage where a CU has one workgroup or two.  Slices of the sums divide the
// stages and cost a second launch and 8 bytes an output at 4 TB/s.  Measured (us, bf16; estimates in brackets): 2047
// x 14336 over 4096 on tiles of 256 / 160 / 128 rows 198 / 225 / 228 (191 / 232 / 245); 2048 x 4096 over 4096
// 90 / 76 / 64 (96 / 77 / 67); 64 x 4096 over 4096 on tiles of 64 x 64 in 1, 2, 4 slices 22.9 / 17.7 / 13.9
// (24.6 / 17.4 / 12.9).  fp32: 77 x 10624 over 6264 on tiles of 128 in 3 and 6 slices 155 and 138 (143 and 131), on
// tiles of 64 in 3 149 (151); 29 x 12440 over 6744 on tiles of 64 in 5 and 6 slices 113 and 124 (101 and 112).
RowsChoice rows_mm_choose(RowsMode mode, int dtype, int P, int Q, int K, int halves, int n_experts) {
    constexpr int64_t kCus = 256;
    const bool fp32 = dtype == JJO_DTYPE_F32, weight = mode == kRowsWeight, input = mode == kRowsInput;
    const int step = fp32 ? 32 : 64, piece = fp32 ? 4 : 8;
    // Rows that are not whole pieces of 16 bytes: tiles of 64 and 128 only, at times of their own; of less than a
    // piece (16 bits) those of 128.
    const int row_a = input || weight ? P : K, row_b = weight ? Q : K;
    const bool odd = row_a % piece != 0 || row_b % piece != 0, copied = !fp32 && (row_a < piece || row_b < piece);
    const int64_t cols = mode == kRowsSwiglu ? 2LL * P : P;  // columns of tiles
    // Experts with rows, as far as it is known without reading the offsets, and the rows (sums) of one.
    const int M = weight ? K : Q;
    const double experts = n_experts == 0 ? 1 : std::min(n_experts, M), mean = M / experts;

    // Few rows: a matrix is best read by the direct kernel up to 16 rows, of 16 bits up to 12 where tiles of 64 columns
    // occupy every other CU (11008 x 4096, 1 / 8 / 16 rows: 18.1 / 21.2 / 25.0 us against 23.6 / 23.9 / 23.9 on tiles,
    // fp32 35 / 40 / 47 against 62; 4096 x 4096, 16 rows: 10.6 against 12.9 in four slices).
    // Not on rows of 16 bits that are not aligned (4096 x 4095, 1 / 16 rows 17.4 / 28 us against 14.7 / 17.5 in four
    // slices; 11008 x 4095 42 / 75 against 29 / 39; fp32 15.3 / 20.4 against 30 / 31).
    // Of experts fp32, whose matrix instructions are slow on rows that are not there, up to 8 rows (8 experts' 4096 x
    // 2048 and 4096 x 4096, 1 row each: 54 and 99 against 75 and 146; 8 rows 65 and 119 against 75 and 145; 16 rows 78
    // and 141 against 75 and 147).  16 bits up to 4 rows: where the tiles are fewer than the CUs (8 experts of 704 and
    // 1408 columns over 2048: 8.5 and 14.2 against 11.8 and 14.5; over 4096: 13 and 20 against 16 and 25; over 512 all
    // within 3%), and, about even on average and ahead where few experts have rows, where sums are long and the tiles
    // leave CUs without a third workgroup (4096 x 14336, 8, 4 and 1 experts of 8 active: 214, 153 and 62 against 219,
    // 144 and 54 to 87; 4096 x 4096: 97, 53 and 22 against 98, 54 and 21 to 28; over 2048 29 against 30, over 2560 32
    // and 32).
    const int64_t tiles64 = (cols + 63) / 64;
    const double in_all = experts * (double)tiles64;
    const bool few = n_experts == 0 ? Q <= (fp32 || tiles64 < kCus / 2 ? 16 : 12)
                     : fp32         ? mean <= 8
                                    : mean <= 4 && (in_all < kCus || (K >= 4096 && in_all < 3 * kCus));
    if (few && (fp32 || !odd) && (mode == kRowsForward || mode == kRowsSwiglu)) {
        // Eight waves, but two for short sums of many workgroups (8 experts' 4096 x 512, 2 / 4 / 8 waves: 10.4 / 11.3 /
        // 15.8 us; x 2048 28.6 / 27.6 / 31.6; x 4096 59 / 54 / 51; one row of 11008 x 4096 19.0 / 18.8 / 18.1).
        const int64_t wgs = (int64_t)experts * ((cols + 15) / 16);
        return {kRowsDirect, K / (16 * piece) < 32 && wgs >= 4 * kCus ? 2 : 8, 1};
    }

    struct Cost {
        int p, q, a_cu;
        float fixed, one, two;
    };
    constexpr Cost k16[] = {{64, 64, 2, 2.2f, 0.35f, 0.5f}, {128, 128, 2, 2.9f, 0.65f, 1.0f},
                            {256, 160, 1, 5.f, 1.13f, 1.13f}, {256, 256, 1, 6.f, 1.4f, 1.4f}};
    // A stage of experts' rows, where few tiles share a matrix's rows and wait for memory: the tile with the least
    // estimate was within 4% of the best one's time on average, 30% at most (16 experts' 4096 x 4096, 64 rows: 153 us,
    // 118 on tiles of 256), over 53 products of 8 to 128 experts with 25 to 1024 rows on average, 704 to 14336 columns
    // and sums.  By the estimate's own rounds a stage took 0.42 to 0.67, 0.98 to 1.48 and 1.1 to 1.9.  Tiles of 160
    // rows were the best by 4% at most (4096 x 4096, 1024 rows: 291, 302 otherwise), and are left to one matrix.
    constexpr float kExperts[] = {0.42f, 0.96f, 0.0f, 1.5f};
    constexpr Cost k32[] = {{64, 64, 2, 2.2f, 0.62f, 1.05f}, {128, 128, 2, 2.9f, 2.0f, 3.5f}};
    // The same of rows that are not aligned.  fp32 by words, 1.01 to 1.2 times the above.  16 bits through registers,
    // of forward, input and weight (4095 x 4095, aligned 4096 x 4096 in brackets: 256 rows 26.5 (23.5), 2047 rows 99
    // (63); rows' gradients 35.5 (29) and 122 (71), weights' 31 (17) and 133 (58).  All rows at addresses of an odd
    // number of elements cost half as much again as those at multiples of four bytes: 512 rows 70, 44 and, staged but
    // aligned, 37).
    constexpr Cost k32Odd[] = {{64, 64, 2, 2.2f, 0.8f, 1.12f}, {128, 128, 2, 2.9f, 2.25f, 3.7f}};
    constexpr Cost k16Odd[][2] = {{{64, 64, 2, 2.2f, 0.4f, 0.74f}, {128, 128, 2, 2.9f, 1.0f, 1.5f}},
                                  {{64, 64, 2, 2.2f, 0.62f, 0.8f}, {128, 128, 2, 2.9f, 1.33f, 1.87f}},
                                  {{64, 64, 2, 2.2f, 0.73f, 0.76f}, {128, 128, 2, 2.9f, 1.55f, 2.0f}}};
    constexpr float kExpertsOdd[] = {0.95f, 1.9f};
    const Cost *const costs = odd ? fp32 ? k32Odd : k16Odd[input ? 1 : weight ? 2 : 0] : fp32 ? k32 : k16;
    RowsChoice best{kRowsTile128, 0, 1};
    double least = 0;
    // The large tiles write whole groups of eight columns.
    const int kinds = fp32 || odd || P % 8 != 0 ? 2 : (int)kRowsTileKinds;
    for (int tile = copied ? kRowsTile128 : kRowsTile64; tile < kinds; ++tile) {
        if ((weight || n_experts > 0) && tile == kRowsTile160) continue;
        Cost c = costs[tile];
        if (n_experts > 0 && !weight && !fp32)
            c.two = odd ? kExpertsOdd[tile] : kExperts[tile], c.one = std::max(c.one, c.two / c.a_cu);
        // Row tiles in all: of experts the mean over a spread of a third of their rows, as routers have.
        double tiles_q, stages;
        if (weight) {
            tiles_q = experts * halves * ((Q + c.q - 1) / c.q), stages = (mean + step - 1) / step;
            if (n_experts > 0) stages += 0.5;
        } else {
            stages = (double)halves * ((K + step - 1) / step);
            tiles_q = 0;
            const double spread = n_experts == 0 ? 0 : mean / 3 + std::sqrt(mean);
            for (int i = -2; i <= 2; ++i) tiles_q += std::ceil(std::max(1.0, mean + 0.6 * i * spread) / c.q) / 5;
            tiles_q *= experts;
        }
        const double tiles = tiles_q * ((cols + c.p - 1) / c.p);
        for (int slices : {1, 2, 3, 4, 5, 6, 8}) {
            const double per = std::ceil(stages / slices), n = std::ceil(tiles * slices), slots = (double)kCus * c.a_cu;
            if (slices > 1 && (per < 8 || tile > kRowsTile128)) break;
            double us;
            if (n_experts > 0 && n > slots / 2) {  // how full the last round is nobody knows: half of one on average
                us = std::max(n / slots + 0.5, 1.0) * (c.fixed + c.two * per);
            } else {
                const double full = std::floor(n / slots), rest = n - full * slots;
                us = full * (c.fixed + c.two * per);
                if (rest > 0) us += c.fixed + (rest <= kCus ? c.one : c.two) * per;
            }
            if (slices > 1) us += 3 + 8e-6 / 4 * slices * (double)cols * (weight ? (double)Q * halves * experts : Q);
            if (least == 0 || us < least) least = us, best = {tile, 0, slices};
        }
    }
    return best;
}

// About four workgroups a CU, two rows a wave at least.  bf16, us with the join: 2048 x 4096 silu 15.9, 4096 x 14336
// 83, 4096 x 4096 without an activation 9.4; with two a CU 19.5, 133, 11.4; with eight 15.9, 77, 11.7.  Two or four of
// a wave's rows loaded at once are no faster (two a CU: 19.8 and 20.3, 134 and 137).
int rows_column_chunks(int T, int N) {
    const int64_t across = ((int64_t)N + kRowsColumns - 1) / kRowsColumns;
    return (int)std::max<int64_t>(1, std::min<int64_t>(1024 / across, ((int64_t)T + 7) / 8));
}

}  // namespace jjo
