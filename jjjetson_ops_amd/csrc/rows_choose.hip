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
// x 14336 over 4096 on tiles of 256 / 160 / 128 rows 198 / 225 / 228 (191 / 232 / 267); 2048 x 4096 over 4096
// 90 / 76 / 64 (96 / 78 / 67); 64 x 4096 over 4096 on tiles of 64 x 64 in 1, 2, 4 slices 22.9 / 17.7 / 13.9
// (25 / 19 / 14).
RowsChoice rows_mm_choose(RowsMode mode, int dtype, int P, int Q, int K, int halves, int n_experts) {
    constexpr int64_t kCus = 256;
    const bool fp32 = dtype == JJO_DTYPE_F32, weight = mode == kRowsWeight;
    const int step = fp32 ? 32 : 64;
    const int64_t cols = mode == kRowsSwiglu ? 2LL * P : P;  // columns of tiles
    // Experts with rows, as far as it is known without reading the offsets, and the rows (sums) of one.
    const int M = weight ? K : Q;
    const double experts = n_experts == 0 ? 1 : std::min(n_experts, M), mean = M / experts;

    // Few rows: a matrix is best read by the direct kernel up to 16 rows, up to 12 where tiles of 64 columns
    // occupy every other CU (11008 x 4096: 1 / 8 / 16 rows 18.1 / 21.2 / 25.0 us against 23.6 / 23.9 / 23.9 on tiles;
    // 4096 x 4096 16 rows 10.6 against 12.9 in four slices).  Of experts only where the tiles leave CUs without two
    // workgroups and rows are long (8 rows of 8 experts, 4096 x 14336: 100 against 122 us; 14336 x 4096: 108
    // against 104; SwiGLU of 64 experts' 1408 x 2048: 19.5 against 16.5).
    const int64_t tiles64 = (cols + 63) / 64;
    const bool few = n_experts == 0 ? Q <= (tiles64 < kCus / 2 ? 16 : 12)
                                    : mean <= 4 && K >= 4096 && (int64_t)experts * tiles64 < 3 * kCus;
    if (few && (mode == kRowsForward || mode == kRowsSwiglu)) {
        const int64_t wgs = (int64_t)experts * ((cols + 15) / 16);
        return {kRowsDirect, wgs >= 4 * kCus ? 2 : 8, 1};  // as above on 2, 4, 8 waves: 100, 111, 110; 1 row 19.0, 18.8, 18.1
    }

    struct Cost {
        int p, q, a_cu;
        float fixed, one, two;
    };
    constexpr Cost k16[] = {{64, 64, 2, 2.2f, 0.35f, 0.5f}, {128, 128, 2, 2.9f, 0.65f, 1.0f},
                            {256, 160, 1, 5.f, 1.13f, 1.13f}, {256, 256, 1, 6.f, 1.4f, 1.4f}};
    // A stage of experts' rows, where few tiles share a matrix's rows and wait for memory.
    constexpr float kExperts[] = {0.5f, 1.3f, 1.4f, 1.9f};
    constexpr Cost k32[] = {{64, 64, 2, 2.2f, 0.62f, 1.05f}, {128, 128, 2, 2.9f, 2.0f, 4.0f}};
    const Cost *const costs = fp32 ? k32 : k16;
    RowsChoice best{kRowsTile128, 0, 1};
    double least = 0;
    for (int tile = 0; tile < (fp32 ? 2 : (int)kRowsTileKinds); ++tile) {
        if (weight && tile == kRowsTile160) continue;
        Cost c = costs[tile];
        if (n_experts > 0 && !weight && !fp32) c.two = kExperts[tile], c.one = std::max(c.one, c.two / c.a_cu);
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
        for (int slices : {1, 2, 3, 4, 6, 8}) {
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

// About four workgroups a CU, two rows a wave at least.  bf16, us with the join: 2048 x 4096 silu 15.9, 4096 x 14336 83,
// 4096 x 4096 without an activation 9.4; with two a CU 19.5, 133, 11.4; with eight 15.9, 77, 11.7.  Two or four of
// a wave's rows loaded at once are no faster (two a CU: 19.8 and 20.3, 134 and 137).
int rows_column_chunks(int T, int N) {
    const int64_t across = ((int64_t)N + kRowsColumns - 1) / kRowsColumns;
    return (int)std::max<int64_t>(1, std::min<int64_t>(1024 / across, ((int64_t)T + 7) / 8));
}

}  // namespace jjo
