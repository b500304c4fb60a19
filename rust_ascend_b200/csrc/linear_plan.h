// Which kernel of the 8-bit linear (linear_i8.cu) takes a call.  Plain host code, so that the choice can be checked without a GPU.
#pragma once
#include <cstdint>

constexpr uint32_t RB_LINEAR_ROWS = 128;      // weight rows of a CTA's tile
constexpr uint32_t RB_LINEAR_BK = 128;        // K of a stage

// tokens 0: a warp per `rows` weight rows; parts 0: CTA pairs on tiles of `tokens` tokens; else tiles of `tokens` tokens with K shared by `parts`
// CTAs of a cluster.
struct rb_linear_plan { uint32_t tokens, parts, rows; };

// Weight rows a warp: more of them mean fewer loads of x and fewer warps.  us for n x k and m tokens at 1 / 2 / 4: 1024 x 4096, 1: 3.0 / 3.7 / 5.3;
// 6144 x 4096, 1: 6.8 / 5.9 / 7.2; 6144 x 4096, 4: - / 9.1 / 6.9; 4096 x 4096, 4: 6.6 / 6.2 / 6.1.
inline uint32_t rb_linear_rows_of(uint32_t m, uint32_t n, uint32_t sms) {
    if (m == 1) return n <= 32 * sms ? 1 : 2;
    if (m == 2) return n <= 16 * sms ? 1 : 2;
    return n <= 32 * sms ? 2 : 4;
}

// By the sizes alone: the least of estimated times in us.  The constants were fitted to 4774 sizes of 3 to 700 tokens (random ones
// and layers of 1024 to 28672 outputs), each timed with every tile and split; what is chosen takes 1.02 to 1.03 of the best one's time
// on average, 1.12 in nine of ten cases, where borders in tokens and K took 1.22 and 1.11 on average.  K is shared by a power of two of CTAs:
// 3 and 6 were timed as well and gained 0.3 % on average.  The terms are the kernels' own:
//   * few tokens: a start; the stages of a CTA's part of K, each at its latency or, where two CTAs share an SM, at the rate of the SM's
//     port to L2 (rows that do not start on cache lines pass it slower), at least the weights' way out of DRAM; the stores; the join
//     of the parts; a further wave, which clusters reach earlier because they do not fill every SM.
//   * pairs: a start and the rounds of tiles.
// sms, pairs: SMs and CTA pairs that the call may use.  limited: other SMs are to stay free.  The pairs keep to their number by themselves; the
// other kernels are offered only while they have no more CTAs than that, so that they cannot spread further.
inline rb_linear_plan rb_linear_plan_of(uint32_t m, uint32_t n, uint32_t k, uint32_t sms, uint32_t pairs, bool limited) {
    const uint32_t num_kb = (k + RB_LINEAR_BK - 1) / RB_LINEAR_BK;
    // One or two tokens, and up to four over short rows: no tensor core, no set-up (one token, 6144 x 4096: 5.9 us against 7.8; four tokens: K of
    // 1536 0.85 to 1.09 of the tiles' time, K of 4096 1.1 to 1.2).
    if (m <= 2 || (m <= 4 && num_kb < 24)) {
        const uint32_t rows = rb_linear_rows_of(m, n, sms);
        if (!limited || (n + 4 * rows - 1) / (4 * rows) <= sms) return {0, 0, rows};
    }
    auto up = [](uint64_t a, uint64_t b) { return (a + b - 1) / b; };
    auto larger = [](double a, double b) { return a > b ? a : b; };
    const bool aligned = k % RB_LINEAR_BK == 0;
    const double weights = (double)n * k * 1e-6;
    rb_linear_plan best{256, 0, 0};
    double least = 1e300;
    auto offer = [&](uint32_t tokens, uint32_t parts, double us) { if (us < least) { least = us; best = {tokens, parts, 0}; } };
    for (uint32_t tokens = 16; tokens <= 128 && (tokens == 16 || tokens < 2 * m); tokens *= 2) {
        const double used = m < tokens ? m : tokens;
        const double latency = 0.195 + 0.0009 * tokens, port = 0.0009 * (RB_LINEAR_ROWS + tokens) * (aligned ? 1.0 : 1.37);
        for (uint32_t parts = 1; parts <= 8 && parts <= num_kb; parts *= 2) {
            const uint64_t ctas = up(n, RB_LINEAR_ROWS) * up(m, tokens) * parts;
            if (limited && ctas > sms) break;
            const uint32_t spare = sms > 32 ? sms : 33;
            const uint32_t seats = parts < 4 ? sms : parts == 4 ? spare - 8 : spare * 13 / 16, wave = parts < 4 ? 2 * sms : parts == 4 ? 2 * spare - 32 : seats;
            const uint64_t share = up(ctas, seats);      // CTAs of the fullest SM
            const double body = up(num_kb, parts) * ((double)(share / 2) * larger(latency, 2 * port) + (double)(share % 2) * larger(latency, port)) + 0.0125 * used * share / parts;
            offer(tokens, parts, 1.85 + 1.4 * (double)(up(ctas, wave) - 1) + larger(body, weights / 5.1) + (parts > 1 ? 0.78 + 0.031 * used : 0.0));
        }
    }
    if (m > 16 || limited) {
        for (uint32_t tokens = 128; tokens <= 256; tokens *= 2) {
            const uint64_t tiles = up(n, 2 * RB_LINEAR_ROWS) * up(m, tokens), rest = tiles % pairs;
            const double halves = tiles < pairs ? 0.72 : 0.63;      // a short last round runs as half tiles, partly under the round in front
            const double rounds = (double)(tiles / pairs) + (rest == 0 ? 0.0 : 2 * rest <= pairs ? halves : 1.0);
            const double tile = num_kb * (0.150 + 0.0006 * tokens) * (aligned ? 1.0 : 1.23) + 0.0104 * (m < tokens ? m : tokens);
            offer(tokens, 0, 3.2 + larger(rounds * tile, weights / 4.6));
        }
    }
    return best;
}
