// How many pieces the keys of a step are best cut into by the tcgen05 prompt kernel (attention_tc.cu), and what it then takes.  A block of it,
// 128 rows, takes about 0.82 us a tile of 64 keys alone on an SM and 1.12 beside another (0.72 and 1.0 with heads of 64), and 4 of its own; 296
// run at once; beyond that blocks follow one another, and the last ones to start add about 0.3 of a block.  With pieces there is a join, which reads
// what they leave.  Of 60 steps (new tokens 64 to 4,500, 8,000 behind them or 30,000, heads of both sizes) 1 to 14 pieces were measured: this choice
// takes 1.7 % more than the best of them on average, at most 21 %; one piece always takes 47 % more, and 8 times as much for one sequence of
// 64 new tokens behind 30,000.
#pragma once

struct AtPieces { int pieces, tiles; double us; };

static inline AtPieces at_pieces(long long T, int B, int max_new, int max_len, int Hq, int Hkv, int hd, int window, int most = 64) {
    const int G = Hq / Hkv, tok = G <= 128 ? 128 / G : 1;
    // blocks with rows: of equal sequences B times the longest one's; of unequal ones (a prompt beside single tokens) no more than all tokens fill, and one each
    const double longest_each = (double)B * ((max_new + tok - 1) / tok), filled = (double)T / tok + B;
    const double blocks = Hkv * (longest_each < filled ? longest_each : filled), alone = hd == 128 ? 0.82 : 0.72, beside = hd == 128 ? 1.12 : 1.0;
    const long long keys = window > 0 && (long long)window + tok < max_len ? (long long)window + tok : max_len, tiles = (keys + 63) / 64 + 1;
    double mean = max_len - 0.5 * (max_new < max_len ? max_new : max_len);              // keys of a row (of a prompt that begins its sequence half)
    if (window > 0 && window < mean) mean = window;
    const double all = blocks * (mean / 64.0 + 1.2) / 296.0;                            // tiles that each of 296 places has to take
    auto takes = [&](double count, double longest) {
        if (count <= 148) return longest * alone + 4.0;
        if (count <= 296) return longest * beside + 4.0;
        return (all + 0.3 * longest > longest ? all + 0.3 * longest : longest) * beside + 4.0 * count / 296.0;
    };
    AtPieces best = {1, (int)tiles, takes(blocks, (double)tiles)};
    if (blocks < 4 * 296) {
        for (int s = 2; s <= most && s <= tiles && (long long)s * B <= 65535; ++s) {       // (the grid's bound)
            const long long p = (tiles + s - 1) / s;
            const double us = takes(blocks * s, (double)p) + 4.0 + (double)T * Hq * s * hd * 8 / 5e6;
            if (us < 0.98 * best.us) best = {s, (int)p, us};
        }
    }
    return best;
}
