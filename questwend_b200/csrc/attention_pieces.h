// How many pieces the keys of a step are best cut into by the tcgen05 prompt kernel (attention_tc.cu), and what it then takes.  A block of it,
// 128 rows, takes about 1.05 us a tile of 64 keys (0.95 with heads of 64) and 3.5 of its own; 296 run at once; with pieces there is a join, which
// reads what they leave.
#pragma once

struct AtPieces { int pieces, tiles; double us; };

static inline AtPieces at_pieces(long long T, int B, int max_new, int max_len, int Hq, int Hkv, int hd, int window) {
    const int G = Hq / Hkv, tok = G <= 128 ? 128 / G : 1;
    const double blocks = (double)B * Hkv * ((max_new + tok - 1) / tok), tile_us = hd == 128 ? 1.05 : 0.95;
    const long long keys = window > 0 && (long long)window + tok < max_len ? (long long)window + tok : max_len, tiles = (keys + 63) / 64 + 1;
    // whole: the longest block, or what all of them have to do (of a prompt that begins its sequence half the keys)
    double mean = max_len - 0.5 * (max_new < max_len ? max_new : max_len);
    if (window > 0 && window < mean) mean = window;
    const double spread = blocks / 296.0 * mean / 64.0;
    AtPieces best = {1, (int)tiles, 3.5 + (spread > tiles ? spread : (double)tiles) * tile_us};
    if (blocks < 4 * 296) {
        for (int s = 2; s <= 64 && s <= tiles; ++s) {
            const long long p = (tiles + s - 1) / s, waves = (long long)((blocks * s + 295) / 296);
            const double us = waves * (p * tile_us + 3.5) + 4.0 + (double)T * Hq * s * hd * 8 / 4e6;
            if (us < 0.95 * best.us) best = {s, (int)p, us};
        }
    }
    return best;
}
