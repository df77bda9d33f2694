// Products on 8-bit integers: which form a call takes, a function of its sizes alone.
#pragma once
#include <stdint.h>

namespace icua {

// That of the least time by a model of each form,
//   start + n each + steps max(late ceil(n / beside), busy n)  us,
// n tiles a CU (256 CUs), steps of 128 codes a wave group, `beside` tiles that a CU holds at a time, `late` the time of
// a step that waits for memory, `busy` of one that has the CU to itself (where beside is 1 the two are one).  The four
// times are fitted to each form's measured ones over 8 to 4096 tokens, 1024 to 12288 channels and depths of 1024 to
// 6144 (root mean square of their ratios 5 to 16 %); the form taken is 3 % slower than the best one on average, also of
// 200 to 6000 tokens, 512 to 6144 channels and depths of 512 to 12288.  128 x 128 tiles alone: 12.6 us for 64 tokens,
// 4096 channels, 2048 deep, where 32 x 32 tiles take 5.6, and 133 us for 4096 tokens of gated 6144, where 256 x 256
// tiles take 107; 256 x 256 tiles alone 23 us for the former.
struct I8Form {
    int tokens, channels, gated_channels, parts, beside;  // of a tile (0: not for gates); groups of waves
    float start, each, late, busy;
};
enum I8FormId {
    I8_STREAM_16, I8_STREAM_32, I8_64x128, I8_128x128, I8_128x256, I8_256x256, I8_32x32, I8_32x64, I8_64x64_DEEP, I8_64x64,
    I8_128x256_DEEP,
    I8_FORMS
};
constexpr int I8_STREAM_ROWS = 128;  // many more tokens would be many small workgroups
constexpr I8Form I8_FORM[I8_FORMS] = {
    {16, 16, 16, 8, 2, 2.05f, 0.13f, 0.835f, 0.864f},
    {32, 16, 16, 8, 2, 2.18f, 0.13f, 1.164f, 1.183f},
    {64, 128, 64, 1, 2, 1.59f, 2.40f, 0.433f, 0.363f},
    {128, 128, 64, 1, 2, 0.12f, 3.51f, 0.686f, 0.572f},
    {128, 256, 128, 1, 1, 0.00f, 4.79f, 0.910f, 0.910f},
    {256, 256, 128, 1, 1, 0.00f, 8.11f, 1.219f, 1.219f},
    {32, 32, 0, 8, 1, 0.77f, 2.56f, 0.990f, 0.990f},
    {32, 64, 0, 4, 1, 0.04f, 3.74f, 0.639f, 0.639f},
    {64, 64, 0, 1, 2, 1.79f, 1.47f, 0.296f, 0.221f},
    {64, 64, 0, 1, 4, 0.57f, 1.25f, 0.487f, 0.212f},
    {128, 256, 128, 1, 1, 0.00f, 4.79f, 0.910f, 0.910f},  // (that of two stages, see below)
};

inline int64_t i8_tiles(const I8Form& f, bool gated, int n_rows, int n_out) {
    const int channels = gated ? f.gated_channels : f.channels;
    return (int64_t)((n_rows + f.tokens - 1) / f.tokens) * ((n_out + channels - 1) / channels);
}

inline float i8_time(const I8Form& f, bool gated, int n_rows, int n_out, int n_in) {
    const int64_t tiles = i8_tiles(f, gated, n_rows, n_out);
    const float n = (float)((tiles + 255) / 256), rounds = (float)((tiles + 256 * f.beside - 1) / (256 * f.beside));
    const int steps = ((n_in + 127) / 128 + f.parts - 1) / f.parts;
    const float late = f.late * rounds, busy = f.busy * n;
    return f.start + n * f.each + steps * (late > busy ? late : busy);
}

// 128 x 256 tiles, of which there are more than 128 where they are taken, have three stages beyond this depth, so that
// memory is waited for less, else two, which start sooner.  Time with three to that with two, means over 200 to 6000
// tokens and 512 to 6144 channels, of up to 256 / more tiles: 1.03 / 1.04 at 1024, 1.02 / 1.02 at 2048, 0.99 / 0.99 at
// 2560, 1.00 / 0.99 at 4096, 0.97 / 0.94 at 5120, 6144 and 7168, 0.87 / 0.86 at 12288; 256 tiles of 4096 tokens 1.01 at
// 2560 and 4096.  (With times for each of the two the model takes the same forms.)
constexpr int I8_TWO_STAGES = 4096;

inline I8FormId i8_form(bool gated, int n_rows, int n_out, int n_in) {
    int best = -1;
    float least = 0.f;
    for (int i = 0; i < I8_128x256_DEEP; ++i) {
        const I8Form& f = I8_FORM[i];
        if ((gated && !f.gated_channels) || (n_rows > I8_STREAM_ROWS && i <= I8_STREAM_32)) continue;
        const float us = i8_time(f, gated, n_rows, n_out, n_in);
        if (best < 0 || us < least) best = i, least = us;
    }
    if (best == I8_128x256 && n_in > I8_TWO_STAGES) best = I8_128x256_DEEP;
    return (I8FormId)best;
}

}  // namespace icua
