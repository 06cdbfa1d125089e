// Which kernel of the 8-bit projection a call takes, and in which form (linear_quant.cu); plain C++ too, for the
// tests on the host.
#pragma once

namespace ma {

constexpr int kLinearSlab = 128;             // bytes of K per stage
constexpr int kMaxSplits = 6;                // parts of K, the CTAs of a cluster

// Which kernel, and in which form, by estimates of its time in nanoseconds (device time of a call in a chain
// of calls, beside a start and an end that all of them have; over 2900 random sizes the choice took 2 % longer
// than the best form would have on the average):
//   few tokens: a block of K takes 160 on an SM that has one CTA, parts have to be exchanged, and the tokens of
//   a tile written; a round beyond the first starts anew.  1 x 4096 x 10240: 3 parts 9.0 us, 2 11.0, 4 (two
//   rounds) 13.4; 17 x 1402 x 213: 6 parts 3.3, 3 3.7, 1 4.7; 10 x 16384 x 2304: 6 parts 9.7, 4 10.7, 3 11.4;
//   many tokens: rounds of a tile per pair of SMs; 4096 x 4096 x 4096: 256 channels 47 us, 128 53, 64 87;
//   1384 x 4096 x 1280: 14.3, 10.3, 14.9; 256 x 128 x 512: 4.5, 3.5, 2.9.
// Up to 32 tokens the first always, above 512 the second; in between 64 x 4096 x 4096 takes 8.4 by the first
// and 9.3 by the second, 64 x 512 x 512 4.1 and 3.3, 300 x 16384 x 2304 19.1 and 25.4, 272 x 930 x 24924 39 and 22.
struct LinearForm {
  long long tiles, time;
  int width, splits, stages;                 // channels of a tile, or tokens; parts of K (0: the kernel for many tokens)
};
inline LinearForm narrow_form(int tokens, int inner, int width, int tn, int sms) {
  constexpr int kParts[5] = {1, 2, 3, 4, kMaxSplits};
  constexpr int kRoom[5] = {100, 100, 94, 95, 91};      // % of two CTAs per SM: clusters leave some over
  const long long blocks = (inner + kLinearSlab - 1) / kLinearSlab;
  const long long tiles = (width + 127LL) / 128 * ((tokens + tn - 1LL) / tn);
  LinearForm best{0, 0, tn, 0, 0};
  long long least = 0;
  for (int i = 0; i < 5 && kParts[i] <= blocks; ++i) {
    const long long n = kParts[i], ctas = tiles * n, room = 2LL * sms * kRoom[i] / 100;
    const long long rounds = (ctas + room - 1) / room, last = ctas - (rounds - 1) * room, part = blocks * 160 / n;
    const long long time = (rounds - 1) * (2 * part + 4000) + part * ((last + sms - 1) / sms) +
                           (n > 1 ? 200 + 60 * n : 0) + (tn / 16 - 1) * (333 + 333 / n);
    if (i == 0 || time < least) least = time;
    // (of two about equal ones the one with more loads in flight: 1 x 8192 x 8192 4 parts 13.2, 2 14.2)
    if (i == 0 || time * 100 <= least * 107) best = {ctas, time, tn, static_cast<int>(n), 0};
  }
  return best;
}
inline LinearForm wide_form(int tokens, int inner, int width, int sms) {
  const long long blocks = (inner + kLinearSlab - 1) / kLinearSlab;
  constexpr int kEnd[3] = {150, 500, 860}, kRound[3] = {550, 830, 1440}, kBlock[3] = {160, 180, 290};
  LinearForm best{0, 0, 0, 0, 0};
  for (int i = 0; i < 3; ++i) {
    const long long tiles = (tokens + 255LL) / 256 * ((width + (64LL << i) - 1) / (64LL << i));
    const long long time = (tiles + sms / 2 - 1) / (sms / 2) * (kRound[i] + blocks * kBlock[i]) + kEnd[i];
    if (i == 0 || time < best.time) best = {tiles, time, 64 << i, 0, i == 0 ? 9 : i == 1 ? 7 : 5};
  }
  return best;
}
inline LinearForm linear_form(int tokens, int inner, int width, int sms) {
  if (tokens <= 512) {
    LinearForm f = narrow_form(tokens, inner, width, tokens <= 16 ? 16 : tokens <= 32 ? 32 : 64, sms);
    if (tokens <= 32 || f.time <= wide_form(tokens, inner, width, sms).time) {
      // An SM that has one CTA only gives it all of its shared memory, where its part is long enough to fill it
      // or SMs are left for the kernel behind this one (48 x 16384 x 2304: 10.9 us for 12.9; 1 x 1524 x 376 3.0 for
      // 3.6; but 16 x 4096 x 4096, 128 CTAs of 8 blocks, 6.7 for 6.1).  Clusters of three and more find no room on
      // some SMs.
      const bool deep = f.tiles <= (f.splits > 2 ? sms * 88 / 100 : sms) &&
                        (f.tiles * 4 <= sms * 3 || inner >= 10 * kLinearSlab * f.splits);
      f.stages = f.width == 16 ? (deep ? 11 : 6) : f.width == 32 ? (deep ? 10 : 5) : (deep ? 8 : 4);
      return f;
    }
  }
  return wide_form(tokens, inner, width, sms);
}

}  // namespace ma
