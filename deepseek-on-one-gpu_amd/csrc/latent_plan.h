// Arithmetic of the split plan of latent_attention, apart from the wave that carries it out.
//
// Tables of many sequences may share pages, so that the tiles of a call pass 2^31: up to 2^26 in each of
// 65535 sequences.  The sums over a wave are of 32 bits: a lane's, of up to 1024 sequences, goes in two parts.
#pragma once

#include <cstdint>

namespace amla {

constexpr int PLAN_PART = 12;  // 64 lanes' low parts stay below 2^18, their high ones at or below 2^30
constexpr int plan_low(int64_t sum) { return (int)(sum & ((1 << PLAN_PART) - 1)); }
constexpr int plan_high(int64_t sum) { return (int)(sum >> PLAN_PART); }
constexpr int64_t plan_total(int low, int high) { return ((int64_t)high << PLAN_PART) + low; }

// Lengths of a split between which the smallest one is whose splits of all sequences, times the chunks, fit the slots.  total:
// tiles of all sequences; most: of the longest.  slots >= chunks * seqs, or chunks * seqs + 128: hi fits since total / hi +
// chunks * seqs slots are enough.
struct PlanRange {
  int lo, hi;
};
constexpr PlanRange plan_range(int64_t total, int most, int chunks, int seqs, int slots) {
  const int64_t units = total * chunks, spare = slots - (int64_t)chunks * seqs;
  const int64_t least = (units + slots - 1) / slots, enough = units / (spare > 1 ? spare : 1) + 1;
  const int lo = least > 1 ? (int)least : 1, top = enough < most ? (int)enough : most;
  return PlanRange{lo, top > lo ? top : lo};
}

}  // namespace amla
