// Bits of the status word for indexes that a kernel met outside their range (bit 30: the embedding lookup).
#pragma once

namespace b200q {

constexpr unsigned int kBadPosition = 1u << 29;  // a rotary position outside the table
constexpr unsigned int kBadSlot = 1u << 28;      // a slot outside the cache
constexpr unsigned int kBadPage = 1u << 27;      // a page outside the cache, or a length beyond its row of the page table
constexpr unsigned int kBadToken = 1u << 26;     // a token outside the vocabulary
constexpr unsigned int kBadStarts = 1u << 25;    // sequences' first rows that fall, or lie outside the rows

}  // namespace b200q
