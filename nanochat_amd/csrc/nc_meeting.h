/*
 * How the workgroups that share a row in sample.hip's split_kernel wait for one another, apart from the kernel so that a
 * host program can replay it.
 *
 * A waiting workgroup keeps its place on a CU, and the ones that it waits for may not have one: with n launches at once,
 * or on a device of few CUs, all places can be held by workgroups that wait (an XCD has 64 places of the 16-token form, and
 * each launch can have 31 workgroups of an unfinished row of 32 there). So no wait is unbounded. A workgroup that has
 * looked `patience` times gives the row up for all of them: they leave, each freeing its place, and the last to leave,
 * which needs nobody, does the row by itself.
 *
 * One word a row holds it all: arrivals at meetings (each workgroup adds 1 a meeting, and never looks for more than
 * `reached` = meetings so far x workgroups), workgroups that have left (MT_LEFT each), and whether the row was given up.
 * It is given up by a compare-and-swap against a word with fewer arrivals than the meeting needs, so never once that
 * meeting is over; and nobody passes a meeting while the mark is there. A workgroup that has not arrived at the next
 * meeting keeps the others from passing it. So either every workgroup of a row passes its last meeting, or none does: the
 * token is written once.
 */
#pragma once

#include <hip/hip_runtime.h>

namespace nc {

constexpr int MT_ARRIVALS = 0xFFFF, MT_LEFT = 1 << 16, MT_MOST_LEFT = 0xFF, MT_GIVEN_UP = 1 << 30;

enum Meeting { MT_WAIT, MT_OVER, MT_GONE };

/* A look at the row's word, `seen`: whether the meeting of `reached` arrivals is over, or the row given up, by others or
 * here, where the patience is used up. Word: bool swap(int &expected, int desired), which leaves what it found in
 * `expected` if that is not what was expected. Such a failure takes another workgroup's step, so few can follow. */
template <typename Word>
__host__ __device__ __forceinline__ Meeting meeting_look(Word &word, int &seen, int reached, int &patience) {
    if (seen & MT_GIVEN_UP) return MT_GONE;
    if ((seen & MT_ARRIVALS) >= reached) return MT_OVER;
    if (patience > 0) {
        patience--;
        return MT_WAIT;
    }
    return word.swap(seen, seen | MT_GIVEN_UP) ? MT_GONE : MT_WAIT;
}

/* Whether a workgroup that found `seen` when it added MT_LEFT is the last of G to leave. */
__host__ __device__ __forceinline__ bool meeting_last(int seen, int G) {
    return (seen / MT_LEFT & MT_MOST_LEFT) == G - 1;
}

}  // namespace nc
