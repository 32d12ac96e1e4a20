// Who joins the parts of a tile that several blocks took: the last one to deliver, found by a ticket in global memory.
// One thread of a block asks, and tells the others by a word in shared memory.
//
// Team is the block's threads that join: leads() is true for the one that asks; meet() is true when all have come, and
// what they wrote before is then visible to all, or false when the caller has waited for too long (a warp gave up
// somewhere, and will not come): the answer is then no, team.ok is false from then on, and the caller leaves too; read / write are for the shared words, held (acquire), take (adds one,
// acquire and release, returns the value before) and clear for tickets. The functions know no more of the device than that, so
// that they also run on the host, with threads for warps that a test delays where it likes (tests/test_join_host.py).
#pragma once

#ifdef __CUDACC__
#define MKX_TEAM_FN __device__ __forceinline__
#else
#define MKX_TEAM_FN inline
#endif

namespace mkxa {

// A word for each question: a warp may still be on its way to read `last` while the next tile's others_done, which
// writes before its first meet(), is under way.
struct JoinWords {
  int last, others;
};

// Whether the other parts - 1 blocks of a tile have all delivered: then this one keeps its part to itself, and joins.
// Leaves the ticket at zero if so. The others' parts are then visible past L1 (__ldcg).
template <class Team, class Words>
MKX_TEAM_FN bool others_done(Team& team, unsigned* ticket, int parts, Words& words) {
  if (team.leads()) {
    const bool all = team.held(ticket) == (unsigned)parts - 1;
    team.write(&words.others, all);
    if (all) team.clear(ticket);
  }
  if (!team.meet()) return false;
  const bool all = team.read(&words.others);
  return team.meet() && all;  // the word is free again
}

// Called after the team wrote its part of a split tile past L1 (__stcg): whether this block is the last of n under
// `ticket`, which is then left at zero. The others' parts are then visible past L1: what a team wrote before its
// meet() is released by the one thread that takes the ticket.
template <class Team, class Words>
MKX_TEAM_FN bool last_of(Team& team, unsigned* ticket, int n, Words& words) {
  if (!team.meet()) return false;
  if (team.leads()) {
    const bool last = team.take(ticket) == (unsigned)n - 1;
    team.write(&words.last, last);
    if (last) team.clear(ticket);
  }
  return team.meet() && team.read(&words.last);  // written again only behind the first meet() of the next last_of
}

}  // namespace mkxa
