// How the gradient of a token table is put on a GPU, as far as that goes by numbers alone: the host's part, without CUDA.
#pragma once

#include <stdint.h>

namespace tbe {

constexpr int kSortThreads = 1024;
constexpr int kSortBlocks = 16;                      // the largest cluster; a GPC of a whole GPU has as many multiprocessors
constexpr int kMostItems = 16;                       // keys to a thread
constexpr int64_t kOneBlockKeys = 2 * kSortThreads;  // so many are sorted by a block alone: 4096 take 16 us in one, 12 in a cluster
constexpr int64_t kClusterKeys = int64_t(kSortBlocks) * kMostItems * kSortThreads;

enum class SortForm { kBlock, kCluster, kTiles };

// `cluster_fits`: the device can hold a cluster of kSortBlocks at all (a partition of a GPU may not).
inline SortForm sort_form(int64_t n, bool cluster_fits)
{
    if (n <= kOneBlockKeys) return SortForm::kBlock;
    return n <= kClusterKeys && cluster_fits ? SortForm::kCluster : SortForm::kTiles;
}

// Blocks that clear `bytes` in the launch of a sort by `cluster` blocks: 64 KB each at least, one per multiprocessor that the sort
// leaves at most, and whole clusters of them, as a grid has to be.  0 where there is no room: then a launch of its own clears.
inline int64_t clearing_blocks(int64_t bytes, int sms, int cluster)
{
    const int64_t want = (bytes + 65535) / 65536, room = sms > cluster ? (sms - cluster) / cluster * cluster : 0;
    const int64_t whole = (want + cluster - 1) / cluster * cluster;
    return whole < room ? whole : room;
}

}  // namespace tbe
