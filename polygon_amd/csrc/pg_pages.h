// Launches of pg_pages.hip for callers whose counts are known on the device only (planes and pointers are the caller's care).
#pragma once
#include "pg_common.h"
#include "../../include/polygon_hip.h"

// groups_dev (nullable): only the first *groups_dev groups
int launch_pages_reorder(const pg_plane* planes, int n_planes, int n_groups, const int* groups_dev, int K, const int32_t* parents,
                         hipStream_t st);
// n_dev (nullable, not count itself): only the first *n_dev pages; map may be null
int launch_pages_compact(const pg_plane* planes, int n_planes, int n_pages, const int* n_dev, const uint8_t* live, int32_t* count,
                         int32_t* map, void* ws, hipStream_t st);
