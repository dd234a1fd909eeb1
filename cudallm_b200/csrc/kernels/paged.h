// Launchers of the paged-cache operators and of beam search's selection. The ABI layer (capi/paged_capi.cpp) has
// checked every argument that the host can see; the kernels bound what it cannot (lengths, tables, positions).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "cudallm.h"

namespace cudallm {

constexpr int kMaxBeams = 64;
constexpr int kMaxKeep = 64;
constexpr int kMaxVocab = 1 << 24;
constexpr int kMaxPageRows = 65536;

void launch_paged_attend(const cudallm_pages& pg, const cudallm_attend_args& a, cudaStream_t stream);
size_t attend_workspace_bytes();

void launch_paged_append(const cudallm_pages& pg, const cudallm_append_args& a, cudaStream_t stream);

void launch_paged_fork(const cudallm_pages& pg, const cudallm_fork_args& a, cudaStream_t stream);
void launch_paged_compact(const cudallm_pages& pg, const cudallm_compact_args& a, cudaStream_t stream);
size_t pages_workspace_bytes(int n_pages, int rows);

void launch_beam_select(const cudallm_beam_args& a, cudaStream_t stream);
size_t beam_workspace_bytes(int rows, int vocab, int keep);

}  // namespace cudallm
