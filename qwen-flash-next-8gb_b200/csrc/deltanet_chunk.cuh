// The chunked kernels of qfn_deltanet_chunk (deltanet_chunk.cu), for its
// entry point in deltanet_batch.cu.
#pragma once

#include "deltanet_batch.cuh"

namespace qfn {

// Up to so many tokens in all, the token recurrence is faster than the chunked kernels.
constexpr int64_t kRecurrenceTokens = 8;

bool dn_chunk_takes(int64_t tokens, int dk);
size_t dn_chunk_workspace(int64_t tokens, int64_t n_seqs, int n_heads, int n_key_heads, int dk);
int dn_chunk(const DnRows& a, const int32_t* cu, int64_t n_seqs, int64_t tokens, int dk, const DeviceInfo& dev,
             void* workspace, qfn_stream_t stream);

}  // namespace qfn
