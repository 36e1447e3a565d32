// The chunked kernels of qfn_deltanet_chunk (deltanet_chunk.cu), for its
// entry point in deltanet_batch.cu.
#pragma once

#include "deltanet_batch.cuh"

namespace qfn {

// Where no sequence is longer, the token recurrence is faster than the chunked
// kernels, whose preparation costs the same for one token as for 64.  Equal
// sequences of 1 / 8 / 12 / 16 tokens, 32 heads of 128 x 128, recurrence against
// chunks in us: 16 of them 12/42/60/78 against 66/67/67/68, 64 of them
// 34/143/207/275 against 230/232/234/235, 256 of them 126/648/936/1226 against
// 882/887/890/894; one sequence of 8 / 10 tokens 11/17 against 15/15.
constexpr int64_t kRecurrenceTokens = 8;

// `longest`: a bound on the sequences' lengths, all the tokens where only the device knows them.
bool dn_chunk_takes(int64_t longest, int dk);
size_t dn_chunk_workspace(int64_t tokens, int64_t n_seqs, int n_heads, int n_key_heads, int dk);
int dn_chunk(const DnRows& a, const int32_t* cu, int64_t n_seqs, int64_t tokens, int dk, const DeviceInfo& dev,
             void* workspace, qfn_stream_t stream);

}  // namespace qfn
