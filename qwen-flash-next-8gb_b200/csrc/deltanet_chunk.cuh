// The chunked kernels of qfn_deltanet_chunk (deltanet_chunk.cu), for its
// entry point in deltanet_batch.cu.
#pragma once

#include "deltanet_batch.cuh"

namespace qfn {

// Whether sequences of up to `longest` tokens (all the tokens where only the device knows the lengths) take the
// chunked kernels, whose preparation and walk cost the same for one token as for 64, or the token recurrence: 1.0 to
// 1.2 us a token while its blocks of 32 columns have SMs of their own, then by dk dv.  Recurrence against chunks, in
// us in a graph, for equal sequences (states = sequences x heads):
//   128 x 128:   32 states, 10 tokens 13 / 13;   512, 12 60 / 71, 16 78 / 71;  8192, 12 936 / 952, 14 1081 / 955
//   128 x 64:    32 states, 10 tokens 13 / 13;   512, 16 49 / 54, 20 61 / 53;  8192, 16 631 / 707, 20 780 / 710
//   64 x 128:    32 states, 10 tokens 11 / 11;   512, 16 49 / 54, 20 60 / 54;  8192, 16 757 / 718
//   64 x 64:     16 states, 10 tokens 11 / 11;  1024, 24 71 / 73, 32 93 / 75;  4096, 24 282 / 278
//   64 x 32:      8 states, 10 tokens 11 / 11;   512, 24 29 / 36, 32 39 / 36
// More sequences never lower the limit, so what one sequence alone leaves to the recurrence, several do.
bool dn_chunk_takes(int64_t longest, int64_t n_seqs, int n_heads, int dk, int dv);
size_t dn_chunk_workspace(int64_t tokens, int64_t n_seqs, int n_heads, int n_key_heads, int dk);
int dn_chunk(const DnRows& a, const int32_t* cu, int64_t n_seqs, int64_t tokens, int dk, const DeviceInfo& dev,
             void* workspace, qfn_stream_t stream);

}  // namespace qfn
