// Selective state-space scan over prompts for gfx950.
#include "gdn_seq.h"
#include "gdn_ssm.h"

#include <algorithm>

namespace gdn {
namespace {

constexpr int kMaxBlock = 1 << 20;

bool scan_sizes_ok(const gdn_ssm_inputs* in, int seqs, int block, bool packed) {
    return ssm_sizes_ok(in) && seqs >= 1 && block >= kChunk && block <= kMaxBlock &&
           block % kChunk == 0 && (packed ? in->batch == 1 : seqs == in->batch);
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_ssm_scan_block(const gdn_ssm_inputs* in, int num_seqs) {
    if (!ssm_sizes_ok(in) || num_seqs < 1) return 0;
    return 64;
}

extern "C" size_t gdn_ssm_scan_workspace_size(const gdn_ssm_inputs* in, int num_seqs, int block,
                                              int packed) {
    if (!scan_sizes_ok(in, num_seqs, block, packed != 0)) return 0;
    return 256;
}

extern "C" hipError_t gdn_ssm_scan(const gdn_ssm_inputs* in, void* y, const float* s0, float* sf,
                                   const int32_t* cu_seqlens, const int32_t* blocks, int num_seqs,
                                   int block, void* workspace, size_t workspace_bytes,
                                   hipStream_t stream) {
    if (!ssm_inputs_ok(in) || !scan_sizes_ok(in, num_seqs, block, cu_seqlens != nullptr) || (blocks && !cu_seqlens))
        return hipErrorInvalidValue;
    if (!sf || !ssm_aligned(sf, 4) || !ssm_aligned(s0, 4) || (in->tokens > 0 && !y) ||
        !ssm_aligned(y, 16) || !ssm_aligned(workspace, 256) || !ssm_aligned(blocks, 16))
        return hipErrorInvalidValue;
    const size_t need = gdn_ssm_scan_workspace_size(in, num_seqs, block, cu_seqlens != nullptr);
    if (need == 0 || !workspace || workspace_bytes < need) return hipErrorInvalidValue;
    return ssm_recurrent(*in, y, s0, sf, cu_seqlens, num_seqs, stream);
}
