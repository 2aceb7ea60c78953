// C ABI (include/seedplane_hip.h) of beam search's selection.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "sp_host.h"
#include "sp_beam.h"

namespace {

// Parts of a row: blocks for every wave that the chip holds (8 a CU), as many lists as the merge takes, at least a chunk each.
int splits_of(int64_t rows, int beams, int vocab) {
    const int most = std::min({beam::MOST_SPLITS, beam::LISTS / beams, (vocab + beam::CHUNK - 1) / beam::CHUNK});
    return (int)std::max<int64_t>(1, std::min<int64_t>(most, std::max<int64_t>(beam::LEAST_SPLITS, 2048 / rows)));
}
void check_beams(int batch, int beams, int vocab, int n) {
    require(batch >= 0 && beams >= 1 && beams <= beam::MOST_BEAMS && n >= beams && n <= beam::MOST_N, SP_EINVAL,
            "n_batch must not be negative, n_beams in [1, 64] and n in [n_beams, 64]");
    require(vocab >= 1 && (int64_t)batch * beams <= 65535, SP_EINVAL, "vocab must be positive and n_batch * n_beams at most 65535");
    require(vocab < (1 << 30), SP_EINVAL, "vocab must be below 2^30");
}

template <class T>
void rows_of(const beam::Args &a, hipStream_t st) {
    const dim3 grid(a.splits, a.B * a.K), block(beam::THREADS);
    if (a.V < beam::VALUES) hipLaunchKernelGGL((beam::k_beam_rows<T, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((beam::k_beam_rows<T, false>), grid, block, 0, st, a);
}

}  // namespace

extern "C" {

size_t sp_op_beam_select_workspace(int32_t n_batch, int32_t n_beams, int32_t vocab, int32_t n) {
    if (n_batch < 1 || n_beams < 1 || n_beams > beam::MOST_BEAMS || vocab < 1 || n < 1 || n > beam::MOST_N) return 0;
    const size_t rows = (size_t)n_batch * n_beams;
    return rows * splits_of(rows, n_beams, vocab) * (n * sizeof(beam::Entry) + sizeof(float2));
}

int sp_op_beam_select(int32_t dtype, const void *logits_dev, int64_t ld, int32_t n_batch, int32_t n_beams, int32_t vocab,
                      const float *scores_dev, int32_t n, int32_t n_eos, const int32_t *eos, float *out_scores_dev, int32_t *out_beams_dev,
                      int32_t *out_tokens_dev, float *next_scores_dev, int32_t *next_rows_dev, int32_t *next_tokens_dev, void *workspace_dev,
                      void *stream) {
    return guarded([&] {
        require(dtype == SP_DT_F32 || dtype == SP_DT_F16 || dtype == SP_DT_BF16, SP_EINVAL,
                "dtype must be SP_DT_F32, SP_DT_F16 or SP_DT_BF16");
        check_beams(n_batch, n_beams, vocab, n);
        require(n_eos >= 0 && n_eos <= beam::MOST_EOS && (n_eos == 0 || eos), SP_EINVAL, "n_eos must be in [0, 8], with eos");
        require(n_batch * n_beams <= 1 || ld >= vocab, SP_EINVAL, "ld must be at least vocab");
        if (n_batch == 0) return;
        require(logits_dev && scores_dev && out_scores_dev && out_beams_dev && out_tokens_dev && next_scores_dev && next_rows_dev &&
                    next_tokens_dev && workspace_dev, SP_EINVAL, "NULL pointer");
        require(((uintptr_t)workspace_dev & 15) == 0, SP_EINVAL, "the workspace must be aligned to 16 bytes");
        beam::Args a{};
        a.logits = logits_dev; a.ld = ld; a.scores = scores_dev;
        a.B = n_batch; a.K = n_beams; a.V = vocab; a.n = n;
        const int64_t rows = (int64_t)n_batch * n_beams;
        a.splits = splits_of(rows, n_beams, vocab);
        a.by_splits = paged::Divisor(a.splits); a.by_n = paged::Divisor(n);
        a.len = ((vocab + a.splits - 1) / a.splits + beam::VALUES - 1) / beam::VALUES * beam::VALUES;
        a.best = (beam::Entry *)workspace_dev;
        a.sums = (float2 *)(a.best + rows * a.splits * n);
        a.out_score = out_scores_dev; a.out_beam = out_beams_dev; a.out_token = out_tokens_dev;
        a.next_score = next_scores_dev; a.next_row = next_rows_dev; a.next_token = next_tokens_dev;
        a.n_eos = n_eos;
        for (int i = 0; i < n_eos; ++i) a.eos[i] = eos[i];
        const hipStream_t st = (hipStream_t)stream;
        if (dtype == SP_DT_F32) rows_of<float>(a, st);
        else if (dtype == SP_DT_F16) rows_of<f16>(a, st);
        else rows_of<paged::bf16>(a, st);
        HIPCHK(hipGetLastError());
        hipLaunchKernelGGL(beam::k_beam_merge, dim3(n_batch), dim3(beam::MERGE_THREADS), 0, st, a);
        HIPCHK(hipGetLastError());
    });
}

}  // extern "C"
