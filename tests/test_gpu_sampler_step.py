"""run_generation_step with a sampler when the step's decode merge gave up."""

from __future__ import annotations

import pytest
import torch

from mini_llm_runtime_amd.kernels import paged_attention as kpa
from mini_llm_runtime_amd.runtime.model_runner import RandomSampler, run_generation_step
from test_gpu_operator_step import serving

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sampler", [None, RandomSampler(3, temperature=1.1, top_k=20)],
                         ids=["greedy", "random"])
def test_a_merge_that_gave_up_is_reported(device, dtype, sampler):
    """What the runner raises is DecodeMergeError, not what the sampler makes of
    logits that are NaN; the workspace is clear afterwards and the next step runs.
    The flag is set from the host, and the logits of that step are NaN as such a
    merge leaves them; every kernel exits normally."""
    model, scheduler = serving(device, dtype)
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream), torch.no_grad():
        run_generation_step(model, scheduler, sampler=sampler)
        # This stream's cached workspace, larger than these steps would make it.
        ws = kpa.decode_workspace(device, 1 << 24)
        ws[:4].view(torch.int32).fill_(1)

        def failed(logits, batch):
            return sampler(torch.full_like(logits, torch.nan), batch)

        with pytest.raises(kpa.DecodeMergeError, match="gave up waiting"):
            run_generation_step(model, scheduler, sampler=sampler and failed)
        assert int(torch.count_nonzero(ws)) == 0
        model, scheduler = serving(device, dtype)
        step = run_generation_step(model, scheduler, sampler=sampler)
        assert len(step.sampled_token_ids) == 3
    torch.cuda.synchronize()


def test_an_error_of_the_sampler_passes_where_the_merge_was_sound(device):
    model, scheduler = serving(device, torch.bfloat16)

    def broken(logits, batch):
        raise KeyError("no such request")

    with torch.no_grad(), pytest.raises(KeyError, match="no such request"):
        run_generation_step(model, scheduler, sampler=broken)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_random_sampler_under_other_defaults(device, dtype):
    """The same tokens whatever the default device and dtype are."""
    outs = []
    for default in ("cpu", "cuda"):
        model, scheduler = serving(device, torch.bfloat16)
        before = torch.get_default_dtype()
        with torch.device(default), torch.no_grad():
            try:
                torch.set_default_dtype(before if default == "cpu" else dtype)
                sampler = RandomSampler(11, temperature=1.3)
                outs.append([run_generation_step(model, scheduler, sampler=sampler)
                             .sampled_token_ids for _ in range(4)])
            finally:
                torch.set_default_dtype(before)
    assert outs[0] == outs[1]
