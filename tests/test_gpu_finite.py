"""Products, rotary positions and appends once more, where a value that is not finite never counts as near a reference that is."""

import pytest
import torch

import test_gpu_linear
import test_gpu_linear_int4
import test_gpu_rope
import test_gpu_rotary
from test_gpu_linear import test_linear_and_partials  # noqa: F401
from test_gpu_linear_int4 import (test_every_kernel_that_the_rule_picks, test_fewer_blocks_than_splits,  # noqa: F401
                                  test_more_rows_than_the_stream_kernel_takes, test_products, test_scales_of_the_other_type, test_swiglu)
from test_gpu_rope import (test_fused_edges_match_oracle, test_fused_norm_rope_append_config1_shape,  # noqa: F401
                           test_rope_matches_oracle_up_to_long_positions)
from test_gpu_rotary import (test_append, test_append_at_given_positions, test_append_past_32_bit_offsets,  # noqa: F401
                             test_append_skips_what_lies_outside, test_apply, test_forward_mode, test_gradients, test_pair_factors_and_amplitude)

pytestmark = pytest.mark.gpu


def compared(loose, at):
    """The comparison ``loose(got, ...)``, whose argument ``at`` is the reference."""
    def compare(got, *rest, **kw):
        assert not (torch.isfinite(rest[at - 1].cpu()) & ~torch.isfinite(got.detach().cpu())).any()
        loose(got, *rest, **kw)

    return compare


@pytest.fixture(autouse=True)
def finite(monkeypatch):
    for module, name, at in ((test_gpu_rotary, "close", 1), (test_gpu_rope, "bf16_close", 1), (test_gpu_rope, "pairs_close", 1),
                             (test_gpu_linear_int4, "close", 1), (test_gpu_linear, "close_sum", 3)):
        monkeypatch.setattr(module, name, compared(getattr(module, name), at))
