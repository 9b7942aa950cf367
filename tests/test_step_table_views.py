"""CPU tests of step tables whose lengths and free pages are named by several views of one
memory."""

import pytest
import torch

from flashprefill_amd.step_tables import build_step_tables


def _step(views):
    """A traced step over fake tensors, with seq_lens_out and num_free_out views of the
    inputs or not given."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.symbolic_shapes import ShapeEnv
    with FakeTensorMode(shape_env=ShapeEnv(allow_scalar_outputs=True,
                                           allow_dynamic_output_shape_ops=True)):
        def ints(*shape, dtype=torch.int32):
            return torch.zeros(*shape, dtype=dtype, device="cuda")
        lens, free = ints(4), ints(1)
        out = dict(seq_lens_out=lens.view(-1), num_free_out=free[:1]) if views else {}
        build_step_tables(lens, ints(4), ints(4, 8), ints(20), free, 16, ints(5),
                          ints(9, dtype=torch.int64), ints(9, dtype=torch.int64), ints(4), **out)
        with pytest.raises(ValueError, match="memory"):
            build_step_tables(lens, lens.view(-1), ints(4, 8), ints(20), free, 16, ints(5),
                              ints(9, dtype=torch.int64), ints(9, dtype=torch.int64), ints(4),
                              **out)


def test_lengths_and_free_pages_by_other_views():
    _step(False)
    _step(True)
