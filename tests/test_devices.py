"""Tensors of another device, or of another size than the kernels go by, are refused before a launch: the kernels would
read or write through their addresses.  Run without a GPU, on host tensors that say they are elsewhere."""
import pytest
import torch


def on(index):
    class Elsewhere(torch.Tensor):
        is_cuda = property(lambda self: True)
        device = property(lambda self: torch.device('cuda', index))

    return lambda *shape: torch.zeros(*shape).as_subclass(Elsewhere)


HERE, THERE = on(0), on(1)


def problem(**over):
    from fly_b200 import ops
    args = dict(query=HERE(1, 5, 2, 8), key=HERE(1, 6, 2, 8), value=HERE(1, 6, 2, 4), W=HERE(3, 8), local_context=2,
                out=HERE(1, 5, 2, 4))
    args.update(over)
    return ops.Problem(**args)


def test_inputs_and_output_on_one_device(sbl_lib):
    assert problem().shape == (1, 2, 5, 6, 8, 4)
    for name, shape in (('query', (1, 5, 2, 8)), ('key', (1, 6, 2, 8)), ('value', (1, 6, 2, 4)), ('out', (1, 5, 2, 4))):
        with pytest.raises(ValueError, match='device'):
            problem(**{name: THERE(*shape)})
    with pytest.raises(ValueError, match='device'):
        problem(out=torch.zeros(1, 5, 2, 4))


def test_row_stats_of_the_problem(sbl_lib):
    n = 2 * 2 * 5 + 2
    for bad in (HERE(n - 1), HERE(n + 1), HERE(n, 1), HERE(n).double(), THERE(n), torch.zeros(n), HERE(2 * n)[::2],
                HERE(1).expand(n)):
        with pytest.raises(ValueError, match='row_stats'):
            problem().backward(HERE(1, 5, 2, 4), bad)


def test_workspace_on_the_device(sbl_lib):
    p = problem()
    n = p.workspace_bytes
    for bad in (torch.zeros(n, dtype=torch.uint8), THERE(n).byte(), HERE(1).byte().expand(n), HERE(2 * n).byte()[::2]):
        with pytest.raises(ValueError, match='workspace'):
            p.forward(workspace=bad)
        with pytest.raises(ValueError, match='workspace'):
            p.check_status(workspace=bad)
