"""What the kernels find wrong reaches users of the function, of the module and of captured steps."""
import ctypes

import pytest
import torch


@pytest.fixture
def watch(monkeypatch):
    from fly_b200 import ops
    fresh = ops._StatusWatch()
    monkeypatch.setattr(ops, 'status_watch', fresh)
    yield fresh


@pytest.mark.parametrize('words,match', [((284, 0, 0), 'wait site 284'), ((0, 1, 0), 'range'), ((0, 0, 1), '16 times')])
def test_the_function_reports(watch, words, match):
    from fly_b200 import SBLocalAttention, _cabi, ops
    x, W = torch.randn(1, 5, 2, 8), torch.randn(4, 8)
    layer = SBLocalAttention(2, 8, 8)
    for call in (lambda: ops.sblocal_attention(x, x, x, W, 2), lambda: layer(x, x, x), lambda: watch.poll(),
                 lambda: watch.poll(wait=True)):
        watch._words = (ctypes.c_int32 * 3)(*words)
        with pytest.raises(_cabi.SblError, match=match):
            call()
        watch.poll(wait=True)                                    # reported once
    watch._words = (ctypes.c_int32 * 3)(*words)
    with pytest.raises(ValueError, match='CUDA'):
        ops.sblocal_attention(x, x, x, W, 2, watch=False)


def inputs(d, scale):
    from tests.test_training_gpu import inputs as make
    q, k, v, dout, W = make(1, 512, 512, 2, d, d, 2 * d, torch.bfloat16, seed=17)
    return [(x.float() * s).bfloat16().requires_grad_() for x, s in ((q, scale), (k, scale), (v, 1.0))], W, dout


@pytest.mark.gpu
@pytest.mark.parametrize('d', [64, 128])
def test_out_of_range_logits_reach_the_functions_user(d, watch, sbl_lib):
    """Inputs 24 times the unit scale: exponentials leave the fp32 range."""
    from fly_b200 import _cabi, ops
    far, W, dout = inputs(d, 24.0)
    near = inputs(d, 1.0)[0]
    for grad in (True, False):
        with torch.set_grad_enabled(grad):
            ops.sblocal_attention(*far, W, 64)
            torch.cuda.synchronize()
            with pytest.raises(_cabi.SblError, match='range'):
                ops.sblocal_attention(*near, W, 64)
            ops.sblocal_attention(*far, W, 64)
            with pytest.raises(_cabi.SblError, match='range'):
                watch.poll(wait=True)
    out = ops.sblocal_attention(*near, W, 64)
    torch.autograd.grad(out, near, dout)
    watch.poll(wait=True)
    ops.sblocal_attention(*far, W, 64, watch=False)
    watch.poll(wait=True)


@pytest.mark.gpu
@pytest.mark.parametrize('module', [False, True])
@pytest.mark.parametrize('grad', [False, True])
def test_captured_steps_report(grad, module, watch, sbl_lib):
    from fly_b200 import SBLocalAttention, _cabi, ops
    xs, W, dout = inputs(64, 1.0)
    if module:
        layer = SBLocalAttention(64, 64, 256).cuda().eval()
        layer.feature_map.new_feature_map('cuda')
        layer.feature_map.projection_matrix.copy_(W)

    def step():
        with torch.set_grad_enabled(grad):
            out = layer(*xs)[0] if module else ops.sblocal_attention(*xs, W, 64)
            return (out.detach(), *torch.autograd.grad(out, xs, dout)) if grad else (out,)

    want = [x.clone() for x in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    watch.poll(wait=True)
    assert all(torch.equal(a, b) for a, b in zip(held, want))
    with torch.no_grad():
        good = [x.clone() for x in xs]
        for x in xs[:2]:
            x.mul_(24)
        graph.replay()
        for x, y in zip(xs, good):
            x.copy_(y)
    graph.replay()                       # a good replay behind the bad one does not hide it
    with pytest.raises(_cabi.SblError, match='range'):
        watch.poll(wait=True)
    graph.replay()
    watch.poll(wait=True)
    assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.gpu
def test_the_gradients_words_are_watched(watch, sbl_lib, monkeypatch):
    """No input makes a wait run out, so the word is planted on its way to the watch."""
    from fly_b200 import _cabi, ops
    xs, W, dout = inputs(64, 1.0)
    out = ops.sblocal_attention(*xs, W, 64)
    post = watch.post
    planted = torch.tensor([262, 0, 0], dtype=torch.int32, device='cuda')
    monkeypatch.setattr(watch, 'post', lambda words, device: post(planted.data_ptr(), device))
    torch.autograd.grad(out, xs, dout)
    with pytest.raises(_cabi.SblError, match='wait site 262'):
        watch.poll(wait=True)


def test_a_word_that_arrives_during_a_report_is_kept(watch):
    from fly_b200 import _cabi

    class Words(list):
        reads = 0

        def __iter__(self):
            seen = [self[i] for i in range(3)]
            self.reads += 1
            if self.reads == 2:            # a kernel of another stream, while the words are taken down
                self[2] = 1
            return iter(seen)

    watch._words = Words([0, 1, 0])
    with pytest.raises(_cabi.SblError, match='range'):
        watch.poll()
    with pytest.raises(_cabi.SblError, match='16 times'):
        watch.poll()


@pytest.mark.gpu
def test_zeros_leave_what_was_collected(sbl_lib):
    from fly_b200 import _cabi
    host = torch.zeros(5, dtype=torch.int32).pin_memory()
    stream = torch.cuda.current_stream().cuda_stream
    for words, want in (((0, 0, 0), (0, 0, 0)), ((0, 1, 0), (0, 1, 0)), ((0, 0, 0), (0, 1, 0)), ((284, 0, 1), (284, 1, 1)),
                        ((0, 0, 0), (284, 1, 1))):
        dev = torch.tensor((9, *words, 9), dtype=torch.int32, device='cuda')
        _cabi.check(sbl_lib.sbl_collect_status(dev.data_ptr() + 4, host.data_ptr() + 4, stream))
        torch.cuda.synchronize()
        assert host.tolist() == [0, *want, 0]


def test_collection_arguments(sbl_lib):
    for args in ((None, 4096), (4096, None), (4098, 4096), (4096, 4097)):
        assert sbl_lib.sbl_collect_status(*args, None) == -1
