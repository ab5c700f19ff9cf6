"""Tensors made of memory that a caller has on the device: shapes that are none, and views while other streams are at work."""
import numpy as np
import pytest

from gpu_util import cuda_backend
from onyxia_b200 import OnyxiaError, ir

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def session():
    b = ir.GraphBuilder()
    b.output("one", b.const_f32([1.0], [1]))
    return cuda_backend().prepare(b.finish())


@pytest.mark.parametrize("shape", [(2 ** 32, 2 ** 32), (2 ** 63,), (2 ** 31, 2 ** 31, 4), (2 ** 62,), (2 ** 62, 4), (2 ** 64 - 4,), (3, 2 ** 64 - 1), (2 ** 16,) * 4], ids=str)
def test_shapes_whose_elements_do_not_count_up_are_refused(session, shape):
    x = torch.ones(64, device="cuda")
    with pytest.raises(OnyxiaError, match="extent|more elements"):
        session.upload_device(ir.F32, shape, x.data_ptr())


def test_empty_shapes_are_taken(session):
    for shape in ((0,), (0, 2 ** 40), (2 ** 40, 0, 2 ** 40)):
        assert session.upload_device(ir.F32, shape, 0).shape == shape
    assert session.download(session.upload_device(ir.F32, (), torch.full((1,), 3.0, device="cuda").data_ptr())).numpy().item() == 3.0


def test_a_view_that_goes_while_its_stream_is_captured_keeps_its_memory(session):
    """The session cannot wait for a stream that is being captured: the memory that the graph reads stays where it is."""
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    x = torch.arange(1024, device="cuda", dtype=torch.float32)
    t = session.upload_device(ir.F32, (1024,), x.data_ptr(), torch.cuda.current_stream().cuda_stream)
    with torch.cuda.stream(side):
        seen = torch.as_tensor(session.view(t, side.cuda_stream), device="cuda")
    torch.cuda.synchronize()
    address = seen.data_ptr()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
        y = seen * 2
        del seen, t
    others = [session.upload_device(ir.F32, (1024,), x.data_ptr()) for _ in range(20)]
    assert address not in [torch.as_tensor(session.view(o), device="cuda").data_ptr() for o in others]
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(y.cpu().numpy(), 2 * np.arange(1024))
