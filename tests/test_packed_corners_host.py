"""What keys and values in 4 bits refuse beside what test_packed_host.py has, asked of the backend's registry without a device."""
import pytest

import packed_util as util
from packed_util import Form
from onyxia_b200 import ir
from test_packed_host import lib  # noqa: F401  (a fixture)


@pytest.fixture
def with_attrs(monkeypatch):
    """Modules whose composites have more attributes."""
    def build(f, dtype, kind, **more):
        class Builder(ir.GraphBuilder):
            def composite(self, name, attrs, *rest):
                return super().composite(name, {**attrs, **(more if name != "onyxia.CacheRead" else {})}, *rest)

        with monkeypatch.context() as m:
            m.setattr(ir, "GraphBuilder", Builder)
            return util.module(f, dtype, kind)

    return build


@pytest.mark.parametrize("dtype", [ir.F32, ir.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["attend", "shared", "write"])
@pytest.mark.parametrize("name", ["interleaved", "gate", "sinks", "temps", "talk"])
def test_attributes_that_only_the_whole_cache_has(lib, with_attrs, name, kind, dtype):  # noqa: F811
    """Pairs side by side, gates, learned sinks, temperatures and mixed heads are not left out without a word."""
    f = Form(4, 2, 64, 128, 64)
    for value, nodes in ((0, 1), (1, 0), (2, 0)):
        m = with_attrs(f, dtype, kind, **{name: value, "gate_offset": 3})
        assert lib.taken(m.handle) == nodes
