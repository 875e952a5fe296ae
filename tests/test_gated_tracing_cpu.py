"""The gated block's registered operators under tracing with symbolic sizes (shape functions only: no kernel runs)."""
import pytest
import torch

import csn_b200.ops  # noqa: F401

csn = torch.ops.csn


class Scan(torch.nn.Module):
    def forward(self, f, x, cu=None):
        y, h, marks = csn.gated_scan_fwd(f, x, None, None, cu)
        return y, h, marks


@pytest.mark.parametrize("packed", [False, True])
def test_scan_exports_with_any_length(packed):
    """The number of marks is an expression in the sizes, so that a traced length stays one."""
    from torch.export import Dim, export
    d = Dim("length", min=2, max=1 << 20)
    b = Dim("batch", min=3, max=4096)  # torch traces a size of 1 apart, and one sequence has two borders
    if packed:
        args = (torch.zeros(300, 8), torch.zeros(300, 8), torch.zeros(6, dtype=torch.int32))
        shapes = ({0: d}, {0: d}, {0: b})
    else:
        args, shapes = (torch.zeros(3, 70, 8), torch.zeros(3, 70, 8)), ({0: b, 1: d}, {0: b, 1: d})
    program = export(Scan(), args, dynamic_shapes=shapes)
    node = next(n for n in program.graph.nodes if "gated_scan_fwd" in str(n.target))
    y, h, marks = node.meta["val"]
    assert not isinstance(y.shape[0 if packed else 1], int) and not isinstance(marks.shape[0], int) and not isinstance(h.shape[0], int)


def test_scan_compiles_once_for_every_length():
    seen = []

    def backend(graph, inputs):
        seen.append(graph)
        return graph.forward

    step = torch.compile(lambda f, x: csn.gated_scan_fwd(f, x, None, None, None)[0], backend=backend)
    for n in (40, 70, 129, 200, 333, 1000):
        f = torch.empty(2, n, 8, device="meta")
        assert step(f, f).shape == (2, n, 8)
    assert len(seen) <= 2  # the first length, then any


@pytest.mark.parametrize("S,T,C,packed", [(1, 1, 1, 0), (3, 64, 8, 0), (5, 129, 24, 0), (4, 0, 8, 0), (0, 5, 8, 0), (5, 5, 0, 0), (4, 1000, 8, 1),
                                          (100, 7, 3, 1), (3, 0, 8, 1)])
def test_number_of_marks_is_the_librarys(S, T, C, packed):
    from csn_b200 import _build, _lib
    _build.build()
    m = lambda *s, d=torch.bfloat16: torch.empty(*s, device="meta", dtype=d)  # noqa: E731
    f, cu = (m(T, C), m(S + 1, d=torch.int32)) if packed else (m(S, T, C), None)
    assert csn.gated_scan_fwd(f, f, None, None, cu)[2].numel() == _lib.load().csn_gated_scan_marks(S, T, C, packed)
