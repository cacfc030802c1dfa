"""The calls that the layer for a few tokens is tested with reach all of its gate_up kernels."""
import moe_few_cases as M


def test_cases_reach_every_gate_up_kernel():
    cases = list(M.cases())
    reached = {(kind, x, *M.kernel(kind, x, tokens, inter)) for kind, x, tokens, _, inter in cases}
    most = {(kind, x): M.loads(kind, x, M.most_entries(x)) for kind in M.KINDS for x in M.X_TYPES}
    shapes = [(share, 1) for share in (4, 2, 1)]
    want = {(kind, x, n, *shape) for (kind, x), m in most.items() for n in range(1, m + 1) for shape in shapes}
    assert len(want) == 66 and want <= reached
    assert {(kind, x, most[kind, x], 1, tiles) for kind, x in most for tiles in (2, 3, 4)} <= reached
