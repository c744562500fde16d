"""The order of a run: what needs the reference's kernels comes last, everything else as it was collected."""
from types import SimpleNamespace

import conftest


def test_what_needs_the_reference_comes_last():
    items = [SimpleNamespace(name=n, fixturenames=f) for n, f in
             [("a", ["cuda", "ref"]), ("b", ["cuda"]), ("c", []), ("d", ["ref"]), ("e", ["cuda", "reference"])]]
    items.append(SimpleNamespace(name="f"))
    conftest.pytest_collection_modifyitems(items)
    assert "".join(i.name for i in items) == "bcefad"
