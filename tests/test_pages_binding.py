"""The request-batch calls of the Python binding without a GPU: shapes that are not taken, pointers of every kind that
the binding's other calls take, arguments that are none."""
import ctypes as C

import pytest

from shukuchi_b200 import cuda as sc


@pytest.mark.parametrize("heads,kv_heads", [(2048, 2048), (1025, 1025), (8192, 8), (4100, 1)])
def test_no_workspace_for_too_many_heads(heads, kv_heads):
    assert sc.pages_attend_ws(1, heads, kv_heads, 128) == 0
    assert sc.pages_attend_ws(1, 4096, 1024, 128) > 0
