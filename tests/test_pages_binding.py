"""The request-batch calls of the Python binding without a GPU: shapes that are not taken, pointers of every kind that
the binding's other calls take, arguments that are none."""
import ctypes as C

import pytest

from shukuchi_b200 import cuda as sc


@pytest.mark.parametrize("heads,kv_heads", [(2048, 2048), (1025, 1025), (8192, 8), (4100, 1)])
def test_no_workspace_for_too_many_heads(heads, kv_heads):
    assert sc.pages_attend_ws(1, heads, kv_heads, 128) == 0
    assert sc.pages_attend_ws(1, 4096, 1024, 128) > 0


class NoContext(sc.Context):
    def __init__(self):
        self.h = None


@pytest.mark.parametrize("pointer", [64, None, C.c_void_p(64), C.c_void_p(None)])
@pytest.mark.parametrize("count", [1, -1])
def test_pointers_and_counts_of_every_kind(pointer, count):
    """Without a context every call is refused by the library, not by the binding."""
    ctx = NoContext()
    pages = sc.Pages(ctx, 64, 64, 64, 64, sc.PAGES_I8, 1, 1, 64, 16)
    calls = [lambda: ctx.pages_assign(count, 16, 4, 1, 1, *[pointer] * 11),
             lambda: ctx.pages_release(count, 16, 4, 1, *[pointer] * 7),
             lambda: ctx.pages_truncate(count, 16, 4, 1, *[pointer] * 7),
             lambda: pages.append(count, pointer, pointer, pointer), lambda: pages.read(count, pointer, pointer, pointer),
             lambda: pages.attend(count, pointer, pointer, 1, pointer, pointer, 1, 1, 1.0, pointer, 1, row_seq=pointer),
             lambda: ctx.sample(pointer, count, 8, pointer, pointer)]
    for call in calls:
        with pytest.raises(sc.ShkError) as e:
            call()
        assert e.value.code == -1
