"""qgemm._lib.addr: an address is taken as it is, without a look at anything else (it is on the
path of every call), and a tensor's own error comes through."""
import pytest

import qgemm._lib as L


def test_an_integer_is_its_own_address():
    class Ptr(int):
        @property
        def data_ptr(self):
            raise AssertionError("looked for")

    assert L.addr(Ptr(1 << 40)) == 1 << 40
    assert L.addr(None) == 0


def test_a_tensor_and_an_address():
    torch = pytest.importorskip("torch")
    t = torch.empty(4)
    assert L.addr(t) == t.data_ptr()

    class Buffer:
        address = 4096

    assert L.addr(Buffer()) == 4096
    with pytest.raises(TypeError):
        L.addr("text")


def test_an_error_of_data_ptr_is_not_hidden():
    class Tensor:
        address = 5

        def data_ptr(self):
            raise AttributeError("no storage")

    with pytest.raises(AttributeError, match="no storage"):
        L.addr(Tensor())


def test_a_proxy_of_a_tensor():
    class Proxy:
        def __init__(self, inner):
            self._inner = inner

        def __getattr__(self, name):
            return getattr(self._inner, name)

    torch = pytest.importorskip("torch")
    t = torch.empty(4)
    assert L.addr(Proxy(t)) == t.data_ptr()
