"""A head blob in host memory is read at every call: what stood at its address before is not remembered."""
import ctypes as C

import numpy as np

from libr3d_b200 import abi
from libr3d_b200.plugin import ArgPack, tensor_desc
from test_plugin_host import _head, planes_blob


def test_another_blob_at_the_same_address_is_seen(plug):
    codes, scale = _head()
    N, K = codes.shape

    def blob(block):
        return np.frombuffer(planes_blob([("codes", abi.RAD_F8E4M3, (1, 1), codes), ("scale", abi.RAD_BF16, block, scale)]), np.uint8)

    good, other = blob((128, 128)), blob((128, 64))
    place, buf = np.zeros(max(good.size, other.size), np.uint8), np.zeros(1 << 16, np.uint8)
    M, R = 2, 4
    t = [None, tensor_desc(place.ctypes.data, abi.RAD_U8, [place.size])]
    t += [tensor_desc(buf.ctypes.data, d, [M, R]) for d in (abi.RAD_I32, abi.RAD_I32, abi.RAD_F32)]
    t[0] = tensor_desc(buf.ctypes.data, abi.RAD_BF16, [M, K], [2 * K, 2])      # refused behind the head's checks: nothing is launched
    f = plug.entry("r3d_rad_logit_rerank_e4m3")

    def call(b):
        place[:b.size] = b
        return f(C.byref(ArgPack(t, dict(M=M, R=R, n_vocab=N, n_embd=K, vocab_off=0, dtype="bf16")).args), None)

    assert [call(b) for b in (good, other, good, other)] == [abi.RAD_E_STRIDE, abi.RAD_E_DTYPE] * 2
