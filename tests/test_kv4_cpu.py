"""The 4-bit cache's format on known blocks, and its calls' refusals without a device."""
import ctypes as C

import numpy as np

import kv4_ref
import qimm


def test_known_blocks():
    x = np.zeros((4, 32))
    x[0, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0]   # midpoints go to the even code, 7 to 6
    x[1, :3] = [7.5, -1.0, 0.6]                               # above 7: the next power of two
    x[2, :3] = [-28.0, 4.0, 1.0]                              # 7 * 4
    x[3, :2] = [3.38e38, 1.0e-40]
    got = kv4_ref.near(x)
    assert got[0, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]
    assert got[1, :3].tolist() == [8.0, -1.0, 1.0]
    assert got[2, :3].tolist() == [-24.0, 4.0, 0.0]
    assert got[3, 0] == 6 * 2.0 ** 125 and got[3, 1] == 0
    assert not kv4_ref.near(np.zeros((2, 64))).any()


def test_values_are_exact_in_bf16_and_off_by_half_a_step():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((64, 128)) * 2.0 ** rng.integers(-20, 20, (64, 1))
    y = kv4_ref.near(x)
    assert np.array_equal(y.astype(np.float32).view(np.uint32) & 0xffff, np.zeros(y.shape, np.uint32))
    b, top = (x - y).reshape(64, 4, 32), np.abs(x).reshape(64, 4, 32).max(-1, keepdims=True)
    # half the spacing at the top of the range is 2^s <= 2 top / 7
    assert (np.abs(b) <= top / 3.5 * 1.0000001).all()


def test_null_arguments():
    lib = qimm.load()
    h = C.c_void_p()
    assert lib.qimm_kv_create_q4(None, 1, 1, 1, 8, 128, C.byref(h)) == 1
    assert lib.qimm_kv_bits(None) == -1
    assert lib.qimm_kv_device_bytes(None) == -1


def test_null_arguments_of_the_adapters():
    lib = qimm.load()
    h = C.c_void_p()
    assert lib.qimm_adapters_create(None, 128, 64, None, 0, C.byref(h)) == 1
    assert lib.qimm_adapters_destroy(None) == 1
    assert lib.qimm_adapters_device_bytes(None) == -1
    assert lib.qimm_qmatmul_adapters(None, None, None, None, None, 1, 64, None, 0, None) == 1
    assert lib.qimm_qmatmul_adapters_reserve(None, None, None, 1, 0) == 1
    assert lib.qimm_block_set_adapters(None, None, 0) == 1
    assert lib.qimm_block_set_adapter_ids(None, None) == 1
