"""What the entry points for code scores and the AdamW step refuse on the host, before any launch (no GPU needed)."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as g
    g.build()
    from mqgan_amd import _lib
    return _lib.load()


A = C.c_void_p(4096)


def refused(lib, rc, words):
    assert rc != 0 and words in lib.mq_last_error(), lib.mq_last_error()


def test_sample_codes_refuses_on_the_host(lib):
    from mqgan_amd._lib import SampleDesc

    def call(z=A, u=A, idx=A, T=None, k=None, p=None, m=None, **kw):
        d = SampleDesc(rows=4, row_stride=10, codes=10, dtype=0, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0)
        for a, v in kw.items():
            setattr(d, a, v)
        return lib.mq_sample_codes(C.byref(d), z, u, T, k, p, m, None, idx, None, None)
    refused(lib, call(z=None), b"NULL")
    refused(lib, call(u=None), b"NULL")
    refused(lib, call(idx=None), b"NULL")
    refused(lib, lib.mq_sample_codes(None, A, A, None, None, None, None, None, A, None, None), b"NULL")
    for kw in ({"rows": 0}, {"rows": -1}, {"rows": 2 ** 31}, {"codes": 0}, {"codes": (1 << 20) + 1, "row_stride": 1 << 21}, {"row_stride": 9}):
        refused(lib, call(**kw), b"bad sizes")
    refused(lib, call(dtype=3), b"dtype")
    refused(lib, call(dtype=-1), b"dtype")
    for v in (-1.0, float("nan")):
        refused(lib, call(temperature=v), b"temperature")
    refused(lib, call(top_k=-1), b"top_k")
    for v in (-0.1, 1.1, float("nan")):
        refused(lib, call(top_p=v), b"top_p")
        refused(lib, call(min_p=v), b"min_p")


def test_code_balance_refuses_on_the_host(lib):
    def sums(z=A, dtype=0, ld=10, idx=A, K=1, rows=4, codes=10, stats=A, counts=A, out=A, loss=A, f=A, ws=A, n=1 << 20):
        return lib.mq_code_balance_fwd(z, dtype, ld, idx, 0, K, None, rows, codes, stats, counts, out, loss, f, ws, n, None)
    for a in ("z", "idx", "stats", "counts", "out", "ws", "loss", "f"):
        refused(lib, sums(**{a: None}), b"NULL")
    refused(lib, sums(dtype=3), b"dtype")
    for kw in ({"rows": 0}, {"rows": 2 ** 31}, {"codes": 0}, {"codes": (1 << 24) + 1, "ld": 1 << 25}, {"K": 0}, {"ld": 9}):
        refused(lib, sums(**kw), b"bad sizes")
    refused(lib, sums(rows=2 ** 30, K=4), b"32 bits")
    need = lib.mq_code_balance_workspace(4, 10, 0)
    assert need > 0 and lib.mq_code_balance_workspace(0, 10, 0) == 0 and lib.mq_code_balance_workspace(4, 0, 0) == 0 and lib.mq_code_balance_workspace(4, 10, 3) == 0
    refused(lib, sums(n=need - 1), b"workspace")
    refused(lib, lib.mq_code_balance_final(A, 0, 1, A, A, None), b"bad arguments")
    refused(lib, lib.mq_code_balance_final(None, 4, 1, A, A, None), b"bad arguments")

    def bwd(z=A, dtype=0, ld=10, rows=4, codes=10, stats=A, s=A, f=A, g=A, dz=A):
        return lib.mq_code_balance_bwd(z, dtype, ld, None, rows, codes, stats, s, f, g, dz, None)
    for a in ("z", "stats", "s", "f", "g", "dz"):
        refused(lib, bwd(**{a: None}), b"NULL")
    refused(lib, bwd(dtype=9), b"dtype")
    for kw in ({"rows": 0}, {"codes": 0}, {"ld": 9}):
        refused(lib, bwd(**kw), b"bad sizes")


def test_adamw_refuses_on_the_host(lib):
    from mqgan_amd._lib import AdamwDesc, AdamwTensor
    sizes = (C.c_int64 * 2)(300, 5000)
    nbytes = lib.mq_adamw_table_bytes(sizes, 2)
    assert nbytes == 192 + 3 * 4 and lib.mq_adamw_control_bytes(2) == 96 and lib.mq_adamw_workspace(sizes, 2) >= 3 * 8
    assert lib.mq_adamw_table_bytes((C.c_int64 * 1)(-1), 1) == 0 and lib.mq_adamw_table_bytes(sizes, 0) == 0
    assert lib.mq_adamw_table_bytes((C.c_int64 * 1)(2 ** 63 - 1), 1) == 0
    assert lib.mq_adamw_table_bytes((C.c_int64 * 1)(2 ** 36 - 4096), 1) > 0 and lib.mq_adamw_table_bytes((C.c_int64 * 1)(2 ** 36 - 4095), 1) == 0      # 2^32 threads

    def fill(bits=32, count=2, size=nbytes, host=True, **kw):
        rows = (AdamwTensor * 2)(AdamwTensor(4096, 8192, 16384, 100, 200, 300, 0, 0.0, 1.0), AdamwTensor(4096, 8192, 16384, 100, 200, 5000, 512, 0.1, 1.0))
        for a, v in kw.items():
            setattr(rows[1], a, v)
        buf = C.create_string_buffer(max(size, nbytes))
        return lib.mq_adamw_table_fill(rows, count, bits, buf if host else None, size)
    assert fill() == 0 and fill(bits=8) == 0
    refused(lib, fill(bits=16), b"32 or 8 bits")
    refused(lib, fill(count=0), b"bad arguments")
    refused(lib, fill(host=False), b"bad arguments")
    refused(lib, fill(size=nbytes - 4), b"bytes")
    for kw in ({"n": -1}, {"position": 100}, {"position": -256}):
        refused(lib, fill(**kw), b"position")
    for kw in ({"param": None}, {"exp_avg": None}, {"exp_avg_sq": None}):
        refused(lib, fill(**kw), b"NULL")
    for kw in ({"param": 4097}, {"exp_avg": 8200}, {"exp_avg_sq": 8196}):
        refused(lib, fill(**kw), b"multiple")
    refused(lib, fill(bits=8, base_avg=None), b"bases")

    def step(grads=(4096, 8192), types=None, numel=sizes, table=A, control=A, ws=A, n=24, **kw):
        d = AdamwDesc(n_tensors=2, state_bits=32, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, max_norm=1.0, grad_scale=1.0, seed=0)
        for a, v in kw.items():
            setattr(d, a, v)
        return lib.mq_adamw_step(C.byref(d), numel, table, (C.c_void_p * 2)(*grads), types, control, ws, n, None)
    refused(lib, step(n=23), b"workspace")
    refused(lib, step(ws=None), b"workspace")
    refused(lib, step(table=None), b"bad arguments")
    refused(lib, step(control=None), b"bad arguments")
    refused(lib, step(numel=None), b"bad arguments")
    refused(lib, step(n_tensors=0), b"no tensors")
    refused(lib, step(state_bits=4), b"32 or 8")
    for kw in ({"lr": -1.0}, {"lr": float("nan")}, {"beta1": 1.0}, {"beta2": -0.1}, {"eps": -1e-8}, {"max_norm": -1.0}, {"max_norm": float("nan")}):
        refused(lib, step(**kw), b"are needed")
    refused(lib, step(grads=(4096, 8194)), b"aligned")
    refused(lib, step(grads=(4096, 8193), types=(C.c_uint8 * 2)(0, 1)), b"aligned")
    refused(lib, step(types=(C.c_uint8 * 2)(0, 3)), b"element type")
    refused(lib, lib.mq_moments8_encode(A, A, 255, A, A, A, A, None), b"256")
    refused(lib, lib.mq_moments8_encode(A, None, 256, A, A, A, A, None), b"bad arguments")
    refused(lib, lib.mq_moments8_encode(C.c_void_p(4100), A, 256, A, A, A, A, None), b"multiples")
    refused(lib, lib.mq_moments8_decode(A, A, A, A, 100, 0, A, A, None), b"256")
    refused(lib, lib.mq_moments8_encode(A, A, 2 ** 34, A, A, A, A, None), b"too many")
    refused(lib, lib.mq_moments8_decode(A, A, A, A, 2 ** 35, 0, A, A, None), b"too many")
    refused(lib, lib.mq_moments8_decode(A, A, A, A, 256, 0, A, C.c_void_p(4104), None), b"multiples")


def test_cpu_tensors_are_refused(lib):
    from mqgan_amd import ops
    from mqgan_amd._lib import MqganHipError
    from mqgan_amd.losses import code_balance_loss
    from mqgan_amd.optim import AdamW
    with pytest.raises(MqganHipError):
        ops.sample_codes(torch.zeros(2, 4), torch.zeros(2))
    with pytest.raises(MqganHipError):
        code_balance_loss(torch.zeros(2, 4), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(MqganHipError):
        AdamW([torch.zeros(4)])


def test_scores_are_read_in_place_where_one_stride_joins_the_rows():
    from mqgan_amd.ops import _score_rows
    z = torch.zeros(3, 5, 20)
    for t, stride, same in ((z, 20, True), (z[..., 2:18], 20, True), (z[:, ::2], 20, False), (z[:, :3], 20, False), (z[::2], 20, False), (z[0, ::2], 40, True),
                            (z.transpose(0, 1), 20, False), (z[..., ::2], 10, False), (z[0, 0], 20, True), (z[:, 0], 100, True),
                            (z[0, 0].expand(6, 20), 20, False), (z[:0], 20, True)):
        got, kind, rows, V, ld = _score_rows(t, "test")
        assert kind == 0 and rows == t.numel() // t.shape[-1] and V == t.shape[-1]
        assert (got.data_ptr() == t.data_ptr()) == same or t.numel() == 0, (t.shape, t.stride())
        if same and rows > 1:
            assert ld == stride
            flat = torch.as_strided(got, (rows, V), (ld, 1), got.storage_offset())
            assert flat.data_ptr() == t.data_ptr() and torch.equal(flat.reshape(t.shape), t)
