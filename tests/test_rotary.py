"""Refusals of the rotation and the cache appends, without a GPU: the entry points raise ValueError
before any device work, the C ABI returns a status and a message before it touches the device."""
import ctypes

import pytest
import torch

import dsa_triton_ascend_amd as dsa
from dsa_triton_ascend_amd import _lib

F = torch.ones(32)
X = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
POS = torch.zeros(2, 3, dtype=torch.int64)


@pytest.mark.parametrize("change,message", [
    (dict(positions=POS.float()), "int32 or int64"), (dict(positions=POS[:1]), "positions must have shape"),
    (dict(inv_freq=F.double()), "float32"), (dict(inv_freq=torch.ones(0)), "pairs"), (dict(inv_freq=torch.ones(33)), "rotary"),
    (dict(rotary_start=2), "rotary dimensions"), (dict(rotary_start=-64), "rotary dimensions"),
    (dict(sections=(16, 15)), "add up"), (dict(sections=(40, -8)), "add up"), (dict(sections=(1, 1, 1, 1, 28)), "1 to 4"),
    (dict(sections=(16, 16)), "shape"), (dict(layout="TND"), r"\[T, N, D\]"), (dict(layout="PA_BSND"), "layout"),
    (dict(x=X.double()), "dtype"), (dict(), "GPU")])
@pytest.mark.parametrize("grad", [False, True])
def test_rotary_refuses(change, message, grad):
    a = dict(x=X, positions=POS, inv_freq=F)
    a.update(change)
    x = a.pop("x")
    with pytest.raises(ValueError, match=message):
        (dsa.rotary_embedding_grad if grad else dsa.rotary_embedding)(x, **a)


def latent_args(**change):
    bf = dict(dtype=torch.bfloat16)
    a = dict(latent=torch.zeros(2, 3, 1, 512, **bf), key_rope=torch.zeros(2, 3, 1, 64, **bf),
             key_cache=torch.zeros(8, 16, 1, 512, **bf), key_rope_cache=torch.zeros(8, 16, 1, 64, **bf),
             block_table=torch.zeros(2, 4, dtype=torch.int32), inv_freq=F, actual_seq_lengths_kv=[3, 64])
    a.update(change)
    return a


BF = torch.bfloat16


@pytest.mark.parametrize("change,message", [
    (dict(latent=torch.zeros(2, 3, 1, 320, dtype=BF)), "D must be"), (dict(latent=torch.zeros(2, 3, 512, dtype=BF)), r"\[B, S"),
    (dict(latent=torch.zeros(2, 3, 1, 512)), "dtype"), (dict(latent=torch.zeros(2, 3, 2, 512, dtype=BF)), "N2=1"),
    (dict(key_rope=torch.zeros(2, 3, 1, 32, dtype=BF)), "rope dim"), (dict(key_rope=torch.zeros(2, 4, 1, 64, dtype=BF)), "N2=1"),
    (dict(key_cache=torch.zeros(8, 16, 512, 1, dtype=BF)), "caches must be"),
    (dict(key_cache=torch.zeros(16, 8, 1, 512, dtype=BF).transpose(0, 1)), "contiguous"),
    (dict(key_cache=torch.zeros(8, 8, 1, 512, dtype=BF)), "same blocks"),
    (dict(key_rope_cache=torch.zeros(8, 16, 1, 64)), "dtype"), (dict(inv_freq=torch.ones(16)), "32 wanted"),
    (dict(actual_seq_lengths_kv=[3]), "batch mismatch"), (dict(actual_seq_lengths_kv=[3, 65]), "outside"),
    (dict(actual_seq_lengths_kv=[-1, 5]), "outside"), (dict(actual_seq_lengths_query=[4, 1]), "between 0 and"),
    (dict(actual_seq_lengths_query=[1, 1, 1]), "per-batch"), (dict(block_table=torch.zeros(3, 4)), "block_table"),
    (dict(norm_weight=torch.ones(64)), "norm weights"), (dict(norm_weight=torch.ones(512).double()), "norm weights"),
    (dict(sections=(16, 16)), "need positions"), (dict(positions=torch.zeros(2, 2, dtype=torch.long)), "shape"),
    (dict(layout="TND"), r"\[T, N, D\]"), (dict(), "GPU")])
def test_latent_append_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        dsa.latent_cache_append(**latent_args(**change))


@pytest.mark.parametrize("change,message", [
    (dict(index_key=torch.zeros(2, 3, 1, 72, dtype=BF)), "D must be"), (dict(index_cache=torch.zeros(8, 16, 2, 128, dtype=BF)), "index_cache"),
    (dict(norm_bias=torch.ones(128)), "needs norm_weight"),
    (dict(norm_weight=torch.ones(128), norm_bias=torch.ones(128).half()), "share a dtype"),
    (dict(rotary_start=4), "multiple of 8"), (dict(rotary_start=72), "rotary dimensions"), (dict(inv_freq=torch.ones(12)), "of 16"),
    (dict(), "GPU")])
def test_index_append_refuses(change, message):
    a = dict(index_key=torch.zeros(2, 3, 1, 128, dtype=BF), index_cache=torch.zeros(8, 16, 1, 128, dtype=BF),
             block_table=torch.zeros(2, 4, dtype=torch.int32), inv_freq=F, actual_seq_lengths_key=[3, 64])
    a.update(change)
    with pytest.raises(ValueError, match=message):
        dsa.index_cache_append(**a)


def test_c_entries_refuse():
    lib = _lib.load()
    p = ctypes.c_void_p(16)   # never dereferenced: validation fails first
    sec = (ctypes.c_int32 * 2)(16, 15)
    neg = (ctypes.c_int32 * 2)(40, -8)

    def refused(fn, base, at, value, what, status=_lib.DSA_ERR_INVALID):
        args = list(base)
        args[at] = value
        assert fn(*args) == status
        assert what in lib.dsa_last_error().decode(), lib.dsa_last_error()

    base = [p, 0, 64, 64, 1, p, 0, 1, None, p, 4, 4, 2, 64, 0, 64, 1, 0, p, None]
    for at, v, what in ((0, None, "null"), (5, None, "null"), (9, None, "null"), (18, None, "null"), (4, 5, "dtype"),
                        (7, 0, "axes"), (7, 5, "axes"), (7, 2, "sections"), (10, -1, "shape"), (11, 0, "shape"),
                        (12, 0, "shape"), (14, 2, "rotary"), (15, 63, "rotary"), (15, 0, "rotary")):
        refused(lib.dsa_rotary, base, at, v, what)
    two = list(base)
    two[7], two[8] = 2, sec
    assert lib.dsa_rotary(*two) == _lib.DSA_ERR_INVALID and b"add up" in lib.dsa_last_error()
    two[8] = neg
    assert lib.dsa_rotary(*two) == _lib.DSA_ERR_INVALID and b"negative" in lib.dsa_last_error()
    refused(lib.dsa_rotary, base, 13, 5000, "width", _lib.DSA_ERR_UNSUPPORTED)
    refused(lib.dsa_rotary, base, 12, 20000, "2^20", _lib.DSA_ERR_UNSUPPORTED)

    lat = [p, 0, 512, p, 0, 64, 1, 512, None, 1, 1e-6, None, 0, 1, None, p, 1, p, p, p, 0, p, 2, 4, 4, 3, 16, 8, p, p, None]
    for at, v, what in ((0, None, "null"), (3, None, "null"), (15, None, "null"), (17, None, "null"), (21, None, "null"),
                        (28, None, "null"), (29, None, "null"), (6, 2, "io_dtype"), (7, 320, "D must"), (13, 2, "sections"),
                        (22, 0, "shape"), (24, 0, "shape"), (25, 0, "shape"), (26, 0, "shape"), (27, 0, "shape"),
                        (28, ctypes.c_void_p(24), "aligned"), (29, ctypes.c_void_p(24), "aligned")):
        refused(lib.dsa_latent_append, lat, at, v, what)
    bad = list(lat)
    bad[20], bad[22] = 1, 19
    assert lib.dsa_latent_append(*bad) == _lib.DSA_ERR_UNSUPPORTED and b"18 sequences" in lib.dsa_last_error()
    bad = list(lat)
    bad[8], bad[9] = p, 7
    assert lib.dsa_latent_append(*bad) == _lib.DSA_ERR_INVALID and b"norm weights" in lib.dsa_last_error()

    idx = [p, 0, 128, 128, 1, 1, 128, p, p, 2, 1e-6, None, 0, 1, None, p, 0, 64, 0, p, p, p, 0, p, 2, 4, 4, 3, 16, 8, p, None]
    for at, v, what in ((0, None, "null"), (15, None, "null"), (30, None, "null"), (4, 2, "io_dtype"), (5, 0, "heads"),
                        (7, None, "norm_bias"), (9, 9, "norm weights"), (17, 256, "rotary")):
        refused(lib.dsa_index_append, idx, at, v, what)
    refused(lib.dsa_index_append, idx, 6, 72, "D=72", _lib.DSA_ERR_UNSUPPORTED)
    refused(lib.dsa_index_append, idx, 16, 4, "multiple of 8", _lib.DSA_ERR_UNSUPPORTED)
    refused(lib.dsa_index_append, idx, 17, 24, "of 16", _lib.DSA_ERR_UNSUPPORTED)
    # nothing to do: no launch
    none = list(idx)
    none[25] = 0
    assert lib.dsa_index_append(*none) == 0


def test_prefill_refuses_positions_without_frequencies():
    z = torch.zeros(4, 1, 64, dtype=BF)
    for kw, message in ((dict(positions=torch.zeros(4, dtype=torch.long)), "need inv_freq"), (dict(sections=(16, 16)), "need inv_freq"),
                        (dict(inv_freq=F, sections=(16, 16)), "need positions"), (dict(inv_freq=torch.ones(16)), "32 wanted")):
        with pytest.raises(ValueError, match=message):
            dsa.dsa_prefill(z, z, z, z, z, z, z, [4], **kw)


@pytest.mark.parametrize("cast", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(), lambda m: m.bfloat16().float(),
                                  lambda m: m.to(torch.float16).to("cpu", torch.float32), lambda m: m.type(torch.bfloat16)])
def test_module_keeps_its_frequencies_through_casts(cast):
    """A model's cast to its type must not round the frequencies: 8 bits of them would turn far positions by
    whole turns, and any other type than float32 is refused."""
    f = 1.0 / 10000 ** (torch.arange(32) / 32)
    model = torch.nn.Sequential(torch.nn.Linear(4, 4), dsa.RotaryEmbedding(f))
    cast(model)
    assert model[1].inv_freq.dtype == torch.float32 and torch.equal(model[1].inv_freq, f)
    assert [n for n, _ in model.named_buffers()] == ["1.inv_freq"] and not any("inv_freq" in k for k in model.state_dict())
    with pytest.raises(ValueError, match="GPU"):   # all that is left to refuse: X is on the CPU
        model[1](X, POS)
    assert model.to("meta")[1].inv_freq.device.type == "meta"


def test_row_positions_refuses():
    lib = _lib.load()
    p = ctypes.c_void_p(16)   # never dereferenced
    for args, what in (((None, 1, 4, p, None), "null"), ((p, 1, 4, None, None), "null"), ((p, 0, 4, p, None), "shape"),
                       ((p, 1, -1, p, None), "shape")):
        assert lib.dsa_row_positions(*args) == _lib.DSA_ERR_INVALID and what in lib.dsa_last_error().decode()
    assert lib.dsa_row_positions(p, 1, 0, p, None) == 0   # no rows: no launch


def test_more_rows_than_a_call_takes():
    """Refused before any launch: the last groups' row numbers would overflow."""
    wide = torch.empty(1, 1, 1, 2, dtype=BF).expand(1, 2 ** 31 - 4096, 1, 2)
    pos = torch.empty(1, 1, dtype=torch.int32).expand(1, 2 ** 31 - 4096)
    with pytest.raises(ValueError, match="more than 2147479551 tokens"):
        dsa.rotary_embedding(wide, pos, torch.ones(1))
    lib, p = _lib.load(), ctypes.c_void_p(16)
    for rows in (2 ** 31 - 4096, 2 ** 31 - 1):
        assert lib.dsa_rotary(p, 0, 64, 64, 1, p, 0, 1, None, p, rows, rows, 2, 64, 0, 64, 1, 0, p, None) == _lib.DSA_ERR_UNSUPPORTED
        assert b"rows" in lib.dsa_last_error()
        lat = [p, 0, 512, p, 0, 64, 1, 512, None, 1, 1e-6, None, 0, 1, None, p, 1, p, p, p, 0, p, 2, rows, 4, 3, 16, 8, p, p, None]
        assert lib.dsa_latent_append(*lat) == _lib.DSA_ERR_UNSUPPORTED and b"rows" in lib.dsa_last_error()
