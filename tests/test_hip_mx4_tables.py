"""A packed table that is kept: copied, pickled, saved and loaded (``ops.Mx4Table``)."""
import copy
import copyreg
import io
import pickle

import pytest
import torch

from biomedkg_amd import ops


def _load(buf, **kw):
    return torch.load(io.BytesIO(buf), weights_only=False, **kw)


def _saved(table):
    buf = io.BytesIO()
    torch.save({"table": table}, buf)
    return buf.getvalue()


COPIES = {
    "copy": copy.copy,
    "deepcopy": copy.deepcopy,
    "deepcopy in a dict": lambda t: copy.deepcopy({"a": [t]})["a"][0],
    "pickle": lambda t: pickle.loads(pickle.dumps(t)),
    "oldest pickle": lambda t: pickle.loads(pickle.dumps(t, protocol=0)),
    "saved": lambda t: _load(_saved(t))["table"],
}


def host_table(whole, rows=5, cols=200):
    """a table on the host: codes and scales in one piece of memory, as a packed one has them, or in two"""
    gen = torch.Generator().manual_seed(rows + cols)
    panels = (cols + 127) // 128
    if whole:
        t = ops.Mx4Table._empty(rows, cols, "cpu")
        t.codes.copy_(torch.randint(0, 256, t.codes.shape, generator=gen))
        t.scales.copy_(torch.randint(100, 140, t.scales.shape, generator=gen))
        return t
    return ops.Mx4Table(torch.randint(0, 256, (panels, rows, 64), generator=gen).to(torch.uint8),
                        torch.randint(100, 140, (panels, rows, 4), generator=gen).to(torch.uint8), (rows, cols))


@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("how", list(COPIES))
def test_a_copy_reads_its_own_memory(how, whole):
    t = host_table(whole)
    c = COPIES[how](t)
    assert c.shape == t.shape and c.device == t.device and c.nbytes == t.nbytes
    assert torch.equal(c.codes, t.codes) and torch.equal(c.scales, t.scales)
    assert (c.codes_ptr, c.scales_ptr) == (c.codes.data_ptr(), c.scales.data_ptr())
    if how != "copy":
        assert c.codes_ptr != t.codes_ptr and c.scales_ptr != t.scales_ptr
        t.codes.zero_()
        assert bool(c.codes.any())


def test_addresses_before_and_after_the_parts_are_looked_at():
    t = ops.Mx4Table._empty(7, 300, "cpu")
    before = (t.codes_ptr, t.scales_ptr, t.device)
    assert before == (t.codes.data_ptr(), t.scales.data_ptr(), t.codes.device) == (t.codes_ptr, t.scales_ptr, t.device)


class WithAttributes(pickle.Pickler):
    """saves a table as its attributes, addresses among them, as tables were saved once"""

    def reducer_override(self, obj):
        if not isinstance(obj, ops.Mx4Table):
            return NotImplemented
        state = {"shape": obj.shape, "device": obj.device, "codes_ptr": 4096, "scales_ptr": 8192, "_store": obj._store}
        return copyreg.__newobj__, (ops.Mx4Table,), (None, state)


@pytest.mark.parametrize("whole", [True, False])
def test_addresses_in_a_saved_table_are_not_taken(whole):
    t, buf = host_table(whole), io.BytesIO()
    WithAttributes(buf, 4).dump(t)
    c = pickle.loads(buf.getvalue())
    assert torch.equal(c.codes, t.codes) and torch.equal(c.scales, t.scales) and c.shape == t.shape and c.device == t.device
    assert (c.codes_ptr, c.scales_ptr) == (c.codes.data_ptr(), c.scales.data_ptr())


def test_a_saved_table_is_written_once():
    t = ops.Mx4Table._empty(1000, 256, "cpu")
    t.codes.zero_()
    for size in (len(pickle.dumps(t)), len(_saved(t))):
        assert t.nbytes <= size <= 1.1 * t.nbytes


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["deepcopy", "pickle", "saved"])
def test_products_against_a_copy_outlive_the_original(how):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(40, 200, generator=gen).cuda()
    table = ops.mx4_quantize(torch.randn(3001, 200, generator=gen).cuda())
    want = [ops.mx4_linear(x, table), ops.mx4_linear(x[:2], table), ops.mx4_linear(ops.mx4_quantize(x), table),
            ops.mx4_dequantize(table)]
    c = COPIES[how](table)
    table.codes.zero_()
    table.scales.zero_()
    del table
    got = [ops.mx4_linear(x, c), ops.mx4_linear(x[:2], c), ops.mx4_linear(ops.mx4_quantize(x), c), ops.mx4_dequantize(c)]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_table_loaded_onto_the_host_and_back():
    gen = torch.Generator().manual_seed(2)
    table = ops.mx4_quantize(torch.randn(50, 96, generator=gen).cuda())
    host = _load(_saved(table), map_location="cpu")["table"]
    assert host.device.type == "cpu" and torch.equal(host.codes, table.codes.cpu())
    with pytest.raises(RuntimeError):                        # (and not a read of host memory on the device)
        ops.mx4_dequantize(host)
    back = ops.Mx4Table(host.codes.cuda(), host.scales.cuda(), host.shape)
    assert torch.equal(ops.mx4_dequantize(back), ops.mx4_dequantize(table))
