"""What the torch-side holders of the paged cache refuse, on tensors without memory: no GPU is needed."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from fblt_b200 import ops

pytestmark = pytest.mark.filterwarnings("ignore:Accessing the data pointer")


@pytest.fixture(autouse=True)
def fake():
    with FakeTensorMode():
        yield


def pool(**device):
    """The tensors of a cache of 8 pages of 16 positions, 2 kv heads of 64."""
    on = lambda name: device.get(name, "cuda:0")  # noqa: E731
    t = {n: torch.empty(8, 2, 16, 64, dtype=torch.uint8, device=on(n)) for n in ("k_codes", "v_codes")}
    t.update({n: torch.empty(8, 2, 16, dtype=torch.int8, device=on(n)) for n in ("k_exp", "v_exp")})
    t["page_table"] = torch.empty(3, 4, dtype=torch.int32, device=on("page_table"))
    return t


def test_page_tables_whose_rows_overlap_are_refused():
    t = pool()
    row = torch.empty(1, 4, dtype=torch.int32, device="cuda")
    for table in (row.expand(3, 4), torch.empty(12, dtype=torch.int32, device="cuda").as_strided((3, 4), (3, 1))):
        with pytest.raises(ValueError, match="page_table"):
            ops.PagedKvCache(**{**t, "page_table": table}, fmt="int8")


def test_page_tables_that_are_accepted():
    t = pool()
    wide = torch.empty(6, 9, dtype=torch.int32, device="cuda")
    for table, stride in ((wide[:, :4], 9), (wide[::2, 2:6], 18), (wide[:1, :4], 9), (wide[:3, :0], 9),
                          (torch.empty(1, 1, dtype=torch.int32, device="cuda").expand(1, 1), 1),
                          (torch.empty(4, dtype=torch.int32, device="cuda").as_strided((1, 4), (1, 1)), 4)):
        c = ops.PagedKvCache(**{**t, "page_table": table}, fmt="e4m3")
        assert (c.batch, c.desc.max_pages, c.desc.page_table_stride) == (*table.shape, stride)


@pytest.mark.parametrize("name", ["k_codes", "v_codes", "k_exp", "v_exp", "page_table"])
def test_a_cache_lies_on_one_device(name):
    with pytest.raises(ValueError, match="device"):
        ops.PagedKvCache(**pool(**{name: "cuda:1"}), fmt="int8")


def attn(cache, rows=3):
    i32 = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
    q, out = (torch.empty(rows, 256, device="cuda") for _ in range(2))
    return ops.make_paged_attn(cache, i32(4), i32(3), q, out, 4, 1, 64, 0.125, splits=4)


def test_workspaces_elsewhere_are_refused():
    d = attn(ops.PagedKvCache(**pool(), fmt="int8"))
    byte = dict(dtype=torch.uint8)
    for ws in (torch.empty(1 << 20, device="cpu", **byte), torch.empty(1 << 20, device="cuda:1", **byte),
               torch.empty(1 << 21, device="cuda", **byte)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            ops.paged_attn(d, ws)


def test_a_single_row_of_any_stride():
    """What a transposed column, or a slice of one row, gives for a row stride is not looked at."""
    cache = ops.PagedKvCache(**pool(), fmt="int8")
    i32 = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
    col = lambda n, **kw: torch.empty(n, 1, device="cuda", **kw).t()  # noqa: E731
    a = ops.make_paged_attn(cache, i32(4), i32(3), col(256), torch.empty(4, 259, device="cuda")[:1, :256], 4, 1, 64, 0.125)
    assert (a.q_stride, a.out_stride) == (256, 256)
    w = ops.make_paged_append(cache, i32(4), i32(3), col(128), col(128), q=col(256), num_heads=4)
    assert (w.k_stride, w.v_stride, w.q_stride, w.q_out_stride) == (128, 128, 256, 256)
    r = ops.make_paged_read(cache, i32(4), col(128, dtype=torch.bfloat16), None)
    assert r.k_out_stride == 128
    n = ops.make_qk_norm_rope(col(256), col(128), i32(1), 4, 2, 64)
    assert (n.q_stride, n.q_out_stride, n.k_stride, n.k_out_stride) == (256, 256, 128, 128)
    two = torch.empty(2, 300, device="cuda")[:, :256]
    assert ops.make_qk_norm_rope(two, None, i32(2), 4, 0, 64).q_stride == 300
