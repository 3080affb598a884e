"""What the router, the gated norms and the adapters refuse of their tensors' shapes and memory before any launch
(no GPU needed: the device check is left out, and no call may reach the library)."""
import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def no_launch(monkeypatch):
    from kb_nano_amd import _ops

    def lib():
        raise AssertionError("launched")
    monkeypatch.setattr(_ops, "_dev_check", lambda what, *t: 0)
    monkeypatch.setattr(_ops, "_host", None)
    monkeypatch.setattr(_ops, "lib", lib)
    return _ops


# ------------------------------------------------------------ adapters' ids

def lora_inputs(*lead):
    n = 1
    for v in lead:
        n *= v
    return (torch.zeros(*lead, 64, dtype=BF16), torch.zeros(*lead, 32, dtype=BF16), torch.zeros(2, 8, 64, dtype=BF16),
            torch.zeros(2, 32, 8, dtype=BF16))


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("lead,ids", [((2, 3), (3, 2)), ((2, 3, 4), (4, 3, 2)), ((2, 3, 4), (6, 4)), ((2, 1, 3), (3, 2)), ((4,), (3,)), ((2, 3), (5,))])
def test_ids_of_another_shape_are_refused(no_launch, lead, ids, inplace):
    """Ids [S, B] beside x [B, S, K] would give tokens each other's adapters."""
    from kb_nano_amd import LoraAdd
    with pytest.raises(ValueError, match="adapter_ids"):
        LoraAdd()(*lora_inputs(*lead), torch.zeros(ids, dtype=torch.int32), None, inplace)


@pytest.mark.parametrize("lead,ids", [((2, 3), (2, 3)), ((2, 3), (6,)), ((6,), (2, 3)), ((2, 1, 3), (2, 3)), ((4, 1), (4,)), ((4,), (4, 1)),
                                      ((4,), (1, 4)), ((), (1,)), ((), ())])
def test_ids_in_the_rows_order_are_taken(no_launch, lead, ids):
    """As x's leading dimensions, flat, or beside flat rows."""
    from kb_nano_amd import LoraAdd
    with pytest.raises(AssertionError, match="launched"):
        LoraAdd()(*lora_inputs(*lead), torch.zeros(ids, dtype=torch.int32))


# ------------------------------------------------------------ shared memory

def norm_args(T=4, H=256):
    d = {k: torch.zeros(T, H, dtype=BF16) for k in ("x", "r", "gate", "r_out", "n_out")}
    d.update(w=torch.zeros(H, dtype=BF16), post=torch.zeros(H, dtype=BF16), q=torch.zeros(T, H, dtype=torch.float8_e4m3fn),
             s=torch.zeros(T, H // 128))
    return d


def run_norm(ops, d):
    ops.gated_add_rmsnorm(d["x"], d["r"], d["w"], d["post"], d["gate"], 1.0, 1e-6, d["r_out"], d["n_out"], d["q"], d["s"])


def bytes_of(t, like):
    """Memory of t as a tensor of like's type and shape (from its start)."""
    return t.view(torch.uint8).reshape(-1)[:like.numel() * like.element_size()].view(like.dtype).view(like.shape)


@pytest.mark.parametrize("out", ["r_out", "n_out", "q", "s"])
@pytest.mark.parametrize("read", ["x", "r", "gate", "w", "post"])
def test_gated_norm_outputs_over_what_is_read(no_launch, out, read):
    d = norm_args()
    if out == "r_out" and read == "r":
        return
    if d[out].numel() * d[out].element_size() <= d[read].numel() * d[read].element_size():
        d[out] = bytes_of(d[read], d[out])
    else:
        d[read] = bytes_of(d[out], d[read])
    with pytest.raises(ValueError, match="overlaps"):
        run_norm(no_launch, d)


@pytest.mark.parametrize("a,b", [("r_out", "n_out"), ("r_out", "q"), ("r_out", "s"), ("n_out", "q"), ("n_out", "s"), ("q", "s")])
def test_gated_norm_outputs_over_each_other(no_launch, a, b):
    d = norm_args()
    d[b] = bytes_of(d[a], d[b])
    with pytest.raises(ValueError, match="overlaps"):
        run_norm(no_launch, d)


def test_gated_norm_residual_in_place(no_launch):
    d = norm_args()
    run = lambda: run_norm(no_launch, d)   # noqa: E731
    with pytest.raises(AssertionError, match="launched"):
        run()
    d["r_out"] = d["r"]
    with pytest.raises(AssertionError, match="launched"):
        run()
    store = torch.zeros(5 * 256 + 256, dtype=BF16)
    d["r"], d["r_out"] = store[:4 * 256].view(4, 256), store[256:5 * 256].view(4, 256)     # a row apart
    with pytest.raises(ValueError, match="overlaps"):
        run()
    d["r"], d["r_out"] = store[:4 * 256].view(4, 256), store.as_strided((4, 256), (264, 1))     # another stride
    with pytest.raises(ValueError, match="overlaps"):
        run()
    d = norm_args()
    d["r"] = d["x"]      # both only read
    d["gate"] = d["x"]
    with pytest.raises(AssertionError, match="launched"):
        run()


def test_columns_of_one_buffer_do_not_overlap(no_launch):
    d = norm_args()
    store = torch.zeros(4, 1024, dtype=BF16)
    for i, k in enumerate(("x", "r", "r_out", "n_out")):
        d[k] = store[:, 256 * i:256 * (i + 1)]
    packed = torch.zeros(4, 256 + 8, dtype=torch.uint8)      # a row's codes, its scales behind them
    d["q"], d["s"] = packed[:, :256].view(torch.float8_e4m3fn), packed[:, 256:].view(F32)
    with pytest.raises(AssertionError, match="launched"):
        run_norm(no_launch, d)
    wide = torch.zeros(4, 1032, dtype=BF16)      # a gate for each token beside the rows
    e = {**d, **{k: wide[:, 256 * i:256 * (i + 1)] for i, k in enumerate(("x", "r", "r_out", "n_out"))}}
    with pytest.raises(AssertionError, match="launched"):
        run_norm(no_launch, {**e, "gate": wide[:, 1024:1025].expand(4, 256)})
    with pytest.raises(ValueError, match="overlaps gate"):
        run_norm(no_launch, {**e, "gate": wide[:, 1000:1001].expand(4, 256)})
    for k, v in (("n_out", store[:, 504:760]), ("r_out", store[:, 8:264]), ("n_out", store[:, 248:504]), ("x", store[:, 760:1016]),
                 ("s", packed[:, 248:256].view(F32))):
        e = {**d, k: v}
        with pytest.raises(ValueError, match="overlaps"):
            run_norm(no_launch, e)


@pytest.mark.parametrize("which", ["x", "weight"])
def test_router_product_over_what_is_read(no_launch, which):
    store = torch.zeros(16 * 256, dtype=F32)
    a, b = store.view(16, 256), torch.zeros(16, 256, dtype=F32)
    x, w = (a, b) if which == "x" else (b, a)
    with pytest.raises(ValueError, match="overlaps"):
        no_launch.moe_router_gemm(x, w, store[:256].view(16, 16))
    with pytest.raises(AssertionError, match="launched"):
        no_launch.moe_router_gemm(x, w, torch.zeros(16, 16))


def test_choice_over_what_is_read(no_launch):
    call = lambda l, b, w, i: no_launch.moe_router_topk(l, 4, "softmax", b, 1, 1, True, 1.0, w, i)   # noqa: E731
    l, bias, w, ids = torch.zeros(8, 64), torch.zeros(64), torch.zeros(8, 4), torch.zeros(8, 4, dtype=torch.int32)
    with pytest.raises(AssertionError, match="launched"):
        call(l, bias, w, ids)
    with pytest.raises(ValueError, match="overlaps"):
        call(l, bias, l.view(-1)[:32].view(8, 4), ids)
    with pytest.raises(ValueError, match="overlaps"):
        call(l, bias, w, l.view(torch.int32).view(-1)[:32].view(8, 4))
    with pytest.raises(ValueError, match="overlaps"):
        call(l, bias, bias[:32].view(8, 4), ids)
    with pytest.raises(ValueError, match="overlaps"):
        call(l, bias, w, w.view(torch.int32))
