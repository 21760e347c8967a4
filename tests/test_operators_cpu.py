"""Refusals of the training operators: wrong arguments are named before anything reaches a GPU."""
import ctypes as C

import pytest
import torch


@pytest.fixture(autouse=True)
def _library(built_library):
    pass


def test_embedding_refuses():
    from landmark_b200.embedding import embedding, embedding_backward

    idx, w = torch.zeros(3, dtype=torch.long), torch.zeros(5, 4)
    with pytest.raises(ValueError, match="CUDA"):
        embedding(idx, w)
    with pytest.raises(TypeError, match="float64"):
        embedding(idx, w.double())
    with pytest.raises(ValueError, match="CUDA"):
        embedding_backward(torch.zeros(3, 4), idx, 5)
    with pytest.raises(TypeError, match="int64"):
        embedding_backward(torch.zeros(3, 4, dtype=torch.int64), idx, 5)


def test_c_entries_refuse():
    from landmark_b200 import _lib

    lib, p = _lib.lib, C.c_void_p(256)
    n = C.c_size_t(0)
    assert lib.gnr_embedding_grad_workspace_bytes(100, 11500, 48, C.byref(n)) == 0 and n.value == 0  # small: in shared memory
    assert lib.gnr_embedding_grad_workspace_bytes(100000, 11500, 48, C.byref(n)) == 0 and n.value >= 1600000
    for t, v, d in ((-1, 5, 4), (2 ** 31, 5, 4), (3, 0, 4), (3, 2 ** 31 - 1, 4), (3, 5, 0)):
        assert lib.gnr_embedding_grad_workspace_bytes(t, v, d, C.byref(n)) < 0
        assert lib.gnr_embedding_lookup(p, 0, v, d, d, p, 64, t, 1.0, p, d, None) < 0
    assert lib.gnr_embedding_grad_workspace_bytes(3, 5, 4, None) < 0
    assert lib.gnr_embedding_lookup(p, 3, 5, 4, 4, p, 64, 3, 1.0, p, 4, None) < 0  # no such type
    assert lib.gnr_embedding_lookup(p, 0, 5, 4, 4, p, 16, 3, 1.0, p, 4, None) < 0 and b"16 bits" in lib.gnr_last_error()
    assert lib.gnr_embedding_lookup(p, 0, 5, 4, 3, p, 64, 3, 1.0, p, 4, None) < 0  # rows that overlap
    assert lib.gnr_embedding_lookup(None, 0, 5, 4, 4, p, 64, 3, 1.0, p, 4, None) < 0
    assert lib.gnr_embedding_lookup(None, 0, 5, 4, 4, None, 64, 0, 1.0, None, 4, None) == 0  # nothing to do
    assert lib.gnr_embedding_grad(p, 0, 4, 4, p, 64, 5000, 5, -1, 1.0, 0, p, 0, 4, p, 16, None) < 0 and b"workspace" in lib.gnr_last_error()
    assert lib.gnr_embedding_grad(p, 0, 4, 4, p, 64, 3, 5, -1, 1.0, 0, p, 0, 3, p, 1 << 30, None) < 0
    assert lib.gnr_embedding_grad(p, 0, 4, 4, p, 64, 3, 5, -1, 1.0, 0, p, 7, 4, p, 1 << 30, None) < 0
    assert lib.gnr_embedding_grad(p, 0, 4, 4, None, 64, 3, 5, -1, 1.0, 0, p, 0, 4, p, 1 << 30, None) < 0
    assert lib.gnr_embedding_grad(p, 0, 4, 4, p, 64, 5000, 5, -1, 1.0, 0, p, 0, 4, None, 1 << 30, None) < 0
    assert lib.gnr_embedding_grad(p, 0, 4, 4, p, 64, 5000, 5, -1, 1.0, 0, p, 0, 4, C.c_void_p(264), 1 << 30, None) < 0  # not on 16 bytes


def test_adamw_entry_refuses():
    from landmark_b200 import _lib

    def call(n=10, bits=32, step=1, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, decay=0.0, ptype=0, gtype=0, **fields):
        t = (_lib.GnrAdamwTensor * 1)()
        for k, v in {"param": 256, "grad": 256, "exp_avg": 256, "exp_avg_sq": 256, "n": n, **fields}.items():
            setattr(t[0], k, v)
        return _lib.lib.gnr_adamw_step(t, 1, ptype, gtype, bits, step, lr, b1, b2, eps, decay, 0, None)

    for bad in ({"bits": 16}, {"step": 0}, {"lr": -1.0}, {"lr": float("nan")}, {"lr": float("inf")}, {"b1": 1.0}, {"b2": -0.1}, {"eps": 0.0}, {"eps": float("nan")},
                {"decay": -1.0}, {"ptype": 5}, {"gtype": -1}, {"n": -1}, {"param": None}, {"grad": None}, {"exp_avg": None}, {"exp_avg_sq": None},
                {"bits": 8}, {"master": 256}):
        assert call(**bad) < 0, bad
        assert _lib.lib.gnr_last_error()
    assert call(n=0) == 0
    assert _lib.lib.gnr_adamw_step(None, 0, 0, 0, 32, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, None) == 0


def test_clock_entries_refuse():
    from landmark_b200 import _lib

    lib, p = _lib.lib, C.c_void_p(256)
    assert lib.gnr_adamw_clock_set(None, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, None) < 0
    assert lib.gnr_adamw_clock_set(C.c_void_p(257), 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, None) < 0
    for bad in ((-2, 1e-3, 0.9, 0.999, 1e-8, 0.0), (0, -1.0, 0.9, 0.999, 1e-8, 0.0), (0, 1e-3, 1.0, 0.999, 1e-8, 0.0), (0, 1e-3, 0.9, 1.0, 1e-8, 0.0),
                (0, 1e-3, 0.9, 0.999, 0.0, 0.0), (0, 1e-3, 0.9, 0.999, 1e-8, -1.0)):
        assert lib.gnr_adamw_clock_set(p, *bad, 0, None) < 0, bad
    assert lib.gnr_adamw_clock_advance(None, None) < 0
    t = (_lib.GnrAdamwTensor * 1)()
    assert lib.gnr_adamw_step_clocked(t, 1, 0, 0, 32, None, None) < 0
    t[0].n = 5
    assert lib.gnr_adamw_step_clocked(t, 1, 0, 0, 32, p, None) < 0
    t[0].n = 0
    assert lib.gnr_adamw_step_clocked(t, 1, 0, 0, 32, p, None) == 0


def test_adamw_refuses():
    from landmark_b200.optim import AdamW, AdamWClock, AdamWTensors, state_blocks

    x = torch.zeros(4)
    with pytest.raises(ValueError, match="CUDA"):
        AdamWClock("cpu", lr=1e-3)
    with pytest.raises(ValueError, match="CUDA"):
        AdamWTensors([x], [x], [x])
    with pytest.raises(TypeError, match="float64"):
        AdamWTensors([x.double()], [x], [x])
    with pytest.raises(ValueError, match="no tensors"):
        AdamWTensors([], [], [])
    for bad in ({"state_bits": 16}, {"lr": -1.0}, {"eps": 0.0}, {"betas": (1.0, 0.9)}, {"weight_decay": -1.0}):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(x)], **bad)
    assert [state_blocks(n) for n in (0, 1, 256, 257)] == [0, 1, 1, 2]
    p = torch.nn.Parameter(x)
    opt = AdamW([p])
    opt.step()  # nothing has a gradient
    p.grad = torch.zeros(4)
    with pytest.raises(ValueError, match="CUDA"):
        opt.step()


def test_random_bits_are_even():
    """The hash that decides roundings: over neighbouring places and over neighbouring steps every one of its 32 bits is set in half of
    the cases (6 standard deviations), and so is the exclusive or of neighbours."""
    def hash32(i, seed):
        mask = 0xFFFFFFFF
        x = (i * 0x9E3779B9 + seed) & mask
        x = x ^ (x >> 16)
        x = (x * 0x6A09E667) & mask
        x = x ^ (x >> 15)
        x = (x * 0xBB67AE85) & mask
        return x ^ (x >> 16)

    n = 1 << 16
    i = torch.arange(n, dtype=torch.int64)
    for h in (hash32(i, 0), hash32(i, hash32(3, hash32(1000, 7))), hash32(77, hash32(2, hash32(i, 5)))):
        for x in (h, h ^ h.roll(1), h ^ h.roll(256)):
            for b in range(32):
                assert abs(int(((x >> b) & 1).sum()) - n / 2) <= 6 * (n / 4) ** 0.5


def test_adamw_refusals_leave_no_state():
    from landmark_b200.optim import AdamW

    for dtype in (torch.float32, torch.bfloat16):
        p = torch.nn.Parameter(torch.zeros(4, dtype=dtype))
        opt = AdamW([p])
        p.grad = torch.zeros_like(p)
        with pytest.raises(ValueError, match="CUDA"):
            opt.step()
        assert len(opt.state) == 0 and opt.state_dict()["state"] == {}


def test_adamw_refuses_groups_it_would_not_obey():
    from landmark_b200.optim import AdamW

    def params():
        return [torch.nn.Parameter(torch.zeros(4)) for _ in range(2)]

    def state_of(cls, **options):
        ps = params()
        opt = cls(ps, lr=0.25, **options)
        for p in ps:
            p.grad = torch.ones(4)
        opt.step()
        return opt.state_dict()

    bad = [(torch.optim.AdamW, {"maximize": True}), (torch.optim.AdamW, {"amsgrad": True}), (torch.optim.Adam, {"weight_decay": 0.1}),
           (torch.optim.Adam, {"maximize": True})]
    for cls, options in bad:
        opt = AdamW(params(), lr=0.5)
        with pytest.raises(ValueError, match="not offered"):
            opt.load_state_dict(state_of(cls, **options))
        assert opt.param_groups[0]["lr"] == 0.5 and len(opt.state) == 0  # nothing has been replaced
    for cls, options in ((torch.optim.AdamW, {}), (torch.optim.Adam, {}), (torch.optim.AdamW, {"foreach": True})):
        opt = AdamW(params(), lr=0.5)
        opt.load_state_dict(state_of(cls, **options))
        assert opt.param_groups[0]["lr"] == 0.25 and [s["step"] for s in opt.state.values()] == [1, 1]
    for name, value in (("maximize", True), ("amsgrad", True), ("differentiable", True), ("decoupled_weight_decay", False)):
        with pytest.raises(ValueError, match="not offered"):
            AdamW([{"params": params(), name: value}], weight_decay=0.1)
        opt = AdamW(params(), weight_decay=0.1)
        with pytest.raises(ValueError, match="not offered"):
            opt.add_param_group({"params": params(), name: value})
        assert len(opt.param_groups) == 1
        opt.param_groups[0][name] = value
        with pytest.raises(ValueError, match="not offered"):
            opt.step()
    opt = AdamW([{"params": params(), "decoupled_weight_decay": False, "weight_decay": 0.0, "maximize": False}], weight_decay=0.1)
    opt.step()


def test_adamw_obeys_hooks_of_loading():
    """Hooks change what is loaded before, and see and change what has been loaded after, as with torch's optimisers."""
    from landmark_b200.optim import AdamW

    p, q = (torch.nn.Parameter(torch.zeros(4, dtype=torch.bfloat16)) for _ in range(2))
    state = {"step": 3, "exp_avg": torch.ones(4), "exp_avg_sq": torch.ones(4), "master": torch.ones(4)}
    saved = AdamW([q]).state_dict()
    saved["state"][0] = state
    opt = AdamW([p])
    seen = []

    def before(_, d):
        return {**d, "state": {0: {**d["state"][0], "step": 7}}, "param_groups": [{**d["param_groups"][0], "lr": 0.125}]}

    def after(o):
        seen.append((o.state[p]["step"], o.state[p]["exp_avg"].dtype))
        o.state[p]["step"] = 9

    handles = opt.register_load_state_dict_pre_hook(before), opt.register_load_state_dict_post_hook(after)
    opt.load_state_dict(saved)
    assert seen == [(7, torch.float32)] and opt.state[p]["step"] == 9 and opt.param_groups[0]["lr"] == 0.125
    assert state["step"] == 3
    for h in handles:
        h.remove()
    opt.load_state_dict(saved)
    assert opt.state[p]["step"] == 3 and opt.state[p]["master"] is not state["master"] and len(seen) == 1
    assert len(opt._optimizer_load_state_dict_pre_hooks) == len(opt._optimizer_load_state_dict_post_hooks) == 0
    bad = opt.register_load_state_dict_pre_hook(lambda o, d: {**d, "param_groups": [{**d["param_groups"][0], "maximize": True}]})
    with pytest.raises(ValueError, match="not offered"):
        opt.load_state_dict(saved)
    bad.remove()
    assert len(opt._optimizer_load_state_dict_pre_hooks) == len(opt._optimizer_load_state_dict_post_hooks) == 0


def test_shared_memory_is_found():
    """Ranges of the tensors of a step: every pair of overlapping ones among many, neighbours that only touch are none."""
    from landmark_b200.optim import _shared

    apart = [(1000 + 16 * k, 16, k) for k in range(50)]
    assert _shared([]) is None and _shared(apart) is None and _shared(apart[::-1]) is None
    for k in range(50):
        for at, size in ((1000 + 16 * k, 1), (1000 + 16 * k + 15, 1), (1000 + 16 * k + 3, 200), (1000 + 16 * k - 4, 5), (0, 10000)):
            assert _shared(apart + [(at, size, "new")]) is not None
    assert _shared(apart + [(1800, 4, "new"), (996, 4, "other")]) is None


def test_rows_that_share_memory_are_found():
    """Against sets of bytes, for all small layouts of two arrays of rows."""
    from landmark_b200.embedding import _rows_share

    def bytes_of(at, rows, stride, width):
        return {at + r * stride + k for r in range(rows) for k in range(width)}

    for a_rows, a_stride, a_width in ((1, 4, 4), (3, 4, 4), (4, 12, 4), (2, 16, 6), (5, 6, 2)):
        for b_rows, b_stride, b_width in ((1, 2, 2), (4, 4, 4), (3, 12, 8), (2, 12, 4), (3, 16, 8), (7, 6, 4), (1, 40, 40)):
            for b in range(100):
                want = bool(bytes_of(50, a_rows, a_stride, a_width) & bytes_of(b, b_rows, b_stride, b_width))
                assert _rows_share(50, a_rows, a_stride, a_width, b, b_rows, b_stride, b_width) == want
    # columns of one wide buffer, many rows
    assert not _rows_share(0, 10 ** 9, 800, 400, 400, 10 ** 9, 800, 400) and _rows_share(0, 10 ** 9, 800, 404, 400, 10 ** 9, 800, 400)


def test_adamw_entry_passes_over_tensors_without_values():
    """They have no addresses, and no say in whether the others have a 32-bit copy: what is refused is a mix among those with values."""
    from landmark_b200 import _lib

    def call(*tensors, bits=32):
        t = (_lib.GnrAdamwTensor * len(tensors))()
        for k, (n, master) in enumerate(tensors):
            t[k].n = n
            if n:
                t[k].param = t[k].grad = t[k].exp_avg = t[k].exp_avg_sq = t[k].exp_avg_scale = t[k].exp_avg_sq_scale = 256
            if master:
                t[k].master = 256
        return _lib.lib.gnr_adamw_step(t, len(tensors), _lib.BF16, _lib.BF16, bits, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, None), _lib.lib.gnr_last_error()

    for bits in (8, 32):
        assert call((0, False), (0, True), bits=bits)[0] == 0  # nothing to do
        for mix in (((10, True), (0, True), (10, False)), ((0, False), (10, True), (10, False)), ((0, True), (10, False), (0, False), (10, True))):
            rc, why = call(*mix, bits=bits)
            assert rc < 0 and b"tensor %d of 10 values" % (len(mix) - 1) in why
