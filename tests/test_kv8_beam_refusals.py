"""What the 8-bit cache and beam search refuse, and that they do so before anything touches a device (no GPU needed)."""
import ctypes

import pytest
import torch

from spec_mcts_amd import _lib, kernels as K

half, i32, u8 = torch.float16, torch.int32, torch.uint8


def cache(B=2, cols=3, Hkv=2, n=7):
    return [torch.zeros((n, Hkv, 64, 128), dtype=u8), torch.zeros((n, Hkv, 128, 64), dtype=u8), torch.zeros((n, Hkv, 2)), torch.zeros((B, Hkv, 64, 128), dtype=half),
            torch.zeros((B, Hkv, 128, 64), dtype=half), torch.zeros((B, cols), dtype=i32)]


def append_args():
    return dict(q=torch.zeros((2, 4, 128), dtype=half), k=torch.zeros((2, 2, 128), dtype=half), v=torch.zeros((2, 2, 128), dtype=half), cos=torch.zeros((9, 64), dtype=half),
                sin=torch.zeros((9, 64), dtype=half), cache=cache(), lens=torch.zeros(2, dtype=i32), cu=None, max_new=1, out=None)


def attn_args():
    return dict(q=torch.zeros((2, 4, 128), dtype=half), cache=cache(), lens=torch.zeros(2, dtype=i32), cu=None, max_new=1, max_len=None, window=0, sinks=0, out=None)


def rows_args():
    return dict(cache=cache(), total=torch.zeros(2, dtype=i32), first=torch.zeros(2, dtype=i32), count=5)


def select_args():
    return dict(logits=torch.zeros((6, 50), dtype=half), scores=torch.zeros(6), beams=3, n=4, ended=None, eos=2)


def reorder_args():
    return dict(parents=torch.zeros((2, 3), dtype=i32), rows=[torch.zeros((6, 8))], columns=[torch.zeros((6, 9), dtype=i32)], upto=torch.zeros(1, dtype=i32))


OPS = {"append": (K.kv8_append, append_args), "attn": (K.kv8_attn, attn_args), "rows": (K.kv8_rows, rows_args), "select": (K.beam_select, select_args),
       "reorder": (K.beam_reorder, reorder_args)}
wide = lambda t: torch.stack((t, t), -1)[..., 0]                             # noqa: E731  (the same values, not contiguous)
CACHE_CHANGES = [(i, f) for i in range(6) for f in ("type", "narrow", "wide")] + [(3, "few"), (4, "few"), (5, "few"), (None, "five")]
CHANGES = ([("append", a, b) for a, b in [("q", "float"), ("k", "float"), ("v", "float"), ("q", "wide"), ("k", "wide"), ("q", "short"), ("k", "short"), ("v", "short"), ("q", "narrow"),
                                          ("k", "narrow"), ("q", "heads"), ("k", "heads"), ("cos", "float"), ("sin", "float"), ("cos", "narrow"), ("sin", "short"), ("cos", "wide"),
                                          ("lens", "long"), ("lens", "more"), ("cu", "few"), ("cu", "long"), ("max_new", 2), ("max_new", -1), ("out", "short"), ("out", "float"),
                                          ("q", "odd stride")]]
           + [("attn", a, b) for a, b in [("q", "float"), ("q", "wide"), ("q", "short"), ("q", "narrow"), ("q", "heads"), ("lens", "long"), ("cu", "few"), ("max_new", 3), ("max_new", -1),
                                          ("max_len", 0), ("window", -1), ("sinks", -1), ("out", "short"), ("out", "float"), ("q", "odd stride")]]
           + [("rows", a, b) for a, b in [("total", "long"), ("first", "long"), ("first", "more"), ("count", -1)]]
           + [(op, "cache", c) for op in ("append", "attn", "rows") for c in CACHE_CHANGES]
           + [("select", a, b) for a, b in [("logits", "float"), ("logits", "wide"), ("scores", "double"), ("scores", "short"), ("scores", "wide"), ("beams", 4), ("beams", 0), ("n", 0),
                                            ("ended", "float"), ("ended", "short")]]
           + [("reorder", a, b) for a, b in [("parents", "long"), ("parents", "wide"), ("upto", "none"), ("upto", "long"), ("rows", "short"), ("rows", "wide"), ("columns", "short"),
                                             ("columns", "half"), ("columns", "cube"), ("rows", "many")]])


def changed(x, how):
    return {"float": lambda: x.float(), "double": lambda: x.double(), "half": lambda: x.to(half), "long": lambda: x.long(), "wide": lambda: wide(x), "short": lambda: x[:-1],
            "more": lambda: torch.cat((x, x)), "narrow": lambda: x[..., :-8].contiguous(), "few": lambda: x[:1], "heads": lambda: x[:, :1].repeat(1, 3, 1),
            "odd stride": lambda: torch.zeros((2, 4 * 128 + 4), dtype=half)[:, :512].view(2, 4, 128), "cube": lambda: x[..., None]}[how]()


@pytest.mark.parametrize("op,name,change", CHANGES, ids=str)
def test_tensors_of_another_kind_are_refused(op, name, change):
    call, args = OPS[op][0], OPS[op][1]()
    if name == "cache":
        i, how = change
        c = args["cache"]
        if how == "five":
            c.pop()
        else:
            c[i] = {"type": lambda: c[i].double(), "narrow": lambda: c[i][..., :-1].contiguous() if i < 5 else c[i].long(), "wide": lambda: wide(c[i]), "few": lambda: c[i][:1]}[how]()
    elif name == "cu":
        args["cu"] = torch.zeros(2, dtype=i32) if change == "few" else torch.zeros(3, dtype=torch.long)
    elif name == "out":
        args["out"] = torch.zeros((1, 4, 128), dtype=half) if change == "short" else torch.zeros((2, 4, 128))
    elif name == "ended":
        args["ended"] = torch.zeros(6) if change == "float" else torch.zeros(5, dtype=u8)
    elif name == "upto" and change == "none":
        args["upto"] = None
    elif name in ("rows", "columns") and op == "reorder":
        args[name] = [args[name][0].clone() for _ in range(17)] if change == "many" else [changed(args[name][0], change)]
    elif isinstance(change, int):
        args[name] = change
    else:
        args[name] = changed(args[name], change)
    with pytest.raises(AssertionError) as e:
        call(**args)
    assert "no CPU fallback" not in str(e.value)


@pytest.mark.parametrize("op", list(OPS))
def test_host_tensors_are_refused_last(op):
    with pytest.raises(AssertionError, match="no CPU fallback"):
        OPS[op][0](**OPS[op][1]())


def err():
    return _lib.load().smh_last_error_string()


def c_cache(**kw):
    a = dict(codes_k=1 << 20, codes_v=1 << 21, scales=1 << 22, open_k=1 << 23, open_v=1 << 24, pages=1 << 12, n_pages=9, stride=4, cols=4)
    a.update(kw)
    return a


def c_append(**kw):
    a = dict(q=1 << 25, k=1 << 26, v=1 << 27, out=1 << 28, T=3, B=3, H=8, Hkv=2, D=128, qs=1024, ks=256, vs=256, cos=1 << 13, sin=1 << 14, table_rows=9, lens=1 << 11, cu=None, max_new=1)
    a.update(c_cache())
    a["stream"] = None
    a.update(kw)
    return _lib.load().smh_kv8_append(*a.values())


def c_attn(**kw):
    a = dict(q=1 << 25, out=1 << 28, T=3, B=3, H=8, Hkv=2, D=128, qs=1024, lens=1 << 11, cu=None, max_new=1, max_len=100, window=0, sinks=0)
    a.update(c_cache())
    a.update(ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return _lib.load().smh_kv8_attn(*a.values())


def c_rows(**kw):
    a = dict(k=1 << 25, v=1 << 26, B=3, Hkv=2, D=128, total=1 << 11, first=1 << 10, count=5)
    a.update(c_cache())
    a["stream"] = None
    a.update(kw)
    return _lib.load().smh_kv8_rows(*a.values())


CACHE_BAD = [(dict(D=64), b"head dim"), (dict(codes_k=None), b"null"), (dict(pages=None), b"null"), (dict(codes_v=(1 << 21) + 8), b"aligned"), (dict(scales=(1 << 22) + 4), b"aligned"),
             (dict(open_k=(1 << 23) + 2), b"aligned"), (dict(open_v=(1 << 24) + 8), b"aligned"), (dict(n_pages=0), b"n_pages"), (dict(cols=-1), b"cols"), (dict(cols=5), b"stride"),
             (dict(cols=1 << 23, stride=1 << 23), b"cols"), (dict(B=0, T=0), b"B="), (dict(B=65536, T=65536), b"B="), (dict(Hkv=0), b"Hkv")]


@pytest.mark.parametrize("call", [c_append, c_attn, c_rows])
@pytest.mark.parametrize("bad,why", CACHE_BAD, ids=lambda x: str(x))
def test_c_calls_refuse_a_bad_cache(call, bad, why):
    if call is c_rows:
        bad = {k: v for k, v in bad.items() if k != "T"}
    assert call(**bad) < 0 and why in err()


@pytest.mark.parametrize("bad,why", [(dict(H=7), b"H="), (dict(T=4), b"without cu"), (dict(T=-1, B=3, cu=1 << 9), b"T="), (dict(max_new=-1, cu=1 << 9), b"max_new"), (dict(table_rows=0), b"table"),
                                     (dict(qs=1016), b"stride"), (dict(ks=257), b"stride"), (dict(vs=248), b"stride"), (dict(q=None), b"null"), (dict(lens=None), b"null"),
                                     (dict(q=(1 << 25) + 8), b"aligned"), (dict(out=(1 << 28) + 8), b"aligned"), (dict(cos=(1 << 13) + 8), b"aligned")], ids=str)
def test_c_append_refuses(bad, why):
    assert c_append(**bad) < 0 and why in err()


@pytest.mark.parametrize("bad,why", [(dict(H=7), b"H="), (dict(T=4), b"without cu"), (dict(max_new=-1, cu=1 << 9), b"max_new"), (dict(max_len=0), b"max_len"), (dict(window=-1), b"window"),
                                     (dict(sinks=-1), b"sinks"), (dict(window=(1 << 29) + 1), b"window"), (dict(qs=1016), b"stride"), (dict(q=None), b"null"), (dict(out=(1 << 28) + 8), b"aligned"),
                                     (dict(max_len=10 ** 6), b"workspace"), (dict(max_len=10 ** 6, ws=1 << 29, ws_bytes=1000), b"workspace"),
                                     (dict(max_len=10 ** 6, ws=(1 << 29) + 4, ws_bytes=1 << 40), b"workspace")], ids=str)
def test_c_attn_refuses(bad, why):
    assert c_attn(**bad) < 0 and why in err()


def test_nothing_to_do_is_no_error():
    assert c_append(T=0, cu=1 << 9) == 0 and c_attn(T=0, cu=1 << 9) == 0 and c_append(max_new=0, cu=1 << 9) == 0 and c_rows(count=0) == 0
    lib = _lib.load()
    assert lib.smh_beam_reorder(1 << 12, 1, 1, 0, None, None, None, None, None, None) == 0


def test_workspaces():
    lib = _lib.load()
    assert lib.smh_kv8_attn_workspace_bytes(3, 3, 8, 2, 1, 100, 0, 0) == 0                    # one part
    assert lib.smh_kv8_attn_workspace_bytes(1, 1, 32, 32, 1, 4096, 0, 0) % (32 * 130 * 4) == 0
    for bad in ((0, 1, 1, 1, 1, 1, 0, 0), (1, 0, 1, 1, 1, 1, 0, 0), (1, 1, 3, 2, 1, 1, 0, 0), (1, 1, 1, 1, 0, 1, 0, 0), (1, 1, 1, 1, 1, 0, 0, 0), (1, 1, 1, 1, 1, 1, -1, 0)):
        assert lib.smh_kv8_attn_workspace_bytes(*bad) == 0
    # a window keeps a long sequence from being cut into more parts than it shows
    assert lib.smh_kv8_attn_workspace_bytes(1, 1, 32, 32, 1, 10 ** 6, 64, 4) < lib.smh_kv8_attn_workspace_bytes(1, 1, 32, 32, 1, 10 ** 6, 0, 0)
    assert lib.smh_beam_select_workspace_bytes(1, 4, 32016, 8) > 4 * 8 * 4
    for bad in ((0, 4, 100, 4), (1, 65, 100, 4), (1, 0, 100, 4), (1, 4, 100, 129), (1, 4, 3, 13), (1 << 20, 2, 100, 4)):
        assert lib.smh_beam_select_workspace_bytes(*bad) == 0


@pytest.mark.parametrize("bad,why", [(dict(W=65), b"beams"), (dict(W=0), b"beams"), (dict(n=0), b"n="), (dict(n=129), b"n="), (dict(n=100, W=2, vocab=49, ld=50), b"n="), (dict(G=0), b"G="),
                                     (dict(ld=40), b"ld="), (dict(eos=-1), b"eos"), (dict(eos=50), b"eos"), (dict(logits=None), b"null"), (dict(ws=None), b"workspace"),
                                     (dict(ws_bytes=8), b"workspace"), (dict(ws=(1 << 20) + 4), b"workspace"), (dict(W=64, vocab=1 << 24, ld=1 << 24), b"slices")], ids=str)
def test_c_select_refuses(bad, why):
    a = dict(logits=1 << 21, ld=50, scores=1 << 12, ended=None, G=2, W=3, vocab=50, n=4, eos=2, o0=1 << 13, o1=1 << 14, o2=1 << 15, o3=1 << 16, ws=1 << 20, ws_bytes=1 << 40, stream=None)
    a.update(bad)
    assert _lib.load().smh_beam_select(*a.values()) < 0 and why in err()


@pytest.mark.parametrize("bad,why", [(dict(W=65), b"W="), (dict(G=0), b"G="), (dict(G=65536), b"G="), (dict(n=17), b"at most 16"), (dict(parents=None), b"null"), (dict(bytes=[6, 8]), b"4 bytes"),
                                     (dict(strides=[4, 8]), b"rows of"), (dict(at=[(1 << 20) + 2, 1 << 21]), b"4 bytes"), (dict(at=[1 << 20, 1 << 20]), b"same"), (dict(units=[0, 4]), b"upto"),
                                     (dict(units=[0, 2], upto=1 << 12), b"4 bytes"), (dict(at=[None, 1 << 21]), b"rows of")], ids=str)
def test_c_reorder_refuses(bad, why):
    a = dict(parents=1 << 12, G=2, W=3, n=2, at=[1 << 20, 1 << 21], strides=[8, 8], bytes=[8, 8], units=[0, 0], upto=None)
    a.update(bad)
    a["at"] = (ctypes.c_void_p * 2)(*a["at"])
    a["strides"], a["bytes"] = (ctypes.c_long * 2)(*a["strides"]), (ctypes.c_long * 2)(*a["bytes"])
    a["units"] = (ctypes.c_int * 2)(*a["units"])
    assert _lib.load().smh_beam_reorder(*a.values(), None) < 0 and why in err()


def test_an_empty_cache():
    c = K.kv8_cache(2, 130, 3, "cpu")
    assert c.codes_k.shape == (6, 3, 64, 128) and c.codes_v.shape == (6, 3, 128, 64) and c.pages.tolist() == [[0, 1, 2], [3, 4, 5]]
    assert int(c.codes_k.min()) == 128 and float(c.scales.abs().max()) == 0
    assert K.kv8_cache(2, 64, 1, "cpu", n_pages=5).pages.tolist() == [[-1], [-1]]
    for bad in (dict(batch=0), dict(max_len=0), dict(n_kv_heads=0), dict(n_pages=0)):
        with pytest.raises(AssertionError):
            K.kv8_cache(**{**dict(batch=1, max_len=1, n_kv_heads=1, device="cpu"), **bad})


@pytest.mark.parametrize("max_new", [0, 2, 64])
def test_one_new_row_without_cu(max_new):
    assert c_append(max_new=max_new) == -1 and b"without cu" in err()
    assert c_attn(max_new=max_new) == -1 and b"without cu" in err()
