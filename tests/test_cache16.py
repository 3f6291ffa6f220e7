"""What rotary positions, the 16-bit cache and attention over shared prefixes refuse, how they describe groups and frequencies, and how they plan their workspaces: no GPU needed, nothing is launched."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from calm_b200 import seqops

L = None


@pytest.fixture(scope="module", autouse=True)
def library():
    global L
    L = seqops._load()


def says(rc, *words):
    text = L.calm_b200_seq_error().decode()
    assert rc == -3 and all(w in text for w in words), (rc, text)


def made(struct, f, over):
    f.update(over)
    return struct(*[f[n] for n, _ in struct._fields_])


def cache(**over):
    return made(seqops._Cache16, dict(k=4096, v=4096, type=1, pages=10, heads=2, page=16, dim=64, table=4096, slots=3, table_pages=4), over)


def portions(**over):
    return made(seqops._Portions, dict(n=2, start=4096, count=4096, slot=4096, pos0=4096, longest=5), over)


def rows(**over):
    return made(seqops._Rows, dict(p=4096, type=1, row_stride=128, head_stride=64, rows=10), over)


def rotation(**over):
    return made(seqops._Rotation, dict(turns=4096, dims=32, neighbours=0, gain=1.0), over)


def shared(**over):
    return made(seqops._Shared, dict(n=1, first=4096, count=4096, positions=4096, group=4096, n_alone=0, alone=None, longest=100, tokens=10, most_own=20, most_alone=0, lengths=None), over)


def ref(x):
    return None if x is None else C.byref(x)


def attend(c=None, p=None, s=None, stream=False, **over):
    a = made(seqops._Attend16, dict(q=rows(), out=rows(), heads=4, scale=1.0, window=0, softcap=0.0, sinks=None, most_keys=100, row_tiles=0, workspace=None, workspace_bytes=0, few=0), over)
    return ref(c or cache()), ref(p or portions()), ref(s), ref(a)


BAD_CACHES = ((dict(dim=0), "channels"), (dict(dim=24), "channels"), (dict(dim=272), "channels"), (dict(heads=0), "heads"), (dict(heads=5000), "heads"), (dict(page=0), "page"), (dict(page=1 << 20), "page"),
              (dict(pages=-1), "pages"), (dict(pages=1 << 27), "2^31"), (dict(k=None), "memory"), (dict(v=None), "memory"), (dict(table=None), "table"), (dict(k=4104), "aligned"), (dict(table=4098), "aligned"),
              (dict(type=0), "type"), (dict(type=3), "type"))
BAD_BATCHES = ((dict(n=-1), "sequences"), (dict(n=70000), "sequences"), (dict(longest=-1), "longest"), (dict(start=None), "description"), (dict(pos0=None), "description"), (dict(count=4098), "aligned"))
BAD_ROTATIONS = ((dict(dims=0), "channels"), (dict(dims=33), "channels"), (dict(dims=66), "channels"), (dict(turns=None), "frequencies"), (dict(turns=4100), "aligned"))


def test_rotate_refusals():
    def rotate(p=None, r=None, x=None, out=None, heads=2, dim=64):
        return L.calm_b200_seq_rotate(ref(p or portions()), ref(r or rotation()), ref(x or rows()), ref(out or rows()), heads, dim, None)

    for over, word in BAD_BATCHES:
        says(rotate(p=portions(**over)), "rotate", word)
    for over, word in BAD_ROTATIONS:
        says(rotate(r=rotation(**over)), "rotate", word)
    for over, word in ((dict(type=7), "type"), (dict(p=None), "missing"), (dict(rows=-2), "missing"), (dict(p=4097), "aligned"), (dict(type=2), "type")):
        says(rotate(x=rows(**over)), "rotate", word)
    for heads, dim in ((0, 64), (70000, 64), (2, 0), (2, 63), (2, 1026)):
        says(rotate(heads=heads, dim=dim), "rotate", "heads of")
    says(L.calm_b200_seq_rotate(None, None, None, None, 1, 2, None), "no batch")
    says(L.calm_b200_seq_rotate(ref(portions()), None, ref(rows()), ref(rows()), 2, 64, None), "no rotation")
    assert rotate(p=portions(n=0, start=None)) == 0 and rotate(p=portions(longest=0)) == 0


def test_store_refusals():
    def store(c=None, p=None, k=None, v=None, r=None, q=None, q_out=None, heads=0):
        return L.calm_b200_seq_cache16_store(ref(c or cache()), ref(p or portions()), ref(k or rows()), ref(v or rows()), ref(r), ref(q), ref(q_out), heads, None)

    for over, word in BAD_CACHES:
        says(store(c=cache(**over)), "store16", word)
    for over, word in BAD_BATCHES:
        says(store(p=portions(**over)), "store16", word)
    for over, word in BAD_ROTATIONS:
        says(store(r=rotation(**over)), "store16", word)
    for over, word in ((dict(type=7), "type"), (dict(p=None), "missing"), (dict(rows=-2), "missing"), (dict(p=4097), "aligned"), (dict(type=0), "values")):
        says(store(k=rows(**over)), "store16", word)
    says(store(q=rows(), q_out=rows(), heads=4), "rotation")
    says(store(q=rows(), r=rotation(), heads=4), "place to go")
    says(store(q=rows(), q_out=rows(type=0), r=rotation(), heads=4), "types")
    says(store(q=rows(type=2), q_out=rows(type=2), r=rotation(), heads=4), "types")
    says(store(q=rows(), q_out=rows(), r=rotation(), heads=0), "query heads")
    says(L.calm_b200_seq_cache16_store(None, None, None, None, None, None, None, 0, None), "no cache")
    assert store(p=portions(n=0, start=None)) == 0 and store(p=portions(longest=0)) == 0


def test_attend_refusals_and_workspace():
    for over, word in BAD_CACHES:
        says(L.calm_b200_seq_attend16(*attend(c=cache(**over)), None), "attend16", word)
    for over, word in BAD_BATCHES:
        says(L.calm_b200_seq_attend16(*attend(p=portions(**over)), None), "attend16", word)
    for over, word in ((dict(n=-1), "groups"), (dict(n=3), "groups"), (dict(longest=-1), "groups"), (dict(tokens=-1), "groups"), (dict(most_own=-1), "groups"), (dict(most_alone=-1), "groups"), (dict(first=None), "groups"), (dict(group=None), "groups"), (dict(n_alone=-1), "no group"), (dict(n_alone=3), "no group"), (dict(n_alone=1), "no group"), (dict(n_alone=1, alone=4098), "aligned"),
                       (dict(positions=4098), "aligned")):
        says(L.calm_b200_seq_attend16(*attend(s=shared(**over)), None), "attend16", word)
    for over, word in ((dict(heads=3), "query heads"), (dict(heads=0), "query heads"), (dict(q=rows(type=4)), "type"), (dict(out=rows(type=2)), "type"), (dict(q=rows(type=0), out=rows(type=0)), "type"),
                       (dict(out=rows(rows=9)), "rows"), (dict(window=-1), "range"), (dict(softcap=-1.0), "range"), (dict(softcap=float("nan")), "range"), (dict(softcap=math.inf), "range"), (dict(scale=float("nan")), "range"),
                       (dict(q=rows(p=None)), "missing"), (dict(sinks=4098), "aligned"), (dict(row_tiles=-1), "row tiles"), (dict(few=-1), "few rows")):
        says(L.calm_b200_seq_attend16(*attend(**over), None), "attend16", word)
    for longest, heads in ((1 << 30, 72), (2 ** 31 - 1, 4)):
        says(L.calm_b200_seq_attend16(*attend(p=portions(longest=longest), heads=heads), None), "attend16", "pairs")
        says(L.calm_b200_seq_attend16(*attend(s=shared(tokens=longest), heads=heads), None), "attend16", "pairs")
    says(L.calm_b200_seq_attend16(*attend(p=portions(n=65535), s=shared(n=1)), None), "attend16", "65535")
    assert L.calm_b200_seq_attend16(*attend(p=portions(n=0, start=None)), None) == 0
    a = dict(p=portions(n=150, longest=1), heads=4, q=rows(rows=150), out=rows(rows=150), most_keys=100000)
    need = L.calm_b200_seq_attend16_workspace(*attend(**a))
    assert 0 < need < 1 << 30
    says(L.calm_b200_seq_attend16(*attend(**a), None), "workspace")
    says(L.calm_b200_seq_attend16(*attend(**a, workspace=4096, workspace_bytes=need - 1), None), "workspace")
    says(L.calm_b200_seq_attend16(*attend(**a, workspace=4100, workspace_bytes=need), None), "workspace")


@pytest.mark.parametrize("over", [dict(scale=math.inf), dict(scale=-math.inf), dict(scale=1.0, softcap=1e-44)])
def test_attend_refuses_scores_that_no_number_holds(over):
    says(L.calm_b200_seq_attend16(*attend(**over), None), "attend16", "range")


def test_the_way_follows_sizes_types_and_pages():
    """Shapes that were measured in all their ways (the rule stands at a16_plan), and what the tensor-memory kernel does not serve."""
    def way(n, longest, heads, kv, dim, page, groups=0, positions=0, own=50, keys=4000, **over):
        s = shared(n=groups, longest=positions, tokens=n * longest // max(groups, 1), most_own=own) if groups else None
        big = rows(rows=n * longest, row_stride=heads * dim, head_stride=dim)
        return L.calm_b200_seq_attend16_way(*attend(c=cache(heads=kv, dim=dim, page=page, pages=5000), p=portions(n=n, longest=longest), s=s, heads=heads, q=big, out=big, most_keys=keys, **over))

    assert way(1, 1, 32, 8, 128, 16) == 4 and way(4, 1, 32, 8, 128, 16, 1, 3000) == 4            # a user's tokens, four beams: clusters
    assert way(1, 1, 32, 8, 128, 16, keys=16000) == 8 and way(150, 1, 32, 8, 128, 16, keys=900) == 0  # shares through memory; none
    assert way(64, 1, 32, 8, 128, 16, 1, 16000, 1000) == 1 and way(64, 1, 32, 8, 128, 16, 1, 600) & 3 == 0
    assert way(16, 300, 32, 8, 128, 16, 1, 12000, 300, keys=12300) & 3 in (1, 2) and way(2, 900, 32, 8, 128, 16, keys=900) & 3 == 2
    for dim, page in ((128, 12), (256, 16), (48, 16)):
        assert way(64, 1, 32, 8, dim, page, 1, 16000, 1000) & 3 == 0 and way(2, 900, 32, 8, dim, page, keys=900) & 3 == 0
    for dim in (64, 80, 96, 112, 128):
        assert way(2, 900, 32, 8, dim, 24, keys=900) & 3 == 2
    assert way(3, 1, 3, 2, 64, 16) == -3


def test_batches_of_groups():
    def batch(shared, counts=(1, 2, 3, 1), before=(9, 9, 12, 4)):
        return seqops.Batch(range(len(counts)), counts, before, device="cpu", shared=shared)

    for bad in ([(0, 2, 10)], [(0, 0, 1)], [(-1, 2, 1)], [(3, 2, 1)], [(0, 2, -1)], [(0, 2, 5), (1, 2, 5)], [(0, 2)], [5], [(0, 1.5, 2)], [(0, 1, 2 ** 31)], [(0, 1, 2), (1, 1)]):
        with pytest.raises(ValueError, match="group"):
            batch(bad)
    with pytest.raises(ValueError, match="CUDA"):
        batch([(0, 2, 9)])


def test_python_refusals():
    x = torch.zeros(2, 2, 32)
    with pytest.raises(ValueError, match="CUDA"):
        seqops.rotate(x, None, None)
    with pytest.raises(ValueError, match="CUDA"):
        seqops.Cache16(torch.zeros(1), torch.zeros(1))
    for args, words in (((0,), "channels"), ((7,), "channels"), ((1.5,), "whole number")):
        with pytest.raises(ValueError, match=words):
            seqops.Rotation(*args, device="cpu")
    for kw in (dict(pairs="x"), dict(base=0.0), dict(base=math.inf), dict(scaling={"kind": "linear"}), dict(scaling={"kind": "linear", "factor": -1.0}), dict(scaling={"kind": "else", "factor": 1.0}),
               dict(scaling={"kind": "linear", "factor": 2.0, "length": 5}), dict(scaling={"kind": "wavelength", "factor": 2.0, "length": 5, "low": 3.0, "high": 1.0}), dict(frequencies=[1.0]),
               dict(frequencies=[1.0, math.nan, 1.0, 1.0]), dict(frequencies=[1.0] * 4, scaling={"kind": "linear", "factor": 2.0}), dict(base=1.0, scaling={"kind": "ramp", "factor": 2.0, "length": 64, "fast": 32.0, "slow": 1.0})):
        with pytest.raises(ValueError):
            seqops.Rotation(8, device="cpu", **kw)
    with pytest.raises(ValueError, match="stretch"):
        seqops.Rotation(2, scaling={"kind": "base", "factor": 2.0}, device="cpu")


def test_frequencies():
    f, gain = seqops.rotation_frequencies(64, 500000.0)
    assert gain == 1.0 and np.allclose(f, [500000.0 ** (-2 * i / 64) for i in range(32)], rtol=1e-15)
    assert np.allclose(seqops.rotation_frequencies(64, 1e4, {"kind": "linear", "factor": 4.0})[0], seqops.rotation_frequencies(64)[0] / 4, rtol=1e-15)
    # a stretched base leaves the fastest pair and divides the slowest by the factor
    f, g = seqops.rotation_frequencies(64), seqops.rotation_frequencies(64, 1e4, {"kind": "base", "factor": 8.0})
    assert g[0][0] == 1.0 and math.isclose(f[0][-1] / g[0][-1], 8.0, rel_tol=1e-12)
    # by wavelength: short waves stay, long ones are divided, between the two a blend that rises
    f, g = seqops.rotation_frequencies(128, 500000.0)[0], seqops.rotation_frequencies(128, 500000.0, {"kind": "wavelength", "factor": 8.0, "length": 8192, "low": 1.0, "high": 4.0})[0]
    w = 8192 * f / (2 * math.pi)
    assert np.array_equal(g[w > 4], f[w > 4]) and np.allclose(g[w < 1], f[w < 1] / 8, rtol=1e-15) and (np.diff(g / f) <= 1e-15).all() and ((w > 1) & (w < 4)).any()
    # by the pair's number
    g, gain = seqops.rotation_frequencies(128, 1e4, {"kind": "ramp", "factor": 16.0, "length": 4096, "fast": 32.0, "slow": 1.0})
    f = seqops.rotation_frequencies(128)[0]
    assert math.isclose(gain, 0.1 * math.log(16) + 1) and g[0] == f[0] and math.isclose(g[-1], f[-1] / 16, rel_tol=1e-12)
    turns = 4096 * f / (2 * math.pi)
    assert np.array_equal(g[turns > 40], f[turns > 40]) and np.allclose(g[turns < 0.8], f[turns < 0.8] / 16, rtol=1e-12)
    assert seqops.rotation_frequencies(8, 1e4, {"kind": "ramp", "factor": 2.0, "length": 64, "fast": 32.0, "slow": 1.0, "gain": 1.5})[1] == 1.5
