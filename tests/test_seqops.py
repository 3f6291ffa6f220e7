"""What the operators on callers' memory refuse, and how they plan their workspaces: no GPU needed, nothing is launched."""
import ctypes as C
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import seqops_plain as plain  # noqa: E402

from calm_b200 import seqops  # noqa: E402

L = None


@pytest.fixture(scope="module", autouse=True)
def library():
    global L
    L = seqops._load()


def says(rc, *words):
    text = L.calm_b200_seq_error().decode()
    assert rc == -3 and all(w in text for w in words), (rc, text)


def beam(**over):
    f = dict(logits=4096, type=0, group_stride=40, row_stride=10, scores=4096, groups=2, beams=4, vocab=10, n=3, tokens=4096, parents=4096, best=4096, workspace=4096, workspace_bytes=1 << 20)
    f.update(over)
    return L.calm_b200_seq_beam_select(C.byref(seqops._Beam(*[f[n] for n, _ in seqops._Beam._fields_])), None)


def test_beam_refusals():
    says(L.calm_b200_seq_beam_select(None, None), "no arguments")
    for over, word in ((dict(beams=0), "beams"), (dict(beams=65), "64"), (dict(groups=-1), "groups"), (dict(vocab=0), "tokens"), (dict(vocab=1 << 30), "2^27"), (dict(n=0), "n = 0"),
                       (dict(n=65), "n = 65"), (dict(groups=20000), "65535"), (dict(type=3), "type"), (dict(logits=None), "pointer"), (dict(scores=None), "pointer"), (dict(tokens=None), "pointer"),
                       (dict(parents=None), "pointer"), (dict(best=None), "pointer"), (dict(workspace=None), "pointer"), (dict(logits=4098), "aligned"), (dict(workspace=4104), "aligned"),
                       (dict(workspace_bytes=8), "are needed"), (dict(type=1, logits=4097), "aligned")):
        says(beam(**over), "beam", word)
    assert beam(groups=0) == 0
    assert L.calm_b200_seq_beam_workspace(2, 65, 10, 3) == 0
    for G, K, V, n in ((1, 1, 1, 1), (32, 8, 128256, 16), (1, 64, 1 << 20, 64), (65535, 1, 3, 1)):
        assert 0 < L.calm_b200_seq_beam_workspace(G, K, V, n) < 1 << 28


def copy(pools, pages=((), ()), rows=None, slots=((), ())):
    u = (seqops._Units * max(1, len(pools)))(*[seqops._Units(*p) for p in pools])
    a = [np.ascontiguousarray(x, np.int32) for x in (*pages, *slots)]
    r = None if rows is None else np.ascontiguousarray(rows, np.int32)
    return L.calm_b200_seq_copy_units(len(pools), u, len(a[0]), a[0].ctypes.data, a[1].ctypes.data, None if r is None else r.ctypes.data, len(a[2]), a[2].ctypes.data, a[3].ctypes.data, None)


def test_copy_refusals():
    page = (4096, 4096, 64, 8, 10, 10, 0)
    slot = (1 << 20, 1 << 20, 64, 0, 5, 5, 1)
    for args, word in (((([page]), ([0], [10])), "page 10"), ((([page]), ([-1], [0])), "page -1"), ((([page]), ([0, 1], [3, 3])), "twice"), ((([page]), ([0, 1], [1, 2])), "read and written"),
                       ((([page]), ([4], [4])), "read and written"), (([(4096, 4096, 64, 65, 10, 10, 0)], ([0], [1])), "rows"), (([(None, None, 64, 8, 10, 10, 0)], ([0], [1])), "memory"),
                       (([(4096, 4096 + 64, 64, 8, 10, 10, 0)], ([0], [1])), "overlap"), (([(4096, 4096, 64, 8, 10, 10, 2)], ([0], [1])), "kind"), (([(4096, 4096, -1, 0, 10, 10, 0)], ([0], [1])), "negative"),
                       (([(4096, 4096, 1 << 40, 0, 10, 10, 0)], ([0], [1])), "256 GB"), (([page, (4096, 1 << 22, 64, 8, 10, 3, 0)], ([0], [3])), "pool of 3")):
        says(copy(*args), "copy", word)
    says(copy([page], ([0], [1]), rows=[-1]), "rows")
    says(copy([slot], slots=([0], [5])), "slot 5")
    assert copy([page, slot]) == 0 and copy([]) == 0  # nothing to copy


def cache8(**over):
    f = dict(k=4096, k_scale=4096, v=4096, v_scale=4096, pages=10, heads=2, page=16, dim=64, table=4096, slots=3, table_pages=4)
    f.update(over)
    return seqops._Cache8(*[f[n] for n, _ in seqops._Cache8._fields_])


def portions(**over):
    f = dict(n=2, start=4096, count=4096, slot=4096, pos0=4096, longest=5)
    f.update(over)
    return seqops._Portions(*[f[n] for n, _ in seqops._Portions._fields_])


def rows(**over):
    f = dict(p=4096, type=0, row_stride=128, head_stride=64, rows=10)
    f.update(over)
    return seqops._Rows(*[f[n] for n, _ in seqops._Rows._fields_])


def attend(c=None, p=None, **over):
    f = dict(q=rows(), out=rows(), heads=4, scale=1.0, window=0, keep_first=0, chunk=0, softcap=0.0, sinks=None, slopes=None, gate=None, gate_row=0, gate_head=0, gate_dim=0, most_keys=100,
             workspace=None, workspace_bytes=0)
    f.update(over)
    a = seqops._Attend8(*[f[n] for n, _ in seqops._Attend8._fields_])
    return C.byref(c or cache8()), C.byref(p or portions()), C.byref(a)


BAD_CACHES = ((dict(dim=0), "channels"), (dict(dim=24), "channels"), (dict(dim=272), "channels"), (dict(heads=0), "heads"), (dict(heads=5000), "heads"), (dict(page=0), "page"), (dict(page=1 << 20), "page"),
              (dict(pages=-1), "pages"), (dict(k=None), "memory"), (dict(v_scale=None), "memory"), (dict(table=None), "table"), (dict(k=4104), "aligned"), (dict(k_scale=4097), "aligned"))
BAD_BATCHES = ((dict(n=-1), "sequences"), (dict(n=70000), "sequences"), (dict(longest=-1), "longest"), (dict(start=None), "description"), (dict(pos0=None), "description"))


def test_store_refusals():
    def store(c=None, p=None, k=None, v=None):
        return L.calm_b200_seq_cache8_store(C.byref(c or cache8()), C.byref(p or portions()), C.byref(k or rows()), C.byref(v or rows()), None)

    for over, word in BAD_CACHES:
        says(store(c=cache8(**over)), "store8", word)
    for over, word in BAD_BATCHES:
        says(store(p=portions(**over)), "store8", word)
    for over, word in ((dict(type=7), "type"), (dict(p=None), "missing"), (dict(rows=-2), "missing"), (dict(p=4098), "aligned"), (dict(type=1), "values")):
        says(store(k=rows(**over)), "store8", word)
    says(L.calm_b200_seq_cache8_store(None, None, None, None, None), "no cache")
    assert store(p=portions(n=0, start=None)) == 0 and store(p=portions(longest=0)) == 0


def test_attend_refusals_and_workspace():
    for over, word in BAD_CACHES:
        says(L.calm_b200_seq_attend8(*attend(c=cache8(**over)), None), "attend8", word)
    for over, word in BAD_BATCHES:
        says(L.calm_b200_seq_attend8(*attend(p=portions(**over)), None), "attend8", word)
    for over, word in ((dict(heads=3), "query heads"), (dict(heads=0), "query heads"), (dict(q=rows(type=4)), "type"), (dict(out=rows(type=2)), "type"), (dict(q=rows(type=1), out=rows(type=0)), "type"),
                       (dict(out=rows(rows=9)), "rows"), (dict(window=-1), "range"), (dict(keep_first=-1), "range"), (dict(chunk=-3), "range"), (dict(softcap=-1.0), "range"),
                       (dict(softcap=float("nan")), "range"), (dict(scale=float("nan")), "range"), (dict(q=rows(p=None)), "missing")):
        says(L.calm_b200_seq_attend8(*attend(**over), None), "attend8", word)
    few, many = portions(n=1, longest=1), portions(n=150, longest=1)
    assert L.calm_b200_seq_attend8_workspace(*attend(p=few, most_keys=100000)) == 0  # clusters fold their shares themselves
    need = L.calm_b200_seq_attend8_workspace(*attend(p=many, most_keys=100000))
    assert need > 0
    says(L.calm_b200_seq_attend8(*attend(p=many, most_keys=100000), None), "workspace")
    says(L.calm_b200_seq_attend8(*attend(p=many, most_keys=100000, workspace=4096, workspace_bytes=need - 1), None), "workspace")
    says(L.calm_b200_seq_attend8(*attend(p=many, most_keys=100000, workspace=4100, workspace_bytes=need), None), "workspace")
    assert L.calm_b200_seq_attend8_workspace(*attend(p=portions(n=4000, longest=1))) == 0
    assert L.calm_b200_seq_attend8(*attend(p=portions(n=0, start=None)), None) == 0


def test_python_refusals():
    x, s = torch.zeros(1, 2, 8), torch.zeros(1, 2)
    with pytest.raises(ValueError, match="CUDA"):
        seqops.beam_select(x, s, 2)
    with pytest.raises(ValueError, match="CUDA"):
        seqops.UnitPool([torch.zeros(2, 2, 2)])
    with pytest.raises(ValueError, match="CUDA"):
        seqops.Cache8(*[torch.zeros(1)] * 4)
    for args in (([0, 0], [1, 1], [0, 0]), ([0], [1, 1], [0]), ([0], [-1], [0]), ([-1], [1], [0]), ([0], [1], [-1]), ([0], [1], [2 ** 31 - 1])):
        with pytest.raises(ValueError):
            seqops.Batch(*args, device="cpu")
    seqops.UnitPool().copy()


def test_the_plain_rounding_is_torchs():
    """The statement that the GPU tests compare with, against the conversions of another implementation."""
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.normal(0, 40, 20000), rng.normal(0, 0.02, 20000), plain.VALUES[:127] * 1.03125, plain.VALUES[:126] + np.diff(plain.VALUES[:127]) / 2]).clip(-448, 448).astype(np.float32)
    t = torch.tensor(x).to(torch.float8_e4m3fn)
    assert np.array_equal(plain.round_e4m3(x), t.float().double().numpy()) and np.array_equal(plain.VALUES[t.view(torch.uint8).numpy()], t.float().double().numpy())
    for a in (0.0, 1.0, 448.0, 448.1, 449.0, 3e38, 1e-30, 2.0 ** -60):
        e = plain.exponent(a)
        assert a <= 448 * 2.0 ** e and (e == -64 or a > 448 * 2.0 ** (e - 1))


def test_a_batch_without_groups():
    """Nothing to select, nothing to hold; what is refused with groups is refused without."""
    for beams in (1, 4, 64):
        assert L.calm_b200_seq_beam_workspace(0, beams, 100, 3) == 0 and beam(groups=0, beams=beams) == 0
    says(beam(groups=0, beams=65), "beam", "64")


def test_a_slice_that_gives_up_waits_for_every_copy_that_it_asked_for():
    """k_beam_slice: a warp that gives up on a tile has the copies of that tile and of the stages behind it in flight, into memory that the block uses for other things next."""
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "calm_b200", "csrc", "seqbeam.cu")).read()
    drain = src[src.index("void beam_drain("):]
    drain = drain[:drain.index("\n}\n")]
    assert "for (int k = 0; k < STAGES && at < end; ++k, at += step) {\n\t\tmbar_wait_warp(full + stage, parity);\n\t\tif (++stage == STAGES) stage = 0, parity ^= 1;" in drain
    loop = src[src.index("bool lost = false;"):]
    loop = loop[:loop.index("\n\t}\n")]
    gave_up = loop.index("if (!mbar_wait_warp(full + stage, parity)) lost = true, beam_drain<STAGES>(full, stage, parity, v0 + warp * WSTEP, end, STEP);")
    assert gave_up < loop.index("if (lane == 0 && !lost) request(stage);") and "&& !lost)" in loop[:gave_up]
    # the loop's requests and the drain's waits, tile by tile
    for stages in (2, 4):
        for tiles in range(1, 12):
            for lost in range(tiles):
                asked, done = set(range(min(stages, tiles))), set()
                for i in range(lost):
                    done.add(i)
                    if i + stages < tiles:
                        asked.add(i + stages)
                stage, parity, waited = lost % stages, lost // stages & 1, set()
                for k in range(stages):
                    if lost + k >= tiles:
                        break
                    t = lost + k
                    assert (stage, parity) == (t % stages, t // stages & 1)
                    waited.add(t)
                    stage += 1
                    if stage == stages:
                        stage, parity = 0, parity ^ 1
                assert waited == asked - done


def test_a_fork_into_fewer_than_no_sequences_is_refused():
    """It would be a branch without children, which closes the sequence."""
    from calm_b200 import seqlib

    asked = []

    class Model(seqlib.SeqDeviceModel):
        def __init__(self):
            pass

        def branch(self, slots, parents):
            asked.append((list(slots), list(parents)))
            return list(range(len(parents)))

        def __del__(self):
            pass

    m = Model()
    assert m.fork(3, 0) == [] and m.fork(3, 2) == [1, 2] and asked == [([3], [0]), ([3], [0, 0, 0])]
    for n in (-1, -2, -100):
        with pytest.raises(seqlib.SeqError, match="bad branch"):
            m.fork(3, n)
    assert len(asked) == 2


def test_numbers_past_32_bits_are_refused_and_not_cut_off():
    from calm_b200 import seqlib

    for v in (2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1, 10 ** 30, 1.5, "3", None):
        with pytest.raises(ValueError, match="window"):
            seqops._whole("window", v)
    assert [seqops._whole("n", v) for v in (0, -1, 2 ** 31 - 1, np.int64(7), True)] == [0, -1, 2 ** 31 - 1, 7, 1]

    class Library:  # the library as it would answer what it is asked
        def __getattr__(self, name):
            return lambda *a: asked.append((name, a)) or 0

    asked, m = [], seqlib.SeqDeviceModel.__new__(seqlib.SeqDeviceModel)
    m.lib, m.handle, m.desc = Library(), None, type("D", (), {})()
    for call in (lambda: m.resize(2 ** 32 + 100), lambda: m.branch([2 ** 32], [0]), lambda: m.branch(np.array([2 ** 32 + 1]), [0]), lambda: m.branch([0], np.array([-2 ** 32])),
                 lambda: m.beams(np.zeros((1, 1), np.float32), 3, row0=2 ** 32), lambda: m.beams(np.zeros((1, 1), np.float32), 2 ** 32 + 1)):
        with pytest.raises(seqlib.SeqError):
            call()
    assert not asked
    m.resize(100), m.branch(np.array([1, 0]), [1, 1]), m.beams(np.zeros((1, 1), np.float32), 3, row0=1)
    assert [a[0] for a in asked] == ["calm_b200_seq_resize", "calm_b200_seq_branch", "calm_b200_seq_beams"]
    m.close = lambda: None


def test_pointers_that_a_kernel_could_not_read_through_are_refused():
    """Four bytes at an odd address are a fault on the device."""
    for name in ("scores", "tokens", "parents", "best"):
        says(beam(**{name: 4098}), "beam", "aligned")
    store = lambda c, p: L.calm_b200_seq_cache8_store(C.byref(c), C.byref(p), C.byref(rows()), C.byref(rows()), None)
    for c, p in [(cache8(table=4097), portions())] + [(cache8(), portions(**{name: 4098})) for name in ("start", "count", "slot", "pos0")]:
        says(store(c, p), "store8", "aligned")
        says(L.calm_b200_seq_attend8(*attend(c=c, p=p), None), "attend8", "aligned")
    for name in ("sinks", "slopes", "gate"):
        says(L.calm_b200_seq_attend8(*attend(**{name: 4099}), None), "attend8", "aligned")


def test_pools_that_overlap_are_found_whatever_their_size():
    for unit, n in ((1 << 38, 1 << 26), (1 << 38, (1 << 26) + 1), (1 << 36, 1 << 27), (1 << 38, 2 ** 31 - 1)):
        says(copy([(4096, 4096 + 64, unit, 0, n, n, 0)], ([0], [1])), "copy", "overlap")
        says(copy([(4096 + 64, 4096, unit, 0, n, n, 1)], slots=([0], [1])), "copy", "overlap")


def test_more_pairs_of_token_and_head_than_are_counted_are_refused():
    """Rows of a sequence are numbered in 31 bits: 2^30 tokens of 36 heads came out as a grid of an eighth of them."""
    for longest, heads in ((1 << 30, 72), (2 ** 31 - 1, 4), (1 << 26, 64)):
        a = attend(p=portions(longest=longest), heads=heads)
        says(L.calm_b200_seq_attend8(*a, None), "attend8", "pairs")
        assert L.calm_b200_seq_attend8_workspace(*a) == 0
    for longest, heads in ((1 << 29, 4), (2 ** 31 - 300, 2)):
        assert L.calm_b200_seq_attend8(*attend(p=portions(longest=longest, n=0, start=None), heads=heads), None) == 0
