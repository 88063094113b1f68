"""Calls of the head norms with the append, the 8-bit caches and the draft trees that a C caller, or a program with
unusual arguments, may make: what each reads and gives, and what is refused."""

import ctypes
import shutil
import struct

import pytest
import torch

from transformer_optimization_amd import _C
from test_cache8_tree_ops import DTYPES, _Abi, _values
from test_limits import _run_check
from test_seq_ops import E, FAKE, U, _cu, _gen, _i32, _randn

gpu = pytest.mark.gpu


def _append_c(q, k, steps, cu, positions, positions_ld, axes, pair_axis):
    """q and k turned by the C entry point itself, norm "rms", no cache."""
    (t, h, hd), hk = q.shape, k.shape[1]
    lib = _C.load_library()
    out = torch.full_like(q, float("nan")), torch.full_like(k, float("nan"))
    st = {n: (ctypes.c_int64 * 3)(n * hd, hd, 1) for n in (h, hk)}
    ptr = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    at = {n: ctypes.addressof(s) for n, s in st.items()}
    code = lib.tx_norm_rotary_append(
        q.data_ptr(), at[h], out[0].data_ptr(), at[h], k.data_ptr(), at[hk], out[1].data_ptr(), at[hk], None, None, None,
        None, None, None, None, None, None, None, None, None, None, None, 0, _C.TX_F32, _C.TX_NORM_RMS, 1e-6,
        steps.data_ptr(), ptr(pair_axis), ptr(positions), positions_ld, axes, cu.data_ptr(), None, None, 0, t,
        cu.numel() - 1, h, hk, hd, 2 * steps.numel(), 0, 0, 0, 1.0, 0, _C._DT[q.dtype],
        torch.cuda.current_stream().cuda_stream)
    return code, out


def _turn_inputs(cuda, lens=(5, 1, 14)):
    t = sum(lens)
    q, k = _randn((t, 4, 64), torch.bfloat16, cuda, 1), _randn((t, 2, 64), torch.bfloat16, cuda, 2)
    steps, _ = _C.rotary_steps(64, 10000.0, device=cuda)
    positions = torch.stack([torch.arange(t) + 3, 7 * torch.arange(t), torch.arange(t) % 4]).to(cuda)
    return q, k, steps, _cu(lens, cuda), positions


@gpu
def test_without_pair_axis_every_pair_goes_by_axis_0(cuda):
    q, k, steps, cu, positions = _turn_inputs(cuda)
    t = q.shape[0]
    zeros = torch.zeros(32, dtype=torch.int32, device=cuda)
    code, want = _append_c(q, k, steps, cu, positions, t, 3, zeros)
    assert code == 0
    code, got = _append_c(q, k, steps, cu, positions, t, 3, None)
    assert code == 0
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all()


@gpu
def test_without_positions_there_is_one_axis(cuda):
    q, k, steps, cu, _ = _turn_inputs(cuda)
    axis = (torch.arange(32, dtype=torch.int32) % 3).to(cuda)
    code, want = _append_c(q, k, steps, cu, None, 0, 1, None)
    assert code == 0
    for pair_axis in (axis, None):
        code, got = _append_c(q, k, steps, cu, None, 0, 3, pair_axis)
        assert code == 0
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# The call with one row of positions for all axes goes on to a later refusal (steps that are not aligned).
@pytest.mark.parametrize("change,code", [(dict(pld=0), U), (dict(pld=64), U), (dict(pld=63), E), (dict(pld=1), E),
                                         (dict(pld=-1), E), (dict(pld=0, t=1), U)])
def test_rows_of_positions_are_apart_or_one(change, code):
    call = dict(axes=3, pos=1 << 39, axis=1 << 40, steps=FAKE + 4, ld=8)
    assert _Abi().append(**call, **change) == code


def test_the_wrapper_names_rows_of_positions_that_overlap():
    q = torch.zeros(6, 4, 64, dtype=torch.bfloat16)
    args = q, q, None, torch.zeros(32, dtype=torch.int64), _cu((6,), "cpu")
    axis = torch.zeros(32, dtype=torch.int32)
    some = torch.zeros(20, dtype=torch.int64)
    with pytest.raises(ValueError, match="rows of positions"):
        _C.norm_rotary_append(*args, positions=some.as_strided((3, 6), (5, 1)), pair_axis=axis)
    for positions in (some[:6].expand(3, 6), some[:18].view(3, 6), some.as_strided((1, 6), (5, 1))):
        with pytest.raises(ValueError, match="GPU tensors"):
            _C.norm_rotary_append(*args, positions=positions, pair_axis=axis)


@gpu
@pytest.mark.parametrize("lens", [(5, 1, 14), (1,)])
def test_one_row_of_positions_for_all_axes(cuda, lens):
    q, k, steps, cu, positions = _turn_inputs(cuda, lens)
    axis = (torch.arange(32, dtype=torch.int32) % 3).to(cuda)
    rows = positions[0].expand(3, q.shape[0])
    got = _C.norm_rotary_append(q, k, None, steps, cu, positions=rows, pair_axis=axis)
    want = _C.norm_rotary_append(q, k, None, steps, cu, positions=rows.contiguous(), pair_axis=axis)
    one = _C.norm_rotary_append(q, k, None, steps, cu, positions=positions[0])
    for g, w, o in zip(got, want, one):
        assert torch.equal(g, w) and torch.equal(g, o)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("h", [2, 24])  # few rows, tiles
def test_scales_that_the_append_of_the_type_does_not_write(cuda, dtype, hd, h):
    """Every scale byte, as another type's append or another program may have written it.  A row that sees one key gives
    its value, rounded once to the type: to subnormal steps at its lower end (of bf16, whose products may take them for
    0: within the smallest normal value), infinite beyond its upper one."""
    batch = 256
    codes = torch.randint(0, 127, (batch, 1, 8, hd), generator=_gen(70), dtype=torch.uint8)
    codes |= (torch.randint(0, 2, codes.shape, generator=_gen(71)) * 128).to(torch.uint8)
    scales = torch.full((batch, 1, 8, hd // 32), 127, dtype=torch.uint8)
    scales[..., 0] = torch.arange(batch)[:, None, None].to(torch.uint8)
    keys = torch.zeros_like(codes)
    q = _randn((batch, h, hd), dtype, cuda, 72)
    got = _C.flash_attn_paged_mx8(q, keys.to(cuda).view(torch.float8_e4m3fn), torch.full_like(scales, 127).to(cuda),
                                  codes.to(cuda).view(torch.float8_e4m3fn), scales.to(cuda),
                                  torch.arange(batch, dtype=torch.int32, device=cuda)[:, None],
                                  torch.arange(batch + 1, dtype=torch.int32, device=cuda), _i32([1] * batch, cuda), 0.125)
    value = _values(codes, scales)[:, :, 0]
    want = value.to(dtype).double().expand(batch, h, hd)
    nan = torch.isnan(want)
    assert bool(torch.isnan(got.cpu()[nan]).all()) and int(nan.sum()) == h * 32
    off = (got.cpu().double() - want)[~nan & torch.isfinite(want)].abs().max()
    assert float(off) <= (2.0**-126 if dtype == torch.bfloat16 else 0.0)
    assert torch.equal(got.cpu().double()[torch.isinf(want)], want[torch.isinf(want)])


@gpu
@pytest.mark.parametrize("tree", [False, True])
def test_a_bound_in_a_tensor_that_changes(cuda, tree):
    """max_q_len may be any whole number, also one that the caller writes again between calls."""
    t, hd = 64, 64
    q = _randn((t, 8, hd), torch.bfloat16, cuda, 73)
    (kc, ks), (vc, vs) = (_C.mx8_cache(64, 2, 16, hd, device=cuda) for _ in "kv")
    seqs = torch.arange(64, dtype=torch.int32, device=cuda)[None], _cu((t,), cuda), _i32([1000], cuda)
    mask = torch.full((t, 1), -1, dtype=torch.int64, device=cuda)
    kc.view(torch.uint8).random_(0, 127)
    vc.view(torch.uint8).random_(0, 127)

    def call(bound):
        if tree:
            return _C.flash_attn_tree(q, kc, vc, *seqs, mask, 0.125, k_scales=ks, v_scales=vs, max_q_len=bound)
        return _C.flash_attn_paged_mx8(q, kc, ks, vc, vs, *seqs, 0.125, max_q_len=bound)

    bound = torch.tensor(1)
    for n in (1, 8, 64, 1):
        assert torch.equal(call(bound.fill_(n)), call(n)), n
    with pytest.raises(TypeError):
        call(2.5)


def test_views_that_alternate_within_a_page_are_refused():
    """Keys and values in turn, slot by slot: no memory is shared, but only pages and rows are told apart."""
    st = dict(kcs=(4096, 128, 256), vcs=(4096, 128, 256))
    for call in (_Abi().append, _Abi().accept):
        assert call(kc=1 << 33, vc=(1 << 33) + 64 * 2, **st) == E


def test_spans_of_far_rows_are_not_lost():
    """Strides whose spans pass 63 bits: memory that is two arguments' at once is still seen."""
    far = dict(t=1 << 22, mld=1 << 40, mask=1 << 50)
    assert _Abi().paged(tree=True, o=1 << 50, **far) == E
    assert _Abi().paged(tree=True, o=(1 << 50) + (1 << 43) * 5, **far) == E
    # rows of the output far apart, the workspace over the first of them
    assert _Abi().paged(t=1 << 22, o=1 << 50, os=(1 << 40, 64), ws=1 << 50, mp=512, ld=512) == E


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs the host C++ compiler")
def test_offsets_of_a_row_s_parts_fit_32_bits(tmp_path):
    _run_check(tmp_path, "cache_join_check")


def _kernels(path):
    """What the compiler wrote beside each kernel of a built library: {name: metadata}."""
    msgpack = pytest.importorskip("msgpack")
    data, found, at = path.read_bytes(), {}, -1
    while (at := data.find(b"__CLANG_OFFLOAD_BUNDLE__", at + 1)) >= 0:
        entry = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            start, size, n = struct.unpack_from("<QQQ", data, entry)
            target, entry = data[entry + 24:entry + 24 + n], entry + 24 + n
            elf = data[at + start:at + start + size]
            if b"amdgcn" not in target or elf[:4] != b"\x7fELF":
                continue
            sections, = struct.unpack_from("<Q", elf, 40)
            each, count = struct.unpack_from("<HH", elf, 58)
            for i in range(count):
                kind, = struct.unpack_from("<I", elf, sections + i * each + 4)
                note, = struct.unpack_from("<Q", elf, sections + i * each + 24)
                if kind != 7:  # notes
                    continue
                name_len, len_, type_ = struct.unpack_from("<III", elf, note)
                if type_ == 32 and elf[note + 12:note + 18] == b"AMDGPU":
                    note += 12 + (name_len + 3) // 4 * 4
                    for k in msgpack.unpackb(elf[note:note + len_], strict_map_key=False)["amdhsa.kernels"]:
                        found[k[".name"]] = k
    return found


def test_attention_over_16_bits_keeps_its_registers():
    """The kernels of calls over a 16-bit cache share their source with those over 8 bits and of trees; what only these
    need costs them no scratch memory (bytes a lane: none, and 48 and 52 for tiles at head dim 128, as before)."""
    kernels = {n: k for n, k in _kernels(_C.LIB_PATH).items() if "seq_attn_" in n}
    of16 = {n: k for n, k in kernels.items() if n.endswith("ELi1EEEvNS_11SeqAttnArgsE")}
    assert len(of16) == 8 and len(kernels) > len(of16)
    for name, k in of16.items():
        tiles128 = "Li128ELb0E" in name
        assert k[".private_segment_fixed_size"] <= (64 if tiles128 else 0), name
