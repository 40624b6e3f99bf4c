"""Paged caches in 8 bits: the packed arguments have the header's layout, and what cannot be done is refused before anything is launched (CPU)."""
import pytest
import torch

from kvcomp_b200 import _lib, ops
from test_packed_arguments import _header_fields
from test_paged_arguments import letters


def flat(struct):
    """A structure's fields, those of a kvc_scales in it in their place."""
    import re, os  # noqa: E401
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "kvcomp_b200.h")).read()
    if re.search(r"kvc_scales scales;[^}]*\} %s;" % struct, text) is None:
        return _header_fields(struct)
    body = re.search(r"typedef struct \{([^}]*)\} %s;" % struct, text).group(1)
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        if decl.startswith("kvc_scales"):
            fields += [("scales." + n, x) for n, x in _header_fields("kvc_scales")]
            continue
        kind, names = re.match(r"(?:const )?(\w+)\s*(.*)", decl, re.S).groups()
        fields += [(n.strip(" *\n"), "q" if "*" in n else {"int64_t": "q", "int32_t": "i", "float": "f"}[kind]) for n in names.split(",")]
    return fields


@pytest.mark.parametrize("struct,packer", [("kvc_scales", "SCALES"), ("kvc_page_slots_args", "PAGE_SLOTS_ARGS"), ("kvc_page_shift_args", "PAGE_SHIFT_ARGS"),
                                           ("kvc_paged_rows_args", "PAGED_ROWS_ARGS")])
def test_layouts(struct, packer):
    assert "".join(letter for _, letter in flat(struct)) == letters(getattr(_lib, packer))


AT = 1 << 20


def values_of(call, **change):
    """Arguments that the checks accept (pointers are never followed by them), with changes: fields of the structure, or s_... of the scales."""
    rows = dict(q=AT, k=2 * AT, v=3 * AT, q_out=4 * AT, kpages=5 * AT, vpages=6 * AT, positions=AT, slots=AT, frequencies=AT, N=4, Hq=8, Hkv=2, D=128, rotary=64, n_pages=10, page_size=16, status=0,
                layout=0, inverse=0, type=0, factor=1.0, q_token=1024, q_head=128, k_token=256, k_head=128, v_token=256, v_head=128, out_token=1024, out_head=128,
                kp_page=4096, kp_row=256, kp_head=128, vp_page=4096, vp_row=256, vp_head=128)
    scales = dict(k=7 * AT, v=8 * AT, k_page=32, k_head=16, v_page=32, v_head=16, codes=1, reserved=0)
    if call == "kvc_paged_attn_codes":
        rows.update(table=AT, lengths=AT, out=4 * AT, lse=0, workspace=AT, workspace_bytes=1 << 40, B=4, table_stride=8, table_width=8, window=0, scaling=0.1)
    if call == "kvc_paged_rows":
        rows.update(k_out=2 * AT, v_out=3 * AT, reserved=0)
    if call == "kvc_page_slots":
        rows = dict(lengths=AT, table=AT, table_stride=8, table_width=8, B=4, page_size=16, tokens=10, slots=AT, starts=AT, status=0)
    if call == "kvc_page_shift":
        rows = dict(starts=AT, first=AT, positions=AT, B=4, tokens=10)
    for name, value in change.items():
        (scales if name.startswith("s_") else rows)[name[2:] if name.startswith("s_") else name] = value
    return rows, scales


def make(call, **change):
    rows, scales = values_of(call, **change)
    lib = _lib.load()
    packed = _lib.SCALES.pack(*(scales[n] for n, _ in _header_fields("kvc_scales")))
    if call == "kvc_paged_rows":
        rows.update({"scales." + n: v for n, v in scales.items()})
        return lib.kvc_paged_rows(_lib.PAGED_ROWS_ARGS.pack(*(rows[n] for n, _ in flat("kvc_paged_rows_args"))), None)
    if call == "kvc_rotary_store_codes":
        return lib.kvc_rotary_store_codes(_lib.ROTARY_ARGS.pack(*(rows[n] for n, _ in _header_fields("kvc_rotary_args"))), packed, None)
    if call == "kvc_paged_attn_codes":
        return lib.kvc_paged_attn_codes(_lib.PAGED_ATTN_ARGS.pack(*(rows[n] for n, _ in _header_fields("kvc_paged_attn_args"))), packed, None, 0, None)
    struct = {"kvc_page_slots": ("kvc_page_slots_args", _lib.PAGE_SLOTS_ARGS), "kvc_page_shift": ("kvc_page_shift_args", _lib.PAGE_SHIFT_ARGS)}[call]
    return getattr(lib, call)(struct[1].pack(*(rows[n] for n, _ in _header_fields(struct[0]))), None)


BAD = {
    "kvc_rotary_store_codes": [dict(k=0), dict(v=0), dict(kpages=0), dict(slots=0), dict(positions=0), dict(frequencies=0), dict(s_k=0), dict(s_v=0), dict(D=120), dict(D=0), dict(rotary=63),
                               dict(Hkv=0), dict(N=-1), dict(type=2), dict(layout=2), dict(s_codes=0), dict(s_codes=3), dict(kpages=5 * AT + 8), dict(kp_row=264), dict(s_k=7 * AT + 2), dict(page_size=0),
                               dict(n_pages=1 << 28), dict(kp_head=64), dict(s_k_head=8), dict(vpages=5 * AT), dict(s_v=7 * AT), dict(s_k=5 * AT), dict(q_out=2 * AT), dict(out_head=64),
                               dict(q_out=AT + 2), dict(k=5 * AT)],
    "kvc_paged_rows": [dict(kpages=0), dict(slots=0), dict(k_out=0), dict(s_k=0), dict(D=120), dict(D=0), dict(N=-1), dict(type=2), dict(s_codes=4), dict(k_out=2 * AT + 8), dict(kp_row=264),
                       dict(k_head=4), dict(page_size=0), dict(n_pages=1 << 28), dict(v_out=2 * AT), dict(k_out=5 * AT), dict(k_head=64), dict(s_v=8 * AT + 1), dict(Hkv=0)],
    "kvc_paged_attn_codes": [dict(s_k=0), dict(s_codes=0), dict(s_codes=7), dict(s_k_page=64), dict(s_v_head=32), dict(vp_row=512), dict(kp_row=264, vp_row=264), dict(kpages=0), dict(D=112),
                             dict(s_k=7 * AT + 2), dict(Hq=7), dict(type=2), dict(workspace=0), dict(kpages=5 * AT + 8)],
    "kvc_page_slots": [dict(lengths=0), dict(table=0), dict(slots=0), dict(starts=0), dict(B=-1), dict(tokens=-1), dict(tokens=1 << 31), dict(page_size=0), dict(table_width=1 << 28)],
    "kvc_page_shift": [dict(starts=0), dict(first=0), dict(positions=0), dict(B=-1), dict(tokens=-1)],
}


@pytest.mark.parametrize("call,change", [(c, d) for c in sorted(BAD) for d in BAD[c]], ids=str)
def test_refusals(call, change):
    assert make(call, **change) == 1
    assert call.replace("_codes", "").encode() in _lib.load().kvc_last_error()


@pytest.mark.parametrize("change,what", [(dict(k_out=7 * AT), "scales"), (dict(v_out=7 * AT + 16), "scales"), (dict(k_out=8 * AT), "scales"), (dict(v_out=8 * AT), "scales"), (dict(k_out=AT), "slots"),
                                         (dict(v_out=AT - 16), "slots"), (dict(k_out=7 * AT - 32), "scales"), (dict(s_codes=0, v_out=AT), "slots")], ids=str)
def test_rows_over_what_is_read(change, what):
    assert make("kvc_paged_rows", **change) == 1 and _lib.load().kvc_last_error().decode() == "kvc_paged_rows: an output overlaps the %s" % what


def test_rows_beside_what_is_read():
    """Neighbours are no overlap.  (So many rows that the call is refused for their number, behind these checks: nothing is launched wherever this runs.)"""
    far, n = dict(N=1 << 30, slots=1 << 48, s_k=1 << 49, s_v=(1 << 49) + AT, v_out=1 << 52), 1 << 50
    for at, what in (((1 << 48) + (4 << 30), None), ((1 << 48) + (4 << 30) - 16, "slots"), ((1 << 49) + AT + 10 * 32 * 4, None), ((1 << 49) + AT + 10 * 32 * 4 - 16, "scales"), (n, None)):
        assert make("kvc_paged_rows", **far, k_out=at) == 1
        assert _lib.load().kvc_last_error().decode() == "kvc_paged_rows: " + ("an output overlaps the " + what if what else "too many rows")


def test_null_and_nothing_to_do():
    lib = _lib.load()
    assert lib.kvc_rotary_store_codes(None, None, None) == 1 and lib.kvc_paged_rows(None, None) == 1 and lib.kvc_page_slots(None, None) == 1 and lib.kvc_page_shift(None, None) == 1
    assert lib.kvc_paged_attn_codes(None, None, None, 0, None) == 1
    assert make("kvc_rotary_store_codes", N=0) == 0 and make("kvc_paged_rows", N=0) == 0 and make("kvc_paged_attn_codes", B=0) == 0 and make("kvc_page_shift", tokens=0) == 0
    assert make("kvc_paged_attn_codes", workspace_bytes=100) == 3


def test_no_cpu_path():
    i, x = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 64, dtype=torch.float16)
    pool, scales = torch.zeros(4, 16, 2, 64, dtype=torch.int8), torch.zeros(4, 2, 16)
    for call in (lambda: ops.rotary_paged_store(None, x, x, i, i, None, pool, pool, kscales=scales, vscales=scales), lambda: ops.paged_rows(pool, pool, i, scales, scales, dtype=torch.float16),
                 lambda: ops.page_slots(i[None], i[:1], 16, 2), lambda: ops.page_shift(i, i[:1], i), lambda: ops.paged_attn(x, pool, pool, i[None], i, 1.0, kscales=scales, vscales=scales),
                 lambda: ops.paged_rows(pool, pool, i, scales, scales, dtype=torch.float32)):
        with pytest.raises(_lib.KvcError):
            call()
