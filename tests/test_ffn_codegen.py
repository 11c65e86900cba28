"""Properties of the generated gfx950 code that the feed-forward kernels rely on, as tests/test_codegen.py has them for the
GEMM kernels whose schedules they share: the accumulation registers are the source's alone, nothing spills to memory, no
register is named while an LDS read is still writing it, and the addresses that inline assembly takes are in scalar
registers.  hipcc cross-compiles without a GPU."""
import os
import re

import pytest

import test_codegen as gen

pytestmark = pytest.mark.skipif(not os.path.exists(gen.HIPCC), reason="hipcc not installed")

INSN = {2: "v_mfma_f32_16x16x32_bf16", 3: "v_mfma_f32_16x16x32_f16", 4: "v_mfma_i32_16x16x64_i8"}
_asm = {}


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    def get(source):
        if source not in _asm:
            _asm[source] = gen.device_asm(tmp_path_factory.mktemp("asm"), source)
        return _asm[source]
    return get


def kernels(text, name):
    """{mangled name: (operand kind, other template arguments)} of the instantiations of a kernel."""
    found = {}
    for k in gen.kernel_metadata(text):
        m = re.search(name + r"I((?:L[ib]\d+E)+)E", k)
        if m:
            args = [int(x) for x in re.findall(r"L[ib](\d+)E", m.group(1))]
            found[k] = (args[0], args[1:])
    return found


@pytest.mark.parametrize("source, name, count", [("ffn_rows.hip", "ffn_rows_kernel", 24), ("ffn_mid.hip", "ffn_mid_kernel", 7), ("ffn_small.hip", "ffn_small_kernel", 14),
                                                 ("ffn_quad.hip", "ffn_quad_kernel", 8), ("ffn_across.hip", "ffn_across_kernel", 8), ("ffn_join.hip", "ffn_join_kernel", 3),
                                                 ("quantize.hip", "quantize_i8_kernel", 27), ("ffn_backward.hip", "glu_backward_prepare_kernel", 2)])
def test_no_kernel_uses_memory_for_registers(asm, source, name, count):
    text = asm(source)
    meta, ks = gen.kernel_metadata(text), kernels(text, name)
    assert len(ks) == count, (source, len(ks))
    for k in ks:
        assert meta[k]["vgpr_spill_count"] == 0 and meta[k]["private_segment_fixed_size"] == 0, (k, meta[k])
        body = gen.kernel_body(text, k)
        assert "scratch_" not in body, k
        assert not re.search(r"v_pk_(add|mul|fma)_f32", body), k


@pytest.mark.parametrize("source, name", [("ffn_quad.hip", "ffn_quad_kernel"), ("ffn_across.hip", "ffn_across_kernel")])
def test_accumulators_of_the_256_tiles(asm, source, name):
    """Tile T of a wave is a[4T : 4T+3] in every matrix instruction, pairs back to back, 64 tiles per step and parity; read
    and cleared behind either parity and cleared once at the start, and named nowhere else."""
    text = asm(source)
    meta = gen.kernel_metadata(text)
    for k, (op, _) in kernels(text, name).items():
        body, insn = gen.kernel_body(text, k), INSN[op]
        assert meta[k]["agpr_count"] == 256 and meta[k]["vgpr_count"] <= 512, (k, meta[k])
        acc = [gen._acc_range(x) for x in re.findall(insn + r" a\[([0-9a-fx]+:[0-9a-fx]+)\]", body)]
        assert len(acc) == 256, (k, len(acc))
        for half in (acc[:128], acc[128:]):
            assert half[0::2] == half[1::2] == [(4 * t, 4 * t + 3) for t in range(64)], k
        assert len(re.findall(insn + r" a\[([0-9a-fx:]+)\], v\[\d+:\d+\], v\[\d+:\d+\], a\[\1\]", body)) == 256, k
        assert body.count("v_accvgpr_read_b32") == 512 and body.count("v_accvgpr_write_b32") == 768 and "v_accvgpr_mov" not in body, k
        assert len(re.findall(r"v_accvgpr_write_b32 a\[?[0-9a-fx]+\]?, 0", body)) == 768, k


@pytest.mark.parametrize("source, name", [("ffn_quad.hip", "ffn_quad_kernel"), ("ffn_across.hip", "ffn_across_kernel"), ("ffn_small.hip", "ffn_small_kernel"),
                                          ("ffn_mid.hip", "ffn_mid_kernel")])
def test_loads_into_lds_take_scalar_addresses(asm, source, name):
    text = asm(source)
    for k in kernels(text, name):
        body = gen.kernel_body(text, k)
        loads = re.findall(r"global_load_lds_dwordx4 (.*)", body)
        assert loads and all(re.fullmatch(r"v\d+, s\[\d+:\d+\]\s*", x.split(";")[0]) for x in loads), (k, loads[:2])
        m0 = re.findall(r"s_(?:add_u32|mov_b32) m0, (\S+)", body)
        assert m0 and all(re.fullmatch(r"s\d+,?|0x[0-9a-f]+,?|\d+,?", x) for x in m0), (k, sorted(set(m0))[:4])


def test_the_quad_schedule_waits_for_what_it_uses(asm):
    """A replay of both copies of the step with the in-order queue of LDS reads: no matrix instruction names a register that
    a read in flight will write, nothing is in flight at the end of a step, and at barrier X exactly the loads that the
    step itself has issued may be."""
    text = asm("ffn_quad.hip")
    for k, (op, _) in kernels(text, "ffn_quad_kernel").items():
        for step in gen._steps_of(gen.kernel_body(text, k), INSN[op]):
            lgkm, mfma_seen, loads, x_seen = [], 0, 0, False
            for line in step:
                what = line.split()[0]
                if what == "ds_read_b128":
                    lgkm.append(gen._reg_range(line.split()[1].rstrip(",")))
                elif what.startswith("global_load_lds"):
                    loads += not x_seen
                elif what == "s_waitcnt":
                    m = re.search(r"lgkmcnt\((\d+)\)", line)
                    if m:
                        lgkm = lgkm[max(0, len(lgkm) - int(m.group(1))):]
                    m = re.search(r"vmcnt\((\d+)\)", line)
                    if m:
                        assert int(m.group(1)) == loads, (k, line, loads)
                        x_seen = True
                elif what == INSN[op]:
                    mfma_seen += 1
                    busy = {r for d in lgkm for r in d}
                    for src in re.findall(r"v\[\d+:\d+\]", line):
                        assert not busy & set(gen._reg_range(src)), (k, mfma_seen, line)
            assert mfma_seen == 128 and x_seen and not lgkm, (k, mfma_seen, x_seen, len(lgkm))


def test_the_small_kernel_touches_no_register_in_flight(asm):
    text = asm("ffn_small.hip")
    meta = gen.kernel_metadata(text)
    for k, (op, (_, high)) in kernels(text, "ffn_small_kernel").items():
        body, insn = gen.kernel_body(text, k), INSN[op]
        assert meta[k]["agpr_count"] == 16 * high and meta[k]["vgpr_count"] <= 64 * high, (k, meta[k])
        assert gen.registers_touched_while_a_read_is_in_flight(body) == [], k
        assert body.count("v_accvgpr_read_b32") == 16 * high and body.count("v_accvgpr_write_b32") == 16 * high, k
        assert body.index("v_accvgpr_read_b32") > body.index("s_nop 15"), k     # behind the wait states after the last matrix instruction
        assert len(re.findall(insn + r" a\[([0-9a-fx:]+)\], v\[\d+:\d+\], v\[\d+:\d+\], a\[\1\]", body)) == 5 * 8 * high, k


def test_across_reads_lds_the_other_way_round(asm):
    """Per step 32 transposed reads for B, and for an A across its sum 32 more in place of 16 plain ones; two steps, and the
    first step's fragments before them (all of B, two rows of A)."""
    text = asm("ffn_across.hip")
    for k, (_, (across_a, *_rest)) in kernels(text, "ffn_across_kernel").items():
        body = gen.kernel_body(text, k)
        assert body.count("ds_read_b64_tr_b16") == (2 * 64 + 32 + 8 if across_a else 2 * 32 + 32), (k, body.count("ds_read_b64_tr_b16"))
        assert body.count("ds_read_b128") == (0 if across_a else 2 * 16 + 4), (k, body.count("ds_read_b128"))
        assert len(re.findall(r"^\s*s_barrier", body, re.M)) == 2 + 2 * 2, k


def test_the_pass_that_looks_for_the_largest_value_uses_no_memory_for_registers(asm):
    text = asm("ffn_backward.hip")
    meta = gen.kernel_metadata(text)
    (k,) = [k for k in meta if "glu_backward_largest_kernel" in k]
    assert meta[k]["vgpr_spill_count"] == 0 and meta[k]["private_segment_fixed_size"] == 0, meta[k]
    assert "scratch_" not in gen.kernel_body(text, k) and not re.search(r"v_pk_(add|mul|fma)_f32", gen.kernel_body(text, k))
