"""What the entry points of beam search and the paged cache refuse, in Python and at the C ABI, before
anything is launched.  Runs without a GPU."""

import ctypes

import pytest
import torch


def test_select_refuses():
    from bdm_amd import ops
    logits, scores = torch.zeros(2, 3, 8), torch.zeros(2, 3)
    ended, lengths = torch.zeros(2, 3, dtype=torch.bool), torch.zeros(2, 3, dtype=torch.int32)
    bad = [
        (logits[0], scores, {}), (logits.half(), scores, {}), (logits, scores[:1], {}), (logits, scores.double(), {}),
        (logits, scores, dict(width=0)), (logits, scores, dict(width=25)), (logits[:, :0], scores[:, :0], {}),
        (logits[..., :0], scores, {}), (logits, scores, dict(finished=ended)),
        (logits, scores, dict(finished=ended.int(), eos=1)), (logits, scores, dict(finished=ended[:1], eos=1)),
        (logits, scores, dict(eos=8)), (logits, scores, dict(eos=-1)), (logits, scores, dict(lengths=lengths.long())),
        (logits, scores, dict(length_penalty=1.0)),
        (logits, scores, {}),  # CPU tensors
    ]
    for x, s, options in bad:
        with pytest.raises(ValueError):
            ops.beam_select(x, s, **options)
    with pytest.raises(NotImplementedError):
        ops.beam_select(torch.zeros(1, 65, 8), torch.zeros(1, 65))
    with pytest.raises(NotImplementedError):
        ops.beam_select(torch.zeros(1, 4, 80), torch.zeros(1, 4), width=65)


def test_reorder_refuses():
    from bdm_amd import ops
    state, parents = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    ops.reorder_states([], parents, beams=4)
    for states, rows, beams in (([state], parents.int(), 4), ([state], parents, 3), ([state], parents, 0),
                                ([state], parents, 4)):
        with pytest.raises(ValueError):
            ops.reorder_states(states, rows, beams=beams)
    with pytest.raises(NotImplementedError):
        ops.reorder_states([torch.zeros(65, 2)], torch.zeros(65, dtype=torch.int64), beams=65)


def test_c_entry_points_refuse():
    from bdm_amd import _lib
    lib = _lib.library()
    assert lib.bdm_beam_select(None, None, 0, None) == -1
    assert lib.bdm_beam_select_workspace_size(None) == 0
    args = _lib.BeamArgs()
    assert lib.bdm_beam_select(ctypes.byref(args), None, 0, None) == -1
    args.batch, args.beams, args.vocab, args.width, args.dtype = 2, 4, 50000, 4, _lib.BDM_BF16
    assert lib.bdm_beam_select(ctypes.byref(args), None, 0, None) == -1 and b'null' in lib.bdm_last_error_string()
    for name in ('logits', 'scores', 'out_scores', 'out_tokens', 'out_parents'):
        setattr(args, name, 4096)
    assert lib.bdm_beam_select_workspace_size(ctypes.byref(args)) > 0
    assert lib.bdm_beam_select(ctypes.byref(args), None, 0, None) == -3
    args.finished, args.eos = 4096, 50000
    assert lib.bdm_beam_select(ctypes.byref(args), None, 0, None) == -1
    args.eos, args.length_penalty = 0, 1.0
    assert lib.bdm_beam_select(ctypes.byref(args), None, 0, None) == -1
    args.lengths, args.length_penalty = 4096, float('nan')
    assert lib.bdm_beam_select(ctypes.byref(args), None, 0, None) == -1
    args.length_penalty, args.beams = 0.0, 65
    assert lib.bdm_beam_select(ctypes.byref(args), None, 0, None) == -2
    args.beams, args.batch = 4, 0
    assert lib.bdm_beam_select(ctypes.byref(args), None, 0, None) == 0
    assert lib.bdm_reorder_states(None, None, 1, None, 1, 4, None) == -1
    assert lib.bdm_reorder_states(None, None, 1, None, 1, 65, None) == -2
    assert lib.bdm_reorder_states(None, None, 0, None, 1, 4, None) == 0
    pointer, size = (ctypes.c_void_p * 1)(None), (ctypes.c_int64 * 1)(16)
    assert lib.bdm_reorder_states(pointer, size, 1, 4096, 1, 4, None) == -1


def test_pages_refuse():
    from bdm_amd import BankPages
    sizes = dict(banks=8, heads=1, bank_size=8, head_width=16)
    for args, options in (((0, 4), sizes), ((4, 0), sizes), ((4, 4), {**sizes, 'layers': 0}), ((4, 4.0), sizes),
                          ((4, 4), {**sizes, 'dtype': torch.float16}), ((4, 4), {**sizes, 'device': 'cpu'})):
        with pytest.raises(ValueError):
            BankPages(*args, **options)
    pool, table = torch.zeros(4, 1, 8, 16), torch.zeros(1, 2, 8, dtype=torch.int32)
    with pytest.raises(ValueError):
        BankPages.over(pool, table, torch.zeros(4, dtype=torch.int32))  # CPU tensors


def test_c_pages_refuse():
    from bdm_amd import _lib
    lib = _lib.library()
    pages, ref = _lib.Pages(), None
    ref = ctypes.byref(pages)
    assert lib.bdm_pages_fork(None, None, None, 0, None) == -1
    assert lib.bdm_pages_fork(ref, 4096, None, 0, None) == -1
    pages.pages, pages.layers, pages.sequences, pages.banks = 64, 2, 4, 8
    pages.heads, pages.bank_size, pages.head_width, pages.dtype = 1, 8, 16, _lib.BDM_BF16
    assert lib.bdm_pages_fork(ref, 4096, None, 4, None) == -1 and b'null' in lib.bdm_last_error_string()
    for name in ('pool', 'table', 'references', 'free_bits', 'status'):
        setattr(pages, name, 4096)
    rows = (ctypes.c_int32 * 2)(1, 1)
    assert lib.bdm_pages_fork(ref, None, rows, 2, None) == -1          # a sequence twice
    assert lib.bdm_pages_fork(ref, 4096, rows, 1, None) == -1          # parents and a list
    assert lib.bdm_pages_fork(ref, 4096, None, 5, None) == -1          # more than the sequences
    assert lib.bdm_pages_fork(ref, None, None, 0, None) == 0
    assert lib.bdm_pages_load(ref, 2, rows, 1, -1, 4096, 4096, 1 << 20, None) == -1   # layer
    assert lib.bdm_pages_load(ref, 0, rows, 2, -1, 4096, 4096, 1 << 20, None) == -1
    assert lib.bdm_pages_load(ref, 0, rows, 1, 1, 4096, 4096, 1 << 20, None) == -1    # the base itself
    assert lib.bdm_pages_load(ref, 0, rows, 1, 4, 4096, 4096, 1 << 20, None) == -1
    assert lib.bdm_pages_load(ref, 0, rows, 1, 0, None, 4096, 1 << 20, None) == -1
    assert lib.bdm_pages_load(ref, 0, rows, 1, 0, 4096, 4096, 8, None) == -3
    assert lib.bdm_pages_load(ref, 0, rows, 0, 0, None, None, 0, None) == 0
    assert lib.bdm_pages_dense(ref, 0, rows, 2, 4096, None) == -1
    assert lib.bdm_pages_dense(ref, 0, rows, 1, None, None) == -1
    assert lib.bdm_pages_compact(ref, None, 0, None) == -3
    step = _lib.DecodeArgs()
    assert lib.bdm_pages_decode(ref, 0, None, None, 0, None) == -1
    assert lib.bdm_pages_decode(ref, 0, ctypes.byref(step), 4096, 1 << 20, None) == -1
    step.batch, step.heads, step.bank_size, step.head_width, step.bank_count = 4, 1, 8, 16, 8
    step.write_banks = step.read_banks = 2
    step.ctrl_dtype = step.state_dtype = _lib.BDM_BF16
    assert lib.bdm_pages_decode(ref, 0, ctypes.byref(step), 4096, 1 << 20, None) == -1   # null operands
    step.write_banks = 17
    assert lib.bdm_pages_decode(ref, 0, ctypes.byref(step), 4096, 1 << 20, None) == -2
    pages.sequences = 513
    assert lib.bdm_pages_fork(ref, 4096, None, 0, None) == -2


def test_struct_mirrors(tmp_path):
    import os
    import subprocess
    from bdm_amd import _lib
    from conftest import ROOT
    mirrors = {'bdm_beam_args': _lib.BeamArgs, 'bdm_pages': _lib.Pages}
    lines = [f'printf("%zu\\n", sizeof({s}));' + ''.join(f'printf("%zu\\n", offsetof({s}, {f}));' for f, _ in m._fields_)
             for s, m in mirrors.items()]
    source = tmp_path / 'm.c'
    source.write_text('#include <stdio.h>\n#include "bdm_hip.h"\nint main(void){' + ''.join(lines) + 'return 0;}')
    subprocess.run(['gcc', '-I', os.path.join(ROOT, 'include'), str(source), '-o', str(tmp_path / 'm')], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / 'm')], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for m in mirrors.values():
        want += [ctypes.sizeof(m)] + [getattr(m, f).offset for f, _ in m._fields_]
    assert got == want


def test_c_entry_points_refuse_grids_of_more_threads_than_a_launch_has():
    """2^32 threads and more: nothing is launched, so a load, a step or a reordering is not left half done."""
    from bdm_amd import _lib
    lib = _lib.library()
    pages = _lib.Pages()
    ref = ctypes.byref(pages)
    pages.pages, pages.layers, pages.sequences, pages.banks = 1 << 20, 1, 512, 1 << 17
    pages.heads, pages.bank_size, pages.head_width, pages.dtype = 1, 1, 8, _lib.BDM_BF16
    for name in ('pool', 'table', 'references', 'free_bits', 'status'):
        setattr(pages, name, 4096)
    rows = (ctypes.c_int32 * 512)(*range(512))
    assert lib.bdm_pages_load(ref, 0, rows, 512, -1, 4096, 4096, 1 << 40, None) == -2
    assert lib.bdm_pages_dense(ref, 0, rows, 512, 4096, None) == -2
    pages.layers = 1 << 15
    assert lib.bdm_pages_fork(ref, 4096, None, 512, None) == -2
    pages.layers, pages.banks, pages.heads, pages.head_width = 1, 16, 1 << 15, 64
    step = _lib.DecodeArgs()
    step.batch, step.heads, step.bank_size, step.head_width, step.bank_count = 512, 1 << 15, 1, 64, 16
    step.write_banks = step.read_banks = 8
    step.ctrl_dtype = step.state_dtype = _lib.BDM_BF16
    for name in ('q', 'k', 'v', 'b', 'g', 'w', 'write_weights', 'read_weights', 'write_indices', 'read_indices', 'output'):
        setattr(step, name, 4096)
    assert lib.bdm_pages_decode(ref, 0, ctypes.byref(step), 4096, 1 << 20, None) == -2
    assert b'grid' in lib.bdm_last_error_string()
    # the 33rd tensor goes into a second launch
    pointers, sizes = (ctypes.c_void_p * 33)(*[4096] * 33), (ctypes.c_int64 * 33)(*[0] * 33)
    sizes[32] = 16
    assert lib.bdm_reorder_states(pointers, sizes, 33, 4096, 1 << 24, 2, None) == -2
    sizes[0], sizes[32] = 16, 1 << 45
    assert lib.bdm_reorder_states(pointers, sizes, 33, 4096, 1, 2, None) == -2
    args = _lib.BeamArgs()
    args.batch, args.beams, args.vocab, args.width, args.dtype = 1 << 18, 64, 4, 4, _lib.BDM_BF16
    for name in ('logits', 'scores', 'out_scores', 'out_tokens', 'out_parents'):
        setattr(args, name, 4096)
    assert lib.bdm_beam_select(ctypes.byref(args), 4096, 1 << 40, None) == -2
