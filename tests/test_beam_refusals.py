"""What beam search's entry points refuse, in Python and at the C ABI, before
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


def test_struct_mirrors(tmp_path):
    import os
    import subprocess
    from bdm_amd import _lib
    from conftest import ROOT
    mirrors = {'bdm_beam_args': _lib.BeamArgs}
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
