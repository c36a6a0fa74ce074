"""What the entry points of the log-probabilities, the clipping and the layer
norm refuse, before a device is touched."""

import ctypes

import pytest
import torch

from bdm_amd import LayerNorm, clip_gradients, gradient_norm, token_log_probs, token_loss
from bdm_amd import _lib, ops
from bdm_amd.lm import BDMConfig, LanguageModelConfig


def tokens(*shape):
    return torch.zeros(shape, dtype=torch.int64)


@pytest.mark.parametrize('logits,given,options,error', [
    (torch.zeros(3, 8), tokens(3), {}, ValueError),                                    # on the CPU
    (torch.zeros(3, 8, dtype=torch.float16), tokens(3), {}, ValueError),
    (torch.zeros(3, 8, dtype=torch.float64), tokens(3), {}, ValueError),
    (torch.zeros(()), tokens(), {}, ValueError),
    (torch.zeros(3, 0), tokens(3), {}, ValueError),
    (torch.zeros(3, 8), tokens(4), {}, ValueError),
    (torch.zeros(3, 8), tokens(3, 1), {}, ValueError),
    (torch.zeros(3, 8), tokens(3).int(), {}, ValueError),
    (torch.zeros(3, 8), tokens(3), dict(alternatives=9), ValueError),
    (torch.zeros(3, 8), tokens(3), dict(alternatives=-1), ValueError),
    (torch.zeros(3, 80), tokens(3), dict(alternatives=33), NotImplementedError),
])
def test_token_log_probs(logits, given, options, error):
    with pytest.raises(error):
        token_log_probs(logits, given, **options)
    if not options:
        with pytest.raises(error):
            token_loss(logits, given)


def test_token_gradient():
    stats = torch.zeros(3, 2)
    for options in (dict(grad_entropy=torch.zeros(3)), dict(grad_top_log_probs=torch.zeros(3, 1)),
                    dict(grad_loss=torch.zeros(()))):
        with pytest.raises(ValueError):
            ops.token_gradient(torch.zeros(3, 8), tokens(3), stats, **options)


@pytest.mark.parametrize('gradients,options', [
    ([torch.zeros(3)], {}),
    ([torch.zeros(3, dtype=torch.float16)], {}),
    ([torch.zeros(3, dtype=torch.int64)], {}),
    ([torch.zeros(3).to_sparse()], {}),
    ([torch.zeros(3)], dict(out=[])),
    ([torch.zeros(3)], dict(out=[None])),
    ([torch.zeros(3)], dict(out=[torch.zeros(4)])),
    ([torch.zeros(3)], dict(max_norm=-1.0)),
    ([torch.zeros(3)], dict(max_norm=float('nan'))),
])
def test_clipping(gradients, options):
    options = {'max_norm': 1.0, **options}
    with pytest.raises(ValueError):
        clip_gradients(gradients, **options)
    if list(options) == ['max_norm'] and options['max_norm'] == 1.0:
        with pytest.raises(ValueError):
            gradient_norm(gradients)


def test_layer_norm():
    x, w = torch.zeros(3, 8), torch.ones(8)
    for call in (lambda: ops.layer_norm(x, w, None, 1e-5),                                 # on the CPU
                 lambda: ops.layer_norm_backward(x, x, w, None, 1e-5),
                 lambda: ops._layer_norm_parameters(x.half(), w, None),
                 lambda: ops._layer_norm_parameters(x, torch.ones(9), None),
                 lambda: ops._layer_norm_parameters(x, w, torch.ones(8, dtype=torch.bfloat16)),
                 lambda: ops._layer_norm_parameters(torch.zeros(()), None, None),
                 lambda: ops._layer_norm_parameters(torch.zeros(3, 0), None, None)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        ops._layer_norm_parameters(torch.zeros(1, 16385), None, None)


def test_layer_norm_on_the_cpu():
    """torch's formula, with a residual too."""
    norm = LayerNorm(12)
    x, r = torch.randn(5, 12), torch.randn(5, 12)
    total, y = norm.add_norm(x, r)
    assert torch.equal(total, r + x)
    assert torch.allclose(y, torch.nn.functional.layer_norm(total, (12,), norm.weight, norm.bias, norm.eps))
    norm = LayerNorm(12, bias=False)
    assert norm.bias is None and torch.allclose(norm(x), torch.nn.functional.layer_norm(x, (12,), norm.weight, None, 1e-5))


def test_configuration():
    assert 'normalization' not in LanguageModelConfig(memory=BDMConfig()).record()
    assert LanguageModelConfig(memory=BDMConfig(), normalization='layer').record()['normalization'] == 'layer'
    with pytest.raises(ValueError, match='normalization'):
        LanguageModelConfig(memory=BDMConfig(), normalization='batch')


# ------------------------------------------------------------------ the C entries: pointers are never followed here

HELD = ctypes.c_void_p(4096)


def test_token_entries():
    lib = _lib.library()

    def status(**fields):
        a = _lib.TokenArgs()
        a.logits = a.tokens = a.log_probs = 4096
        a.rows, a.row_stride, a.vocab, a.dtype = 4, 8, 8, _lib.BDM_F32
        for name, value in fields.items():
            setattr(a, name, value)
        return lib.bdm_token_log_probs(ctypes.byref(a), None, 0, None)

    assert lib.bdm_token_log_probs(None, None, 0, None) == -1
    for fields in (dict(rows=-1), dict(vocab=0), dict(row_stride=-1), dict(dtype=7), dict(logits=None), dict(tokens=None),
                   dict(log_probs=None), dict(alternatives=9), dict(alternatives=-1), dict(alternatives=2)):
        assert status(**fields) == -1, fields
    assert status(alternatives=40, vocab=100) == -2
    assert status(vocab=2 ** 30 + 1) == -2
    assert status(rows=2 ** 32) == -2
    assert status(rows=0, logits=None) == 0

    def backward(**fields):
        a = _lib.TokenGradArgs()
        a.logits = a.tokens = a.stats = a.grad_logits = 4096
        a.rows, a.row_stride, a.vocab, a.dtype = 4, 8, 8, _lib.BDM_F32
        for name, value in fields.items():
            setattr(a, name, value)
        return lib.bdm_token_log_probs_backward(ctypes.byref(a), None)

    assert lib.bdm_token_log_probs_backward(None, None) == -1
    for fields in (dict(stats=None), dict(grad_logits=None), dict(grad_entropy=4096), dict(grad_top_log_probs=4096),
                   dict(grad_loss=4096), dict(vocab=-5), dict(dtype=9)):
        assert backward(**fields) == -1, fields
    assert lib.bdm_token_loss(HELD, HELD, -1, 0, HELD, HELD, None) == -1
    assert lib.bdm_token_loss(HELD, HELD, 4, 0, None, HELD, None) == -1
    assert lib.bdm_token_loss(None, HELD, 4, 0, HELD, HELD, None) == -1


def test_gradient_entries():
    lib = _lib.library()
    keep = []

    def arrays(data=4096, out=4096, size=8, dtype=_lib.BDM_F32, out_dtype=_lib.BDM_F32):
        made = ((ctypes.c_uint64 * 1)(data), (ctypes.c_uint64 * 1)(out), (ctypes.c_int64 * 1)(size),
                (ctypes.c_int32 * 1)(dtype), (ctypes.c_int32 * 1)(out_dtype))
        keep.append(made)
        return made

    def clip(count=1, max_norm=1.0, norm=HELD, workspace=HELD, nbytes=1 << 20, **fields):
        data, out, size, dtype, out_dtype = arrays(**fields)
        return lib.bdm_clip_gradients(data, out, size, dtype, out_dtype, count, max_norm, norm, workspace, nbytes, None)

    def norm(count=1, max_norm=1.0, norm=HELD, scale=None, workspace=HELD, nbytes=1 << 20, **fields):
        data, _, size, dtype, _ = arrays(**fields)
        return lib.bdm_gradient_norm(data, size, dtype, count, max_norm, norm, scale, workspace, nbytes, None)

    for fields in (dict(size=-1), dict(dtype=5), dict(data=0), dict(count=-1), dict(norm=None), dict(workspace=None),
                   dict(nbytes=4), dict(workspace=ctypes.c_void_p(4100))):
        assert clip(**fields) == norm(**fields) == -1, fields
    for fields in (dict(out=0), dict(out_dtype=3), dict(out=4100), dict(out=4096, out_dtype=_lib.BDM_BF16),
                   dict(max_norm=-1.0), dict(max_norm=float('nan'))):
        assert clip(**fields) == -1, fields
    assert norm(max_norm=-1.0, scale=HELD) == -1
    assert clip(size=2 ** 40 + 1) == norm(size=2 ** 40 + 1) == -2
    assert lib.bdm_clip_gradients(None, None, None, None, None, 1, 1.0, HELD, HELD, 1 << 20, None) == -1
    assert lib.bdm_gradient_norm(None, None, None, 1, 1.0, HELD, None, HELD, 1 << 20, None) == -1
    # a sum for each workgroup: one a chunk of 16384 elements, 2048 at most in all
    sizes = (ctypes.c_int64 * 3)(1, 16385, 0)
    assert lib.bdm_gradient_norm_workspace_size(sizes, 3) == 3 * 8
    many = (ctypes.c_int64 * 500)(*[2 ** 31] * 500)
    assert lib.bdm_gradient_norm_workspace_size(many, 500) <= (2048 + 64) * 8
    assert lib.bdm_gradient_norm_workspace_size(None, 0) == 8


def test_layer_norm_entries():
    lib = _lib.library()

    def forward(x=HELD, residual=None, out=HELD, total=None, rows=4, width=8, dtype=0, param=0):
        return lib.bdm_layer_norm(x, residual, None, None, total, out, rows, width, dtype, param, 1e-5, None)

    for fields in (dict(x=None), dict(out=None), dict(residual=HELD), dict(rows=-1), dict(width=0), dict(dtype=4),
                   dict(param=4)):
        assert forward(**fields) == -1, fields
    assert forward(width=16385) == forward(rows=2 ** 40) == -2
    assert forward(rows=0, x=None) == 0
    size = lib.bdm_layer_norm_backward_workspace_size(4, 8)
    assert size > 0 and lib.bdm_layer_norm_backward_workspace_size(0, 8) == 0

    def backward(x=HELD, dy=HELD, dx=HELD, rows=4, width=8, workspace=HELD, nbytes=size):
        return lib.bdm_layer_norm_backward(x, dy, None, None, dx, None, None, rows, width, 0, 0, 1e-5, workspace, nbytes,
                                           None)

    for fields in (dict(x=None), dict(dy=None), dict(dx=None), dict(workspace=None), dict(nbytes=size - 1),
                   dict(workspace=ctypes.c_void_p(4100)), dict(width=-1)):
        assert backward(**fields) == -1, fields
    assert backward(width=20000) == -2


def test_struct_layouts_match_the_header(tmp_path):
    """sizeof and offsetof of the two argument structs, compiled from the header with gcc, equal the ctypes mirrors."""
    import os
    import shutil
    import subprocess
    from conftest import ROOT
    gcc = shutil.which('gcc')
    if gcc is None:
        pytest.skip('no host C compiler')
    mirrors = {'bdm_token_args': _lib.TokenArgs, 'bdm_token_grad_args': _lib.TokenGradArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{os.path.join(ROOT, "include", "bdm_hip.h")}"',
             'int main(void) {']
    for struct, mirror in mirrors.items():
        lines.append(f'printf("%zu\\n", sizeof({struct}));')
        lines += [f'printf("%zu\\n", offsetof({struct}, {field}));' for field, _ in mirror._fields_]
    source, program = tmp_path / 'layout.c', tmp_path / 'layout'
    source.write_text('\n'.join([*lines, 'return 0; }']))
    subprocess.run([gcc, str(source), '-o', str(program)], check=True)
    got = [int(x) for x in subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for mirror in mirrors.values():
        want += [ctypes.sizeof(mirror), *(getattr(mirror, field).offset for field, _ in mirror._fields_)]
    assert got == want


def test_block_calls_an_own_norm():
    """A block's norm that has a forward of its own is called, not passed over by the residual add before it."""
    from bdm_amd import BSDMConfig
    from bdm_amd.lm import BDMLanguageModel, LanguageModelConfig

    class Halved(LayerNorm):
        def forward(self, x):
            return super().forward(x) * 0.5

    memory = BSDMConfig(dim=64, bank_count=16, bank_size=8, selected_banks=4, value_width=64, num_heads=2)
    block = BDMLanguageModel(LanguageModelConfig(memory=memory, vocab_size=50, layers=1, ffn_multiple_of=32,
                                                 normalization='layer')).layers[0]
    block.attention_norm = block.attention = torch.nn.Identity()
    block.feed_forward = torch.nn.Identity()
    block.ffn_norm = Halved(64)
    called = []
    block.ffn_norm.add_norm = lambda *a: called.append(a) or LayerNorm.add_norm(block.ffn_norm, *a)
    hidden = torch.randn(2, 3, 64)
    total = hidden + hidden
    assert torch.equal(block(hidden), total + block.ffn_norm(total))
    assert not called
