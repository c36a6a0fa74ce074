"""MI355X-native routed-memory path of the Block Delta Memory layer.

Public surface mirrors the reference packages ``bdm`` and ``bsdm``:
``BDMConfig``/``BSDMConfig``, the ``BankedDeltaMemory`` module (alias
``BlockSparseDeltaMemory``), the routed operator ``bank_training``, the
router ``product_key_route``, ``bank_occupancy`` (the bank-union
regularizer), ``written_banks`` (the copy-on-write state count at nested
prefixes), ``GraphDecoder`` (a layer's decode step replayed from a HIP
graph), ``beam_search`` over the language model with its ``beam_select`` and
``reorder_states``, and ``BankPages``, the paged copy-on-write cache.  Kernels live in ``libbdm_hip.so``.
"""

from .beam import BeamResult, beam_search
from .config import BDMConfig, BSDMConfig, near_square_factors, replay_interval
from .graphs import GraphDecoder, LanguageModelGraphDecoder
from .model import BankedDeltaMemory
from .ops import BeamSelection, beam_select, reorder_states, route_validation, set_route_validation
from .occupancy import bank_occupancy, written_banks
from .pages import BankPages
from .routed_update import bank_training, role_bank_training
from .routing import SharedResidualRouter, product_key_route

BlockSparseDeltaMemory = BankedDeltaMemory

__all__ = ['BDMConfig', 'BSDMConfig', 'BankPages', 'BankedDeltaMemory', 'BeamResult', 'BeamSelection',
           'BlockSparseDeltaMemory', 'GraphDecoder', 'LanguageModelGraphDecoder', 'beam_search', 'beam_select',
           'reorder_states',
           'SharedResidualRouter', 'bank_occupancy', 'bank_training', 'role_bank_training', 'product_key_route',
           'near_square_factors', 'replay_interval', 'route_validation', 'set_route_validation', 'written_banks']
