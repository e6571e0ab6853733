"""What stands for the torch binding where it does not load.

The binding is built for one torch; the calls that go through ctypes need none.
They stay usable without it, and every call that needs it raises ImportError.
"""

from __future__ import annotations


class NoBinding:
    def __init__(self, why: ImportError):
        message = (f"the torch binding of b200moe does not load ({why}); build it with "
                   "`python -m moe_serving_profile_b200.build`")

        def refuse(*args, **kwargs):
            raise ImportError(message) from why

        self._refuse = refuse
        self.QuantRows = type("QuantRows", (), {"__new__": refuse})
        self.Int8Matrix = type("Int8Matrix", (), {"__new__": refuse})

    def __getattr__(self, name: str):   # any function of the binding
        if name.startswith("__"):
            raise AttributeError(name)
        return self._refuse
