"""Base of the dataclasses that keep a description of their fields (an argument struct) for their calls."""

from __future__ import annotations


class Described:
    """`describe()` derives what the calls take of the fields. Assigning a field derives it again; a value
    that does not fit the other fields raises and is not taken."""

    def __post_init__(self):
        self.describe()
        self._described = True

    def describe(self) -> None:
        raise NotImplementedError

    def __setattr__(self, name, value):
        known = self.__dict__.get("_described", False) and name in self.__dataclass_fields__
        old = getattr(self, name) if known else None
        object.__setattr__(self, name, value)
        if known:
            try:
                self.describe()
            except BaseException:
                object.__setattr__(self, name, old)
                raise
